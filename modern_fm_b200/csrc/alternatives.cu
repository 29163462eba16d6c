// alternatives.cu — what else a row of class scores says: its label's log-probability
// and rank, the entropy and the best classes, and the gradient of the scores for the
// gradients of all of these.
//
// Per row x of C scores: m = max x, S = sum exp(x - m), D = sum exp(x - m) (x - m);
// lse = m + log S, entropy = log S - D / S; classes are ordered by falling score, ties by
// index. With p = exp(x - lse), G the sum of the log-probabilities' gradients (the
// label's and the best classes') and gH the entropy's:
//   d/dx[c] = sum of the gradients of log-probabilities of class c - p (G + gH (x - lse + entropy))
//
// Bound by HBM: the scores are read once (the gradient reads and writes them once), one
// exponential a value.
#include "score_rows.cuh"

#include <algorithm>

namespace mfm {
namespace {

constexpr int kNT = 256;
constexpr int kSmallC = 32;    // classes that a thread takes by itself
constexpr int kSmallNT = 128;
constexpr int kTop = 32;       // the most classes that are listed
constexpr int kCand = 288;     // candidates of a row: the vectors of kTop threads (256 values) and the row's edges

// x - off where its exponential is not 0, or so low that it is: 0 times it stays 0. (The
// exponential is taken of the difference itself, which may be NaN.)
__device__ __forceinline__ float floor_of(float d) { return fmaxf(d, -150.0f); }
__device__ __forceinline__ double floor_of(double d) { return fmax(d, -800.0); }

template <class A>
struct Args {
    Labels labels;  // p = NULL: none
    int64_t n, c;
    int top, ids64;
    A *lp, *lse, *entropy, *top_lp;
    void *ranks, *top_ids;
    __device__ __forceinline__ void id(void* at, int64_t i, int64_t v) const {
        if (ids64)
            static_cast<int64_t*>(at)[i] = v;
        else
            static_cast<int32_t*>(at)[i] = (int32_t)v;
    }
    // The label of a row, -1 for one that masks it; 0 without labels.
    __device__ __forceinline__ int label(int64_t t) const { return labels.p ? labels.in(t, c) : 0; }
    // A row without a result: masked by its label, or with no score but -infinity, or NaN.
    __device__ __forceinline__ void nothing(int64_t t, A l, A v) const {
        if (lp) lp[t] = v;
        lse[t] = l;
        entropy[t] = v;
        if (ranks) id(ranks, t, -1);
    }
    __device__ __forceinline__ void no_class(int64_t t, int j, A v) const {
        id(top_ids, t * top + j, -1);
        top_lp[t * top + j] = v;
    }
};

template <class A>
struct Stats {
    A m, s, d;  // maximum, sums of exp(x - m) and of exp(x - m) (x - m)
    // Taken relative to `to`, which is not below m.
    __device__ __forceinline__ void raise(A to) {
        if (m != minus_inf<A>()) {
            const A f = exp_of(m - to);
            d = f == A(0) ? A(0) : f * (d + s * (m - to));
            s *= f;
        }
        m = to;
    }
};

// The statistics of `width` neighbouring lanes joined, on each of them.
template <class A>
__device__ __forceinline__ void join(Stats<A>& r, int width) {
    A m = r.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < width) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    r.raise(m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < width) {
            r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
            r.d += __shfl_xor_sync(0xffffffffu, r.d, o);
        }
}

template <class A>
__device__ __forceinline__ A entropy_of(A ls, A s, A d) {
    const A h = ls - d / s;
    return h < A(0) ? A(0) : h;  // a rounding below 0; NaN stays
}

// ------------------------------------------------------------ few classes --

// A thread per row over tiles of 32 rows copied through shared memory. Every class's
// place is counted against every other: c (c - 1) / 2 comparisons.
template <class T, class A, int CW>
__global__ void __launch_bounds__(kSmallNT)
    small_kernel(const T* __restrict__ x, int64_t ld, Args<A> a, bool whole) {
    extern __shared__ uint4 small_smem[];
    const int c = (int)a.c, lane = threadIdx.x & 31;
    T* const tile = reinterpret_cast<T*>(small_smem) + (threadIdx.x / 32) * (kTileRows * c);
    const int64_t tiles = ceil_div(a.n, (int64_t)kTileRows);
    for (int64_t i = (int64_t)blockIdx.x * (kSmallNT / 32) + threadIdx.x / 32; i < tiles; i += (int64_t)gridDim.x * (kSmallNT / 32)) {
        const int64_t t0 = i * kTileRows, t = t0 + lane;
        const int rows = (int)(a.n - t0 < kTileRows ? a.n - t0 : kTileRows);
        tile_fetch(x, ld, t0, rows, c, whole, tile);
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        if (lane < rows) {
            const T* row = tile + lane * c;
            const int y = a.label(t);
            A v[CW], m = minus_inf<A>();
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                v[j] = j < c ? widen<A>(row[j]) : minus_inf<A>();
                m = fmax(m, v[j]);
            }
            const A off = offset_of(m);
            A s = A(0), d = A(0);
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                const A e = exp_of(v[j] - off);
                s += e;
                d += e * floor_of(v[j] - off);
            }
            const bool empty = m == minus_inf<A>() && s == A(0);
            if (y < 0 || empty || s != s) {
                const A v0 = y >= 0 && !empty ? s : A(0);
                a.nothing(t, y < 0 ? A(0) : empty ? minus_inf<A>() : s, v0);
                for (int j = 0; j < a.top; ++j) a.no_class(t, j, v0);
            } else {
                const A ls = log_of(s), xy = widen<A>(row[y]);
                a.lse[t] = off + ls;
                a.entropy[t] = entropy_of(ls, s, d);
                if (a.lp) a.lp[t] = (xy - off) - ls;
                int rank = 0, place[CW];
#pragma unroll
                for (int j = 0; j < CW; ++j) {
                    rank += j < c && (v[j] > xy || (v[j] == xy && j < y)) ? 1 : 0;
                    place[j] = 0;
                }
                if (a.ranks) a.id(a.ranks, t, rank);
                if (a.top) {
#pragma unroll
                    for (int j = 1; j < CW; ++j)
#pragma unroll
                        for (int q = 0; q < j; ++q)
                            if (v[j] > v[q])
                                ++place[q];
                            else
                                ++place[j];
#pragma unroll
                    for (int j = 0; j < CW; ++j)
                        if (j < c && place[j] < a.top) {
                            a.id(a.top_ids, t * a.top + place[j], j);
                            a.top_lp[t * a.top + place[j]] = (v[j] - off) - ls;
                        }
                }
            }
        }
        __syncwarp();  // the tile is filled again
    }
}

// --------------------------------------------------------------- any rows --

// A row's group of L threads within a block.
template <int L>
__device__ __forceinline__ void group_sync() {
    if (L == 32)
        __syncwarp();
    else if (L == kNT)
        __syncthreads();
    else
        asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.x / L), "n"(L) : "memory");
}

// exp and exp times its argument over N values.
template <int N>
__device__ __forceinline__ void add_terms(const float (&v)[N], float off, float& s, float& d) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
        const float z = v[q] - off, e = exp_of(z);
        s += e;
        d += e * floor_of(z);
    }
}
template <int N>
__device__ __forceinline__ void add_terms(const double (&v)[N], double off, double& s, double& d) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
        const double z = v[q] - off, e = exp_of(z);
        s += e;
        d += e * floor_of(z);
    }
}

template <class A>
struct Candidate {
    A v;
    int i;
    __device__ __forceinline__ bool before(const Candidate& o) const { return v > o.v || (v == o.v && i < o.i); }
};

constexpr int kSegments = 16;  // of a thread's vectors, each with its largest value

// What a group shares.
template <class A, int L>
struct Shared {
    A m[L / 32], s[L / 32], d[L / 32];
    int rank[L / 32];
    A sorted[L / 32][32];  // each warp's threads' largest values in falling order
    A most[kSegments][L];
    Candidate<A> cand[kCand];
    int count;
};

// The 32 lanes' values in falling order.
template <class A>
__device__ __forceinline__ A sorted_lanes(A v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 2; k <= 32; k *= 2)
#pragma unroll
        for (int j = k / 2; j > 0; j /= 2) {
            const A o = __shfl_xor_sync(0xffffffffu, v, j);
            const bool first = (lane & j) == 0, falling = (lane & k) == 0;
            v = first == falling ? fmax(v, o) : fmin(v, o);
        }
    return v;
}

// Walks the values of a row that thread `lane` of L has, by segments whose largest is at
// least `bound`: f(value, index).
template <class T, class A, int L, class F>
__device__ __forceinline__ void walk(const T* row, const RowShape<T>& sh, int lane, const Shared<A, L>& g, A mine,
                                     A bound, A edge, F&& f) {
    constexpr int V = 16 / sizeof(T), U = 8;
    if (!(mine >= bound)) return;
    if (lane < sh.edges && edge >= bound) f(edge, sh.edge(lane));
    const int batches = (sh.nv + L * U - 1) / (L * U), per = (batches + kSegments - 1) / kSegments;
    for (int b = 0; b < batches; ++b) {
        if (!(g.most[b / per][lane] >= bound)) continue;
        for (int u = 0; u < U; ++u) {
            const int j = (b * U + u) * L + lane;
            if (j >= sh.nv) break;
            A p[V];
            Pack<T>::unpack(load16(row + sh.head + (int64_t)j * V), p);
#pragma unroll
            for (int q = 0; q < V; ++q)
                if (p[q] >= bound) f(p[q], sh.head + j * V + q);
        }
    }
}

// The first `want` values of the row that equal v, in index order, by one warp:
// f(place, index).
template <class T, class A, class F>
__device__ __noinline__ void first_equal(const T* row, int c, A v, int want, F&& f) {
    const int lane = threadIdx.x & 31;
    int found = 0;
    for (int64_t j0 = 0; j0 < c && found < want; j0 += 32 * 8) {
        unsigned bits = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int64_t j = j0 + lane * 8 + q;
            if (j < c && widen<A>(row[j]) == v) bits |= 1u << q;
        }
        const int mine = __popc(bits);
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += other;
        }
        const int all = __shfl_sync(0xffffffffu, before, 31);
        before += found - mine;
        for (int q = 0; q < 8; ++q)
            if (bits >> q & 1) {
                if (before < want) f(before, (int)(j0 + lane * 8 + q));
                ++before;
            }
        found += all;
    }
}

template <class T, class A, int L>
__global__ void __launch_bounds__(kNT)
    rows_kernel(const T* __restrict__ x, int64_t ld, Args<A> a) {
    constexpr int V = 16 / sizeof(T), U = 8, W = L / 32;
    extern __shared__ uint4 rows_smem[];
    Shared<A, L>& g = reinterpret_cast<Shared<A, L>*>(rows_smem)[threadIdx.x / L];
    const int lane = threadIdx.x % L, warp = lane / 32;
    const int64_t t = (int64_t)blockIdx.x * (kNT / L) + threadIdx.x / L;
    if (t >= a.n) return;  // the whole group
    const int y = a.label(t), top = a.top;
    if (y < 0) {
        if (lane == 0) a.nothing(t, A(0), A(0));
        if (lane < top) a.no_class(t, lane, A(0));
        return;
    }
    const T* row = x + t * ld;
    const RowShape<T> sh(row, (int)a.c);
    const A xy = widen<A>(row[y]);
    const A edge = lane < sh.edges ? widen<A>(row[sh.edge(lane)]) : minus_inf<A>();
    const int batches = (sh.nv + L * U - 1) / (L * U), per = (batches + kSegments - 1) / kSegments;
    int rank = lane < sh.edges && (edge > xy || (edge == xy && sh.edge(lane) < y)) ? 1 : 0;
    Stats<A> r{edge, A(0), A(0)};
    r.s = exp_of(edge - offset_of(edge));  // 1, 0 for -infinity, NaN
    A part = minus_inf<A>();
    for (int b = 0; b < batches; ++b) {
        uint4 v[U];
        A best = minus_inf<A>();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = (b * U + u) * L + lane;
            v[u] = j < sh.nv ? load16(row + sh.head + (int64_t)j * V) : Pack<T>::minus_inf();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) best = fmax(best, Pack<T>::top(v[u]));
        part = b % per == 0 ? best : fmax(part, best);
        g.most[b / per][lane] = part;
        if (best > r.m) r.raise(best);
        const A off = offset_of(r.m);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            A p[V];
            Pack<T>::unpack(v[u], p);
            add_terms(p, off, r.s, r.d);
            const int i0 = sh.head + ((b * U + u) * L + lane) * V;
#pragma unroll
            for (int q = 0; q < V; ++q) rank += p[q] > xy || (p[q] == xy && i0 + q < y) ? 1 : 0;
        }
    }
    // -infinity behind the row's end counts as a tie of a label of -infinity
    if (xy == minus_inf<A>()) {
        rank = lane < sh.edges && (edge > xy || sh.edge(lane) < y) ? 1 : 0;
        for (int j = lane; j < sh.nv; j += L) {
            A p[V];
            Pack<T>::unpack(load16(row + sh.head + (int64_t)j * V), p);
#pragma unroll
            for (int q = 0; q < V; ++q) rank += p[q] > xy || sh.head + j * V + q < y ? 1 : 0;
        }
    }
    const A mine = r.m;
    join(r, 32);
    rank = __reduce_add_sync(0xffffffffu, rank);
    if (top) {
        const A in_order = sorted_lanes(mine);
        g.sorted[warp][lane & 31] = in_order;
    }
    if ((lane & 31) == 0) {
        g.m[warp] = r.m;
        g.s[warp] = r.s;
        g.d[warp] = r.d;
        g.rank[warp] = rank;
    }
    if (lane == 0) g.count = 0;
    group_sync<L>();
    if (W > 1) {
        const int w = lane & 31;
        r.m = w < W ? g.m[w] : minus_inf<A>();
        r.s = w < W ? g.s[w] : A(0);
        r.d = w < W ? g.d[w] : A(0);
        rank = w < W ? g.rank[w] : 0;
        join(r, 32);
        rank = __reduce_add_sync(0xffffffffu, rank);
    }
    const A off = offset_of(r.m), ls = log_of(r.s);
    const bool empty = r.m == minus_inf<A>() && r.s == A(0);
    if (empty || r.s != r.s) {
        const A v0 = empty ? A(0) : r.s;
        if (lane == 0) a.nothing(t, empty ? minus_inf<A>() : r.s, v0);
        if (lane < top) a.no_class(t, lane, v0);
        return;
    }
    if (lane == 0) {
        if (a.lp) a.lp[t] = (xy - off) - ls;
        a.lse[t] = off + ls;
        a.entropy[t] = entropy_of(ls, r.s, r.d);
        if (a.ranks) a.id(a.ranks, t, rank);
    }
    if (top == 0) return;
    // A value that at least `top` values of the row reach: the top-th of one warp's threads'
    // largest, or what ceil(top / W) threads of every warp reach.
    A one = minus_inf<A>(), every = (A)INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        one = fmax(one, g.sorted[w][top - 1]);
        every = fmin(every, g.sorted[w][(top + W - 1) / W - 1]);
    }
    const A bound = fmax(one, every);
    auto take = [&](A v, int i) {
        const int at = atomicAdd(&g.count, 1);
        if (at < kCand) g.cand[at] = Candidate<A>{v, i};
    };
    auto put = [&](int place, A v, int i) {
        a.id(a.top_ids, t * top + place, i);
        a.top_lp[t * top + place] = (v - off) - ls;
    };
    // the places of the candidates among each other: those below `top` are the answer
    auto choose = [&](int count) {
        for (int q = lane; q < count; q += L) {
            const Candidate<A> me = g.cand[q];
            int place = 0;
            for (int o = 0; o < count; ++o) place += g.cand[o].before(me) ? 1 : 0;
            if (place < top) put(place, me.v, me.i);
        }
    };
    walk<T, A, L>(row, sh, lane, g, mine, bound, edge, take);
    group_sync<L>();
    int count = g.count;
    if (count <= kCand) {
        choose(count);
        return;
    }
    // Too many reach it: mostly ties, as of masked classes. Those above it, and the first
    // of those that are equal.
    group_sync<L>();
    if (lane == 0) g.count = 0;
    group_sync<L>();
    walk<T, A, L>(row, sh, lane, g, mine, bound, edge, [&](A v, int i) {
        if (v > bound) take(v, i);
    });
    group_sync<L>();
    count = g.count;
    if (count <= kCand) {
        choose(count);
        if (count < top && warp == 0)
            first_equal<T, A>(row, (int)a.c, bound, top - count, [&](int place, int i) { put(count + place, bound, i); });
        return;
    }
    // Too many above it (a few threads hold most of the large values): one at a time, each
    // the first behind the one before.
    Candidate<A> last{(A)INFINITY, -1};
    for (int place = 0; place < top; ++place) {
        Candidate<A> best{minus_inf<A>(), INT32_MAX};
        for (int64_t j = lane; j < a.c; j += L) {
            const Candidate<A> o{widen<A>(row[j]), (int)j};
            if (last.before(o) && o.before(best)) best = o;
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) {
            const Candidate<A> o{__shfl_xor_sync(0xffffffffu, best.v, s), __shfl_xor_sync(0xffffffffu, best.i, s)};
            if (o.before(best)) best = o;
        }
        if (W > 1) {
            group_sync<L>();
            if ((lane & 31) == 0) g.cand[warp] = best;
            group_sync<L>();
            for (int w = 0; w < W; ++w)
                if (g.cand[w].before(best)) best = g.cand[w];
        }
        last = best;
        if (lane == 0) put(place, best.v, best.i);
    }
}

// ---------------------------------------------------------------- gradient --

template <class A>
struct GradArgs {
    Labels labels;  // p = NULL: none
    int64_t n, c;
    int top, ids64;
    const A *lse, *entropy, *g_lp, *g_entropy, *g_top;
    const void* top_ids;
    __device__ __forceinline__ int64_t id(int64_t i) const {
        return ids64 ? static_cast<const int64_t*>(top_ids)[i] : (int64_t)static_cast<const int32_t*>(top_ids)[i];
    }
};

// L threads a row: every value by p alone, then again those of the label and the best
// classes with their gradients, summed over all places that name the class.
template <class T, class A, int L>
__global__ void __launch_bounds__(kNT)
    grad_kernel(const T* __restrict__ x, int64_t ld, T* __restrict__ out, int64_t ld_out, GradArgs<A> a) {
    constexpr int V = 16 / sizeof(T), U = 4;
    __shared__ A own[kNT / L][kTop + 1];
    __shared__ int at[kNT / L][kTop + 1];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const int64_t t = a.n - 1 - ((int64_t)blockIdx.x * (kNT / L) + group);
    if (t < 0) return;  // the whole group
    const T* row = x + t * ld;
    T* to = out + t * ld_out;
    const RowShape<T> sh(row, (int)a.c);
    const bool whole = alike(row, to);
    const int y = a.labels.p ? a.labels.in(t, a.c) : 0;
    const A l = a.lse[t];
    const bool dead = y < 0 || l == minus_inf<A>();
    const int places = dead ? 0 : a.top + 1;  // the last one is the label's
    // places are at most 33, threads at least 32
    for (int j = lane; j < places; j += L) {
        const int64_t i = j < a.top ? a.id(t * a.top + j) : (int64_t)y;
        const bool in = i >= 0 && i < a.c && (j < a.top || a.g_lp);
        at[group][j] = in ? (int)i : -1;
        own[group][j] = in ? (j < a.top ? a.g_top[t * a.top + j] : a.g_lp[t]) : A(0);
    }
    group_sync<L>();
    A sum = A(0);
    for (int j = 0; j < places; ++j) sum += own[group][j];
    const A gh = dead || !a.g_entropy ? A(0) : a.g_entropy[t];
    const A h = gh == A(0) ? A(0) : a.entropy[t];
    const bool none = sum == A(0) && gh == A(0);
    auto slope = [&](A v) {
        const A z = v - l;
        return -exp_of(z) * (sum + gh * (floor_of(z) + h));
    };
    if (lane < sh.edges) {
        const int j = sh.edge(lane);
        to[j] = narrow<T>(none ? A(0) : slope(widen<A>(row[j])));
    }
    for (int j0 = lane; j0 < sh.nv; j0 += L * U) {
        uint4 v[U];
        if (!none) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j0 + u * L < sh.nv) v[u] = load16(row + sh.head + (int64_t)(j0 + u * L) * V);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + u * L < sh.nv) {
                A p[V];
                if (none) {
#pragma unroll
                    for (int q = 0; q < V; ++q) p[q] = A(0);
                } else {
                    Pack<T>::unpack(v[u], p);
#pragma unroll
                    for (int q = 0; q < V; ++q) p[q] = slope(p[q]);
                }
                store16<T, A>(to + sh.head + (int64_t)(j0 + u * L) * V, p, whole);
            }
    }
    group_sync<L>();  // the places' values come after all others
    for (int j = lane; j < places; j += L) {
        const int i = at[group][j];
        if (i < 0) continue;
        A mine = A(0);
        for (int o = 0; o < places; ++o)
            if (at[group][o] == i) mine += own[group][o];
        to[i] = narrow<T>(mine + (none ? A(0) : slope(widen<A>(row[i]))));
    }
}

// ------------------------------------------------------------- launchers --

template <class T, class A>
void rows_launch(int device, const T* x, int64_t ld, const Args<A>& a, cudaStream_t s) {
    if (a.c <= kSmallC) {
        const size_t bytes = (size_t)(kSmallNT / 32) * kTileRows * a.c * sizeof(T);
        const int64_t blocks = std::min(ceil_div(a.n, kTileRows * (kSmallNT / 32)), (int64_t)sm_count(device) * 16);
        const bool whole = ld == a.c && (uintptr_t)x % 16 == 0;
        auto go = [&](auto w) {
            small_kernel<T, A, decltype(w)::value><<<(unsigned)blocks, kSmallNT, bytes, s>>>(x, ld, a, whole);
        };
        if (a.c <= 8)
            go(std::integral_constant<int, 8>{});
        else if (a.c <= 16)
            go(std::integral_constant<int, 16>{});
        else
            go(std::integral_constant<int, 32>{});
        return;
    }
    auto go = [&](auto l) {
        constexpr int L = decltype(l)::value, bytes = (int)sizeof(Shared<A, L>) * (kNT / L);
        auto k = rows_kernel<T, A, L>;
        static bool asked[64];
        allow_smem(k, device, bytes, asked, "row shared memory");
        k<<<(unsigned)ceil_div(a.n, kNT / L), kNT, bytes, s>>>(x, ld, a);
    };
    const int64_t nv = a.c / Pack<T>::N, warps = (int64_t)sm_count(device) * 32;
    if (nv >= 1024 && a.n * 4 < warps)
        go(std::integral_constant<int, kNT>{});
    else if (nv >= 512)
        go(std::integral_constant<int, 128>{});
    else
        go(std::integral_constant<int, 32>{});
}

template <class T, class A>
void grad_launch(const T* x, int64_t ld, T* out, int64_t ld_out, const GradArgs<A>& a, cudaStream_t s) {
    auto go = [&](auto l) {
        constexpr int L = decltype(l)::value;
        grad_kernel<T, A, L><<<(unsigned)ceil_div(a.n, kNT / L), kNT, 0, s>>>(x, ld, out, ld_out, a);
    };
    if (a.c / Pack<T>::N >= 1024)
        go(std::integral_constant<int, kNT>{});
    else
        go(std::integral_constant<int, 32>{});
}

}  // namespace
}  // namespace mfm

using namespace mfm;

extern "C" int mfm_label_alternatives_device(int dtype, int device, const void* logits, int64_t ld, int64_t n_tokens,
                                             int64_t n_classes, int labels64, const void* labels, int top,
                                             void* logprobs, void* lse, void* entropy, void* ranks, void* top_ids,
                                             void* top_logprobs, void* stream) {
    return guarded([&] {
        check_scores(dtype, logits, ld, n_tokens, n_classes, labels ? labels : logits);
        if (top < 0 || top > kTop || top > n_classes)
            fail(MFM_ERR_INVALID, fmt("top must be in [0, min(%d, n_classes)]", kTop));
        if (n_tokens == 0) return;
        if (!lse || !entropy) fail(MFM_ERR_INVALID, "lse and entropy must be provided");
        if ((labels != nullptr) != (logprobs != nullptr) || (labels != nullptr) != (ranks != nullptr))
            fail(MFM_ERR_INVALID, "logprobs and ranks go with labels");
        if (top > 0 && (!top_ids || !top_logprobs)) fail(MFM_ERR_INVALID, "top_ids and top_logprobs must be provided");
        DeviceGuard guard(device);
        with_score_types(dtype, [&](auto* p) {
            using T = Elem<decltype(p)>;
            using A = typename Arith<T>::type;
            const Args<A> a{Labels{labels, labels64}, n_tokens, n_classes, top, labels64, (A*)logprobs, (A*)lse,
                            (A*)entropy, (A*)top_logprobs, ranks, top_ids};
            rows_launch<T, A>(device, (const T*)logits, ld, a, (cudaStream_t)stream);
        });
        MFM_CHECK_LAUNCH("label alternatives launch");
    });
}

extern "C" int mfm_label_alternatives_grad_device(int dtype, int device, const void* logits, int64_t ld,
                                                  int64_t n_tokens, int64_t n_classes, int labels64,
                                                  const void* labels, const void* lse, const void* entropy,
                                                  const void* grad_logprobs, const void* grad_entropy, int top,
                                                  const void* top_ids, const void* grad_top, void* d_logits,
                                                  int64_t ld_out, void* stream) {
    return guarded([&] {
        check_scores(dtype, logits, ld, n_tokens, n_classes, labels ? labels : logits);
        if (top < 0 || top > kTop) fail(MFM_ERR_INVALID, fmt("top must be in [0, %d]", kTop));
        if (n_tokens == 0) return;
        if (!lse || !d_logits) fail(MFM_ERR_INVALID, "lse and d_logits must be provided");
        if (grad_logprobs && !labels) fail(MFM_ERR_INVALID, "grad_logprobs needs labels");
        if (grad_entropy && !entropy) fail(MFM_ERR_INVALID, "grad_entropy needs entropy");
        if (top > 0 && (!top_ids || !grad_top)) fail(MFM_ERR_INVALID, "top_ids and grad_top must be provided");
        check_out(d_logits, ld_out, n_tokens, n_classes);
        DeviceGuard guard(device);
        with_score_types(dtype, [&](auto* p) {
            using T = Elem<decltype(p)>;
            using A = typename Arith<T>::type;
            const GradArgs<A> a{Labels{labels, labels64}, n_tokens, n_classes, top, labels64, (const A*)lse,
                                (const A*)entropy, (const A*)grad_logprobs, (const A*)grad_entropy,
                                (const A*)grad_top, top_ids};
            grad_launch<T, A>((const T*)logits, ld, (T*)d_logits, ld_out, a, (cudaStream_t)stream);
        });
        MFM_CHECK_LAUNCH("label alternatives gradient launch");
    });
}
