// preference.cu — losses of class scores by label log-probabilities: the
// log-probabilities themselves, the paired preference loss and the clipped
// policy loss with a KL term, each with the gradient of the scores.
//
// Per token row x of C scores with label y: lse = m + log sum exp(x - m), m = max x;
// lp = x[y] - lse; a loss with derivative g in lp has d/dx[c] = g ([c = y] - exp(x[c] - lse)).
//
// All of it is a stream over the scores: bound by HBM where the rows are read
// and written once (policy, forward, gradient), with one or two exponentials per
// value (16 a clock and SM) close behind for 16-bit scores. Rows are worked on
// in three ways:
//  * up to kSmallC classes: a thread per row, tiles of 32 rows copied through
//    shared memory so that global accesses are whole vectors (small_rows_kernel);
//  * rows of up to 8 KB: 8 to 32 lanes hold the row in registers (at most sixteen
//    16-byte vectors a lane), so it is read once for the maximum, the sum and the
//    gradient (cached_rows_kernel);
//  * longer rows of the policy loss: persistent blocks stream rows through a ring
//    in shared memory that bulk copies fill ahead of the work (ring_rows_kernel);
//    the forward alone scans them (scan_rows_kernel), and the gradient for given
//    statistics is elementwise (label_grad_kernel).
#include "score_rows.cuh"

#include <algorithm>

namespace mfm {
namespace {

constexpr int kNT = 256;
constexpr int kSmallC = 32;
constexpr int kSmallNT = 128;
constexpr int kSmallPerSm = 8;  // blocks of 64 registers a thread

// once a row: to the last bit or two
__device__ __forceinline__ float ratio_of(float d) { return expf(d); }
__device__ __forceinline__ double ratio_of(double d) { return exp_call(d); }

// x - off - log s with nothing rounded to 32 bits but the sum s itself: a sequence adds
// up hundreds of them, and a margin is the difference of two such sums.
template <class T, class A>
__device__ __noinline__ double exact_logprob(T x, A off, A s) {
    return (widen<double>(x) - (double)off) - log((double)s);
}

// What a row's loss needs, in global memory; which pointers are set goes by the mode.
enum Mode { STATS, POLICY, GRAD };

template <class A>
struct RowArgs {
    Labels labels;
    int64_t n, c;
    A* lp;         // log-probabilities, or
    double* lp64;  // the same unrounded, for sums over sequences
    // STATS
    A* lse;
    A* zero;            // cleared per token, or NULL
    unsigned* counter;  // cleared by the first block, or NULL
    // POLICY
    const A *old, *adv, *ref, *weight;
    A clip_lo, clip_hi, kl_coef;  // ratio bounds
    const double* wpart;          // partial sums of the weights
    int n_wpart;
    double* part;  // four sums per block
    A* stats;
    unsigned* done;      // blocks finished
    unsigned* empties;   // set where a row with a label has no score but -inf
    double* live_total;  // then: the weights' sum without such rows
    const unsigned* only_if;  // a second pass: only if this is set, for the gradient alone
    // GRAD
    const A *g, *lse_in;
    const double* scale;  // factor of every g, NULL = 1
    // The factor of a token's gradient: 0 for a masked one and for one whose derivative
    // is 0 (of no sequence, or of a pair of weight 0), whatever the scale: weights that
    // are NaN, or whose sum is too small to divide by, give one that is not finite.
    __device__ __forceinline__ A factor(A g, int y, A l, double s) const {
        if (y < 0 || l == minus_inf<A>() || g == A(0)) return A(0);
        return scale ? (A)((double)g * s) : g;
    }
};

// em1 = exp(u) - 1 and kl = exp(u) - u - 1. Below 1 both by the series of kl, where the
// differences would lose what is left: to u^11 / 11! in 32 bits (what is cut off is 2^-27
// of kl), to u^18 / 18! in 64 bits (2^-55).
__device__ __forceinline__ void kl_terms(float u, float& em1, float& kl) {
    if (fabsf(u) < 1.0f) {
        float r = 1.0f / 39916800.0f;
        r = r * u + 1.0f / 3628800.0f;
        r = r * u + 1.0f / 362880.0f;
        r = r * u + 1.0f / 40320.0f;
        r = r * u + 1.0f / 5040.0f;
        r = r * u + 1.0f / 720.0f;
        r = r * u + 1.0f / 120.0f;
        r = r * u + 1.0f / 24.0f;
        r = r * u + 1.0f / 6.0f;
        r = r * u + 0.5f;
        kl = r * u * u;
        em1 = u + kl;
    } else {
        em1 = expf(u) - 1.0f;
        kl = u == INFINITY ? u : em1 - u;
    }
}
__device__ __forceinline__ void kl_terms(double u, double& em1, double& kl) {
    em1 = expm1(u);
    if (fabs(u) < 1.0) {
        double r = 1.0 / 6402373705728000.0;
        r = r * u + 1.0 / 355687428096000.0;
        r = r * u + 1.0 / 20922789888000.0;
        r = r * u + 1.0 / 1307674368000.0;
        r = r * u + 1.0 / 87178291200.0;
        r = r * u + 1.0 / 6227020800.0;
        r = r * u + 1.0 / 479001600.0;
        r = r * u + 1.0 / 39916800.0;
        r = r * u + 1.0 / 3628800.0;
        r = r * u + 1.0 / 362880.0;
        r = r * u + 1.0 / 40320.0;
        r = r * u + 1.0 / 5040.0;
        r = r * u + 1.0 / 720.0;
        r = r * u + 1.0 / 120.0;
        r = r * u + 1.0 / 24.0;
        r = r * u + 1.0 / 6.0;
        r = r * u + 0.5;
        kl = r * u * u;
    } else {
        kl = u == INFINITY ? u : em1 - u;
    }
}

// A token's own inputs, loaded ahead of its row's statistics.
template <class A>
struct Token {
    A w = A(0), adv = A(0), old = A(0), ref = A(0);
    __device__ __forceinline__ void load(const RowArgs<A>& a, int64_t t) {
        w = a.weight ? a.weight[t] : A(1);
        adv = a.adv[t];
        old = a.old[t];
        if (a.ref) ref = a.ref[t];
    }
};

// A token's derivative g, and its weighted loss terms and weight e.
template <class A>
__device__ __forceinline__ A policy_terms(const RowArgs<A>& a, const Token<A>& k, A lp, bool live,
                                          double inv_total, A (&e)[4]) {
    e[0] = e[1] = e[2] = e[3] = A(0);
    // masked, or a token of weight 0: left out, whatever its ratio
    if (!live || k.w == A(0)) return A(0);
    const A ratio = ratio_of(lp - k.old);
    const A bent = fmin(fmax(ratio, a.clip_lo), a.clip_hi);
    // no advantage, no term, also where the ratio is beyond the type's range
    const A plain = k.adv == A(0) && ratio == ratio ? A(0) : ratio * k.adv;
    const bool cut = plain > bent * k.adv;
    A slope = cut ? A(0) : -plain, kl = A(0), part = A(0);
    if (a.ref) {
        A em1;
        kl_terms(k.ref - lp, em1, kl);
        if (a.kl_coef != A(0)) {  // without one the term may be infinite, and is not the loss's
            slope -= a.kl_coef * em1;
            part = a.kl_coef * kl;
        }
    }
    e[0] = k.w * (part - (cut ? bent * k.adv : plain));
    e[1] = k.w * kl;
    e[2] = cut ? k.w : A(0);
    e[3] = k.w;
    // in 64 bits: the inverse of very small or very large weights' sum leaves 32 bits
    return (A)((double)(k.w * slope) * inv_total);
}

template <class A>
__device__ __forceinline__ double weight_total(const RowArgs<A>& a) {  // on every lane
    wait_previous();
    double total = 0.0;
    for (int i = threadIdx.x & 31; i < a.n_wpart; i += 32) total += a.wpart[i];
    return warp_sum(total);
}

// 1 / the sum of the weights; weights that sum to 0 give gradient 0.
__device__ __forceinline__ double inverse(double total) { return total != 0.0 ? 1.0 / total : 0.0; }

// The block's four sums to `part`; the block that finishes last adds all of
// them, in block order, into the results. `total` is what the labels alone say: where
// rows turned out empty, the means are over the weights of the others (last sum).
template <class A>
__device__ __forceinline__ void policy_finish(const RowArgs<A>& a, const double (&e)[4],
                                              double total, double* sm) {
    __shared__ unsigned last;
    if (a.only_if) return;  // the first pass has done this
    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; ++i) a.part[4 * (int64_t)blockIdx.x + i] = e[i];
        __threadfence();
        last = atomicAdd(a.done, 1u) == gridDim.x - 1 ? 1u : 0u;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (int i = 3; i >= 0; --i) {
        if (i == 3 && !__ldcg(a.empties)) continue;
        double v = 0.0;
        for (int64_t b = threadIdx.x; b < gridDim.x; b += blockDim.x) v += __ldcg(a.part + 4 * b + i);
        v = block_sum(v, sm);
        if (i == 3)
            total = v;
        else if (threadIdx.x == 0)
            a.stats[i] = total != 0.0 ? (A)(v / total) : A(0);
    }
    if (threadIdx.x == 0) *a.live_total = total;
}

// Whether this is a second pass without a row to be done again. The gradient is scaled
// by the weights' sum, which may have been taken before any row's scores were read; a
// row of -inf then counts there by its label. So the kernel is launched once more, with
// the sum that leaves such rows out, and ends here unless there are any.
template <class A>
__device__ __forceinline__ bool idle_pass(const RowArgs<A>& a) {
    if (!a.only_if) return false;
    wait_previous();
    return *a.only_if == 0;
}

// ------------------------------------------------------------ few classes --

// The thread's row of the gradient: k e with e = exp(x - off) in v, and g + k e at the
// label (its e in ey), rounded once; 0 for a token without one (y < 0, where g is 0),
// whatever its scores are. TURN: the thread's first column is not 0.
template <class T, class A, int CW, bool TURN>
__device__ __forceinline__ void small_grad(T* row, const A (&v)[CW], int c, int first, A g, A k, A ey,
                                           int y) {
    int col = first;
#pragma unroll
    for (int j = 0; j < CW; ++j)
        if (j < c) {
            row[TURN ? col : j] = narrow<T>(g == A(0) ? A(0) : v[j] * k);
            if (TURN) col = col + 1 == c ? 0 : col + 1;
        }
    if (y >= 0 && g != A(0)) row[y] = narrow<T>(g + k * ey);  // there is no row[-1]
}

// c <= CW classes, a row in a thread's registers.
template <class T, class A, int CW, bool TURN, Mode M>
__global__ void __launch_bounds__(kSmallNT, IsF64<A>::value || CW > 16 ? 4 : kSmallPerSm)
    small_rows_kernel(const T* __restrict__ x, int64_t ld, T* __restrict__ out, int64_t ld_out,
                      RowArgs<A> a, bool whole_in, bool whole_out) {
    extern __shared__ uint4 small_smem[];  // per warp two tiles of kTileRows x c
    __shared__ double sm[kSmallNT / 32];
    const int c = (int)a.c, lane = threadIdx.x & 31;
    T* const tiles = reinterpret_cast<T*>(small_smem) + (threadIdx.x / 32) * (2 * kTileRows * c);
    const int first = TURN ? first_column<T>(c) : 0;
    if (M == POLICY && idle_pass(a)) return;
    if (M == GRAD) wait_previous();
    const double scale = M == GRAD && a.scale ? *a.scale : 1.0;
    double e[4] = {0.0, 0.0, 0.0, 0.0};
    const int64_t n_tiles = ceil_div(a.n, (int64_t)kTileRows), step = (int64_t)gridDim.x * (kSmallNT / 32);
    int64_t tile = (int64_t)blockIdx.x * (kSmallNT / 32) + threadIdx.x / 32;
    // the gradient goes from the last row to the first: the forward that read the
    // scores just before left the last ones in L2
    auto begin = [&](int64_t i) { return (M == GRAD ? n_tiles - 1 - i : i) * kTileRows; };
    auto rows_of = [&](int64_t t0) { return (int)(a.n - t0 < kTileRows ? a.n - t0 : kTileRows); };
    Token<A> tok;
    int y = -1;
    auto inputs = [&](int64_t t0) {  // a thread's own inputs of the tile
        y = -1;
        tok = Token<A>();
        if (lane >= rows_of(t0)) return;
        y = a.labels.in(t0 + lane, a.c);
        if (M == POLICY) tok.load(a, t0 + lane);
        if (M == GRAD) {
            tok.w = a.g[t0 + lane];
            tok.old = a.lse_in[t0 + lane];
        }
    };
    if (tile < n_tiles) {
        tile_fetch(x, ld, begin(tile), rows_of(begin(tile)), c, whole_in, tiles);
        inputs(begin(tile));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    const double total = M == POLICY ? weight_total(a) : 0.0, inv = inverse(total);
    for (int buf = 0; tile < n_tiles; tile += step, buf ^= 1) {
        const int64_t t0 = begin(tile), t = t0 + lane;
        const int rows = rows_of(t0), y_now = y;
        const Token<A> now = tok;
        if (tile + step < n_tiles) {
            const int64_t next = begin(tile + step);
            tile_fetch(x, ld, next, rows_of(next), c, whole_in, tiles + (buf ^ 1) * (kTileRows * c));
            inputs(next);
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        T* row = tiles + buf * (kTileRows * c) + lane * c;
        if (lane < rows) {
            A v[CW];
            A m = minus_inf<A>(), s = A(0);
            const A at = y_now >= 0 ? widen<A>(row[y_now]) : A(0);
            int col = first;
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                v[j] = minus_inf<A>();
                if (j < c) {
                    v[j] = widen<A>(row[TURN ? col : j]);
                    if (TURN) col = col + 1 == c ? 0 : col + 1;
                }
                if (M != GRAD) m = fmax(m, v[j]);
            }
            const A off = M == GRAD ? now.old : offset_of(m);
            if (M != GRAD) {
#pragma unroll
                for (int j = 0; j < CW; ++j) {
                    v[j] = exp_of(v[j] - off);
                    s += v[j];
                }
                const bool empty = m == minus_inf<A>() && s == A(0);
                const A ls = log_of(s);
                const bool live = y_now >= 0 && !empty;
                const A lp = live ? (at - off) - ls : A(0);
                if (a.lp) a.lp[t] = lp;
                if (M == STATS) {
                    if (a.lp64) a.lp64[t] = live ? exact_logprob(at, off, s) : 0.0;
                    if (a.lse) a.lse[t] = empty ? minus_inf<A>() : off + ls;
                    if (a.zero) a.zero[t] = A(0);
                } else {
                    A f[4];
                    const A g = policy_terms(a, now, lp, live, inv, f);
                    for (int i = 0; i < 4; ++i) e[i] += (double)f[i];
                    if (empty && y_now >= 0) *a.empties = 1;
                    if (out) small_grad<T, A, CW, TURN>(row, v, c, first, g, -g / s, exp_of(at - off), y_now);
                }
            } else {
                const A g = a.factor(now.w, y_now, off, scale);
#pragma unroll
                for (int j = 0; j < CW; ++j) v[j] = exp_of(v[j] - off);
                small_grad<T, A, CW, TURN>(row, v, c, first, g, -g, exp_of(at - off), y_now);
            }
        }
        __syncwarp();
        if (M != STATS && out) tile_put(out, ld_out, t0, rows, c, whole_out, tiles + buf * (kTileRows * c));
        __syncwarp();  // the tile's buffer is filled again
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (M == STATS) {
        if (a.counter && blockIdx.x == 0 && threadIdx.x == 0) *a.counter = 0;
    } else if (M == POLICY) {
        for (int i = 0; i < 4; ++i) e[i] = block_sum(e[i], sm);
        policy_finish(a, e, total, sm);
    }
}

// ---------------------------------------------------------- rows at once --

// Lane 0 of a group hands over the finished row: statistics, or loss terms and
// the gradient's two factors: out[c] = k exp(x[c] - off), plus g at the label.
template <class T, class A, Mode M>
struct RowResult {
    A g = A(0), k = A(0);
    A e[4] = {A(0), A(0), A(0), A(0)};
    __device__ __forceinline__ RowResult(const RowArgs<A>& a, const Token<A>& tok, int64_t t,
                                         int y, T xy, A m, A s, double inv_total, bool first) {
        const A off = offset_of(m);
        const bool empty = m == minus_inf<A>() && s == A(0);
        const bool live = y >= 0 && !empty;
        const A ls = log_of(s);
        const A lp = live ? (widen<A>(xy) - off) - ls : A(0);
        if (first && a.lp) a.lp[t] = lp;
        if (M == STATS) {
            if (first && a.lp64) a.lp64[t] = live ? exact_logprob(xy, off, s) : 0.0;
            if (first && a.lse) a.lse[t] = empty ? minus_inf<A>() : off + ls;
            if (first && a.zero) a.zero[t] = A(0);
        } else {
            g = policy_terms(a, tok, lp, live, inv_total, e);
            k = -g / s;
            if (first && empty && y >= 0) *a.empties = 1;
        }
    }
};

// Blocks per SM by the registers that K vectors take.
template <class A>
constexpr int cached_blocks(int k) { return IsF64<A>::value || k > 8 ? 2 : 4; }

// L lanes per row, the row in their registers: K vectors a lane. Persistent warps
// walk the rows, so what a block adds up, it adds up once.
template <class T, class A, int L, int K, Mode M>
__global__ void __launch_bounds__(kNT, cached_blocks<A>(K))
    cached_rows_kernel(const T* __restrict__ x, int64_t ld, T* __restrict__ out, int64_t ld_out,
                       RowArgs<A> a) {
    constexpr int V = 16 / sizeof(T), R = 32 / L;            // rows per warp
    constexpr int E = (2 * (V - 1) + L - 1) / L;             // edge elements per lane
    __shared__ double sums[kNT / 32];
    // a group's terms: in registers they would cost every lane eight (and spill)
    __shared__ double terms[M == POLICY ? 4 : 1][kNT / L];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    if (M == POLICY && idle_pass(a)) return;
    if (M == GRAD) wait_previous();
    const double total = M == POLICY ? weight_total(a) : 0.0, inv = inverse(total);
    const double scale = M == GRAD && a.scale ? *a.scale : 1.0;
    if (M == POLICY && lane == 0)
        for (int i = 0; i < 4; ++i) terms[i][group] = 0.0;
    const int64_t warps = (int64_t)gridDim.x * (kNT / 32);
    for (int64_t t0 = ((int64_t)blockIdx.x * (kNT / 32) + threadIdx.x / 32) * R; t0 < a.n; t0 += warps * R) {
        // the gradient goes from the last row to the first: the forward that read
        // the scores just before left the last ones in L2
        const int64_t at = t0 + threadIdx.x % 32 / L, t = M == GRAD ? a.n - 1 - at : at;
        const bool in = at < a.n;
        const T* row = x + (in ? t : 0) * ld;
        const RowShape<T> sh(row, in ? (int)a.c : 0);
        uint4 v[K];
        A edge[E];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int j = lane + i * L;
            v[i] = j < sh.nv ? load16(row + sh.head + j * V) : Pack<T>::minus_inf();
        }
#pragma unroll
        for (int i = 0; i < E; ++i)
            edge[i] = lane + i * L < sh.edges ? widen<A>(row[sh.edge(lane + i * L)]) : minus_inf<A>();
        const int y = in ? a.labels.in(t, a.c) : -1;
        const T xy = row[y >= 0 ? y : 0];  // the label's score, on its way with the row
        Token<A> tok;
        if (M == POLICY && in) tok.load(a, t);
        A off, g = A(0), k = A(0);
        if (M == GRAD) {
            off = in ? a.lse_in[t] : A(0);
            g = a.factor(in ? a.g[t] : A(0), y, off, scale);
            k = -g;
        } else {
            A m = edge[0];
#pragma unroll
            for (int i = 1; i < E; ++i) m = fmax(m, edge[i]);
#pragma unroll
            for (int i = 0; i < K; ++i) m = fmax(m, Pack<T>::top(v[i]));
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
            off = offset_of(m);
            ExpSum<A> ex(off);
#pragma unroll
            for (int i = 0; i < K; ++i) {
                A p[V];
                Pack<T>::unpack(v[i], p);
                ex.add(p);
            }
            A s = ex.sum();
#pragma unroll
            for (int i = 0; i < E; ++i) s += exp_of(edge[i] - off);
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (in) {
                const RowResult<T, A, M> r(a, tok, t, y, xy, m, s, inv, lane == 0);
                g = r.g;
                k = r.k;
                if (M == POLICY && lane == 0)
                    for (int i = 0; i < 4; ++i) terms[i][group] += (double)r.e[i];
            }
        }
        if (M != STATS && out && in) {
            T* to = out + t * ld_out;
            const bool whole = alike(row, to), none = g == A(0);
            const ExpSum<A> ex(off);
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (lane + i * L < sh.edges) {
                    const int j = sh.edge(lane + i * L);
                    to[j] = narrow<T>(none ? A(0) : (j == y ? g : A(0)) + k * exp_of(edge[i] - off));
                }
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const int j = lane + i * L;
                if (j < sh.nv) {
                    A p[V];
                    if (none) {  // uniform over the row
#pragma unroll
                        for (int q = 0; q < V; ++q) p[q] = A(0);
                    } else {
                        Pack<T>::unpack(v[i], p);
                        ex.scaled(p, k);
                    }
                    store16<T, A>(to + sh.head + j * V, p, whole);
                }
            }
            if (!none && lane == label_lane<T, L>(sh, y)) to[y] = narrow<T>(g + k * exp_of(widen<A>(xy) - off));
        }
    }
    if (M == STATS) {
        if (a.counter && blockIdx.x == 0 && threadIdx.x == 0) *a.counter = 0;
    } else if (M == POLICY) {
        double e[4];
        for (int i = 0; i < 4; ++i) e[i] = block_sum(lane == 0 ? terms[i][group] : 0.0, sums);
        policy_finish(a, e, total, sums);
    }
}

// ------------------------------------------- long rows, statistics alone --

// Rows read once with a running maximum: L lanes a row, U vectors a lane in flight.
// What a row costs besides its values (reductions, log) is paid once a warp, so short
// rows take few lanes, long ones as many as keep their loads in flight, and few rows a
// whole block each. 32, 64, 128, 256 lanes a row, bf16: 60000 x 4096 92, 111, 178,
// 354 us; 100000 x 5000 184, 264, 291, 581; 8195 x 32000 108, 104, 98, 100; 2000 x 65536
// 66, 61, 63, 59; 50 x 65536 41, 27, 18, 12. (The rule takes 64 for the first two.)
template <class T, class A, int L>
__global__ void __launch_bounds__(kNT, IsF64<A>::value ? 2 : 4)
    scan_rows_kernel(const T* __restrict__ x, int64_t ld, RowArgs<A> a) {
    constexpr int V = 16 / sizeof(T), U = 8, W = L / 32;
    __shared__ A sm_m[kNT / 32], sm_s[kNT / 32];
    const int lane = threadIdx.x % L, warp = threadIdx.x / 32;
    const int64_t t = (int64_t)blockIdx.x * (kNT / L) + threadIdx.x / L;
    const bool in = t < a.n;
    const T* row = x + (in ? t : 0) * ld;
    const RowShape<T> sh(row, in ? (int)a.c : 0);
    const int y = in ? a.labels.in(t, a.c) : -1;
    const T edge = lane < sh.edges ? row[sh.edge(lane)] : narrow<T>(minus_inf<A>());
    RowStats<A> r{widen<A>(edge), A(0)};
    r.s = exp_of(r.m - offset_of(r.m));
    const T* at = row + sh.head;
    for (int j0 = lane; j0 < sh.nv; j0 += L * U) {
        uint4 v[U];
        A top = r.m;
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = j0 + u * L < sh.nv ? load16(at + (j0 + u * L) * V) : Pack<T>::minus_inf();
#pragma unroll
        for (int u = 0; u < U; ++u) top = fmax(top, Pack<T>::top(v[u]));
        if (top > r.m) {
            r.s *= exp_of(r.m - top);
            r.m = top;
        }
        ExpSum<A> ex(offset_of(r.m));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            A p[V];
            Pack<T>::unpack(v[u], p);
            ex.add(p);
        }
        r.s += ex.sum();
    }
    const T xy = row[y >= 0 ? y : 0];
    across(r, 32);
    if (W > 1) {
        if ((lane & 31) == 0) {
            sm_m[warp] = r.m;
            sm_s[warp] = r.s;
        }
        __syncthreads();
        r.m = sm_m[warp / W * W + (lane & (W - 1))];
        r.s = sm_s[warp / W * W + (lane & (W - 1))];
        across(r, W);
    }
    if (in) RowResult<T, A, STATS>(a, Token<A>(), t, y, xy, r.m, r.s, 0.0, lane == 0);
    if (a.counter && blockIdx.x == 0 && threadIdx.x == 0) *a.counter = 0;
}

// ------------------------------------------------------------- long rows --

// mbarriers and bulk copies. Every wait ends: after kWaitLimit polls it raises the
// block's flag, which ends all later waits at once; the block then runs to its
// end on whatever is in shared memory and reports NaN.
constexpr int kWaitLimit = 1 << 24;

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_at(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_at(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_at(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, unsigned parity) {
    unsigned ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_at(b)), "r"(parity)
        : "memory");
    return ok;
}
__device__ __forceinline__ void bar_wait(uint64_t* b, unsigned parity, volatile int* stop) {
    for (int i = 0; !bar_try(b, parity); ++i) {
        if (*stop) return;
        if (i >= kWaitLimit) {
            *stop = 1;
            return;
        }
    }
}
// 16-byte aligned addresses, bytes a multiple of 16.
__device__ __forceinline__ void bulk_copy(void* to, const void* from, unsigned bytes, uint64_t* b) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_at(to)), "l"(from), "r"(bytes), "r"(smem_at(b))
                 : "memory");
}

// Rows streamed through a ring of shared-memory chunks by bulk copies: one warp
// keeps copies of the rows ahead in flight while L threads work, so the loads do
// not stop for a row's reductions or its gradient. A row that fits the ring is
// kept there until its gradient is written; of a longer one the last chunks are,
// and the others come a second time, from L2. A chunk is kRingVecs vectors a
// thread. Two blocks of 256 threads an SM work on two rows: one's barrier and
// statistics hide behind the other's values (4096 x 65536 bf16: 218 us with one
// block of 512 that keeps whole rows, 217 us with two of 256 that keep half, 270 us
// with four of 128 that keep a quarter; 239 us with one of 768). Shorter rows take
// more and smaller blocks, since a row's statistics cost each of its warps about
// 250 instructions (16384 x 16384 bf16: 271, 236, 226 us with 256, 128, 64 threads
// a row; 8192 x 32000: 230 us with 256, 220 us with 128).
constexpr int kRingVecs = 4;
constexpr int kRingLanes = 512;  // of an SM
constexpr int ring_blocks(int L) { return kRingLanes / L; }
constexpr int ring_slots(int L) { return 200704 / ring_blocks(L) / (L * kRingVecs * 16); }
// How many of a row's chunks stay for its gradient: all, or as many as leave two
// slots for the others to pass through.
__host__ __device__ constexpr int kept_chunks(int chunks, int slots) { return chunks <= slots ? chunks : slots - 2; }

template <class T, class A, int L>
__global__ void __launch_bounds__(L + 32, ring_blocks(L))
    ring_rows_kernel(const T* __restrict__ x, int64_t ld, T* __restrict__ out, int64_t ld_out,
                     RowArgs<A> a) {
    constexpr int V = 16 / sizeof(T), S = ring_slots(L), CV = L * kRingVecs, W = L / 32;
    extern __shared__ uint4 ring[];  // S x CV
    __shared__ uint64_t full[S], empty[S];
    __shared__ A sm_m[2][W], sm_s[2][W];
    __shared__ double sums[32];
    __shared__ int stop_flag;
    volatile int* stop = &stop_flag;
    if (idle_pass(a)) return;
    if (threadIdx.x == 0) {
        stop_flag = 0;
        for (int i = 0; i < S; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], W);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const bool grad = out != nullptr;
    double e[4] = {0.0, 0.0, 0.0, 0.0}, total = 0.0;
    if (threadIdx.x >= L) {
        if (threadIdx.x == L) {
            unsigned seq = 0;
            for (int64_t t = blockIdx.x; t < a.n; t += gridDim.x) {
                const T* row = x + t * ld;
                const RowShape<T> sh(row, (int)a.c);
                const int chunks = (sh.nv + CV - 1) / CV;
                // the row, then for its gradient the chunks that were not kept
                const int all = chunks + (grad ? chunks - kept_chunks(chunks, S) : 0);
                for (int i = 0; i < all; ++i, ++seq) {
                    const unsigned slot = seq % S;
                    bar_wait(&empty[slot], (seq / S + 1) & 1, stop);
                    if (*stop) break;
                    const int c = i < chunks ? i : i - chunks, left = sh.nv - c * CV;
                    const unsigned bytes = (unsigned)(left < CV ? left : CV) * 16;
                    bar_expect(&full[slot], bytes);
                    bulk_copy(ring + slot * CV, row + sh.head + (int64_t)c * CV * V, bytes, &full[slot]);
                }
            }
            // copies in flight end before the block does
            for (unsigned q = seq > S ? seq - S : 0; q < seq; ++q)
                for (int i = 0; i < kWaitLimit && !bar_try(&full[q % S], (q / S) & 1); ++i) {}
        }
        __syncwarp();
    } else {
        const int lane = threadIdx.x, warp = lane / 32;
        unsigned seq = 0;
        int64_t t = blockIdx.x;
        int y = t < a.n ? a.labels.in(t, a.c) : -1;
        total = weight_total(a);
        const double inv = inverse(total);
        for (int it = 0; t < a.n; t += gridDim.x, ++it) {
            const T* row = x + t * ld;
            const RowShape<T> sh(row, (int)a.c);
            const int chunks = (sh.nv + CV - 1) / CV;
            const int kept = grad ? kept_chunks(chunks, S) : 0, again = chunks - kept;
            const T edge = lane < sh.edges ? row[sh.edge(lane)] : narrow<T>(minus_inf<A>());
            const T xy = row[y >= 0 ? y : 0];
            Token<A> tok;
            tok.load(a, t);
            const int64_t tn = t + gridDim.x;
            const int y_next = tn < a.n ? a.labels.in(tn, a.c) : -1;
            RowStats<A> r{widen<A>(edge), A(0)};
            r.s = exp_of(r.m - offset_of(r.m));
            for (int c = 0; c < chunks; ++c, ++seq) {
                const unsigned slot = seq % S;
                bar_wait(&full[slot], (seq / S) & 1, stop);
                const uint4* at = ring + slot * CV + lane;
                const int left = sh.nv - c * CV - lane;
                uint4 v[kRingVecs];
                A top = r.m;
#pragma unroll
                for (int u = 0; u < kRingVecs; ++u) v[u] = u * L < left ? at[u * L] : Pack<T>::minus_inf();
                if (c < again) {  // the chunk is in registers and not kept
                    __syncwarp();
                    if ((lane & 31) == 0) bar_arrive(&empty[slot]);
                }
#pragma unroll
                for (int u = 0; u < kRingVecs; ++u) top = fmax(top, Pack<T>::top(v[u]));
                if (top > r.m) {
                    r.s *= exp_of(r.m - top);
                    r.m = top;
                }
                ExpSum<A> ex(offset_of(r.m));
#pragma unroll
                for (int u = 0; u < kRingVecs; ++u) {
                    A p[V];
                    Pack<T>::unpack(v[u], p);
                    ex.add(p);
                }
                r.s += ex.sum();
            }
            // (m, s) over the warp, then over the block: one barrier a row
            across(r, 32);
            if ((lane & 31) == 0) {
                sm_m[it & 1][warp] = r.m;
                sm_s[it & 1][warp] = r.s;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(L) : "memory");
            r.m = (lane & 31) < W ? sm_m[it & 1][lane & 31] : minus_inf<A>();
            r.s = (lane & 31) < W ? sm_s[it & 1][lane & 31] : A(0);
            across(r, 32);
            const RowResult<T, A, POLICY> res(a, tok, t, y, xy, r.m, r.s, inv, lane == 0);
            for (int i = 0; i < 4; ++i) e[i] += (double)res.e[i];
            if (grad) {
                T* to = out + t * ld_out;
                const bool whole = alike(row, to), none = res.g == A(0);
                const A off = offset_of(r.m);
                const ExpSum<A> ex(off);
                if (lane < sh.edges) {
                    const int j = sh.edge(lane);
                    to[j] = none ? narrow<T>(A(0))
                                 : narrow<T>((j == y ? res.g : A(0)) + res.k * exp_of(widen<A>(edge) - off));
                }
                // the kept chunks again, the row's last, and behind them the others
                const unsigned kept_at = seq - (unsigned)kept;
                for (int i = 0; i < chunks; ++i) {
                    const int c = i < kept ? again + i : i - kept;
                    const unsigned at_seq = kept_at + (unsigned)i, slot = at_seq % S;
                    if (i >= kept) bar_wait(&full[slot], (at_seq / S) & 1, stop);
                    const uint4* at = ring + slot * CV + lane;
                    const int left = sh.nv - c * CV - lane;
                    uint4 v[kRingVecs];
#pragma unroll
                    for (int u = 0; u < kRingVecs; ++u)
                        if (u * L < left) v[u] = at[u * L];
                    __syncwarp();
                    if ((lane & 31) == 0) bar_arrive(&empty[slot]);
                    T* at_out = to + sh.head + (c * CV + lane) * V;
#pragma unroll
                    for (int u = 0; u < kRingVecs; ++u)
                        if (u * L < left) {
                            A p[V];
                            if (none) {  // uniform over the row
#pragma unroll
                                for (int q = 0; q < V; ++q) p[q] = A(0);
                            } else {
                                Pack<T>::unpack(v[u], p);
                                ex.scaled(p, res.k);
                            }
                            store16<T, A>(at_out + u * L * V, p, whole);
                        }
                }
                seq += (unsigned)again;
                if (!none && lane == label_lane<T, L>(sh, y)) to[y] = narrow<T>(res.g + res.k * exp_of(widen<A>(xy) - off));
            }
            if (*stop && lane == 0) {
                a.lp[t] = (A)NAN;
                e[0] = e[1] = e[2] = e[3] = NAN;
                if (a.only_if) a.stats[0] = (A)NAN;  // the first pass has written it
            }
            y = y_next;
        }
    }
    __syncthreads();
    total = weight_total(a);  // the copying warp too
    policy_finish(a, e, total, sums);
}

// ---------------------------------------------------------------- gradient --

// out = f ([c = y] - exp(x - lse)), f = g times *scale. Elementwise once lse is known. Rows
// are walked from the last to the first: the forward that read them just before
// left the last ones in L2.
template <class T, class A, int L>
__global__ void __launch_bounds__(kNT)
    label_grad_kernel(const T* __restrict__ x, int64_t ld, T* __restrict__ out, int64_t ld_out,
                      RowArgs<A> a) {
    wait_previous();
    constexpr int V = 16 / sizeof(T), U = 4;
    const int lane = threadIdx.x % L;
    const int64_t t = a.n - 1 - ((int64_t)blockIdx.x * (kNT / L) + threadIdx.x / L);
    if (t < 0) return;
    const T* row = x + t * ld;
    T* to = out + t * ld_out;
    const RowShape<T> sh(row, (int)a.c);
    const bool whole = alike(row, to);
    const int y = a.labels.in(t, a.c);
    const A l = a.lse_in[t], f = a.factor(a.g[t], y, l, a.scale ? *a.scale : 1.0);
    const T xy = row[y >= 0 ? y : 0];
    const bool none = f == A(0);
    if (lane < sh.edges) {
        const int j = sh.edge(lane);
        to[j] = narrow<T>(none ? A(0) : -f * exp_of(widen<A>(row[j]) - l) + (j == y ? f : A(0)));
    }
    const ExpSum<A> ex(l);
    for (int j0 = lane; j0 < sh.nv; j0 += L * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + u * L < sh.nv) v[u] = load16(row + sh.head + (j0 + u * L) * V);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + u * L < sh.nv) {
                A p[V];
                if (none) {  // uniform over the row
#pragma unroll
                    for (int q = 0; q < V; ++q) p[q] = A(0);
                } else {
                    Pack<T>::unpack(v[u], p);
                    ex.scaled(p, -f);
                }
                store16<T, A>(to + sh.head + (j0 + u * L) * V, p, whole);
            }
    }
    if (!none && lane == label_lane<T, L>(sh, y)) to[y] = narrow<T>(f - f * exp_of(widen<A>(xy) - l));
}

// Sums of v over [indptr[s], indptr[s+1]), one warp each, in float64.
__device__ __forceinline__ void seq_bounds(const int64_t* indptr, int64_t s, int64_t n, int64_t& lo,
                                           int64_t& hi) {
    lo = indptr[s];
    hi = indptr[s + 1];
    lo = lo < 0 ? 0 : (lo > n ? n : lo);
    hi = hi < lo ? lo : (hi > n ? n : hi);
}

template <class A>
__device__ __forceinline__ double warp_seq_sum(const A* v, int64_t lo, int64_t hi) {
    double a = 0.0;
    for (int64_t t = lo + (threadIdx.x & 31); t < hi; t += 32) a += (double)v[t];
    return warp_sum(a);
}

template <class A>
__global__ void __launch_bounds__(kNT)
    seq_sums_kernel(const A* __restrict__ lp, int64_t n, const int64_t* __restrict__ indptr,
                    int64_t n_seq, A* __restrict__ sums) {
    const int64_t s = (int64_t)blockIdx.x * (kNT / 32) + threadIdx.x / 32;
    if (s >= n_seq) return;
    int64_t lo, hi;
    seq_bounds(indptr, s, n, lo, hi);
    const double a = warp_seq_sum(lp, lo, hi);
    if ((threadIdx.x & 31) == 0) sums[s] = (A)a;
}

// One group of W threads per pair: sums, margin, the pair's weighted loss and its
// unnormalised derivative, written to every token of the two sequences. The block
// that finishes last adds the losses and the weights, in a fixed order.
template <class A, int W>
__global__ void __launch_bounds__(kNT)
    pair_kernel(const double* lp, int64_t n, const int64_t* __restrict__ indptr, int64_t n_pairs,
                const A* __restrict__ reference, double beta, double eps,
                const A* __restrict__ weight, A* __restrict__ margins, A* __restrict__ sums,
                double* __restrict__ pair_loss, A* g, unsigned* done, A* __restrict__ loss,
                double* __restrict__ scale) {
    after_previous();
    __shared__ double sm[kNT / 32];
    __shared__ unsigned last;
    const int64_t p = (int64_t)blockIdx.x * (kNT / W) + threadIdx.x / W;
    const int lane = threadIdx.x % W;
    if (p < n_pairs) {  // uniform over the group
        int64_t lo[2], hi[2];
        double s[2];
        for (int i = 0; i < 2; ++i) {
            seq_bounds(indptr, p + i * n_pairs, n, lo[i], hi[i]);
            s[i] = 0.0;
            for (int64_t t = lo[i] + lane; t < hi[i]; t += W) s[i] += lp[t];
            s[i] = W == 32 ? warp_sum(s[i]) : block_sum(s[i], sm);
        }
        const double z = beta * ((s[0] - (double)reference[p]) - (s[1] - (double)reference[n_pairs + p]));
        const double w = weight ? (double)weight[p] : 1.0;
        const double up = 1.0 / (1.0 + exp(-z)), down = 1.0 / (1.0 + exp(z));
        // a pair of weight 0 is left out, whatever its margin
        const double slope = w == 0.0 ? 0.0 : -beta * w * ((1.0 - eps) * down - eps * up);
        if (lane == 0) {
            margins[p] = (A)z;
            sums[p] = (A)s[0];
            sums[n_pairs + p] = (A)s[1];
            const double soft = log1p(exp(-fabs(z)));
            // a margin may be infinite (a label whose score is -infinity): a side without a
            // factor is left out, not multiplied by 0
            const double wrong = eps < 1.0 ? (1.0 - eps) * fmax(-z, 0.0) : 0.0, right = eps > 0.0 ? eps * fmax(z, 0.0) : 0.0;
            pair_loss[p] = w == 0.0 ? 0.0 : w * (soft + wrong + right);
        }
        if (g)
            for (int i = 0; i < 2; ++i)
                for (int64_t t = lo[i] + lane; t < hi[i]; t += W) g[t] = (A)(i ? -slope : slope);
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(done, 1u) == gridDim.x - 1 ? 1u : 0u;
    __syncthreads();
    if (!last) return;
    __threadfence();
    double a = 0.0, b = 0.0;
    for (int64_t q = threadIdx.x; q < n_pairs; q += kNT) {
        a += __ldcg(pair_loss + q);
        b += weight ? (double)weight[q] : 1.0;
    }
    a = block_sum(a, sm);
    b = block_sum(b, sm);
    if (threadIdx.x == 0) {
        *loss = b != 0.0 ? (A)(a / b) : A(0);
        *scale = b != 0.0 ? 1.0 / b : 0.0;
    }
}

template <class A>
__global__ void zero_loss_kernel(A* v, int n) {  // nothing to take a mean of
    if ((int)threadIdx.x < n) v[threadIdx.x] = A(0);
}

constexpr int kWeightBlocks = 512;

// Whether a row has no score but -infinity, by a whole warp.
template <class T>
__device__ __forceinline__ bool empty_row(const T* row, int c) {
    using A = typename Arith<T>::type;
    constexpr int V = Pack<T>::N, U = 4;
    const int lane = threadIdx.x & 31;
    const RowShape<T> sh(row, c);
    // != also holds for NaN, which is no empty row
    bool some = lane < sh.edges && widen<A>(row[sh.edge(lane)]) != minus_inf<A>();
    for (int j0 = 0; j0 < sh.nv && !__any_sync(0xffffffffu, some); j0 += 32 * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * 32 + lane;
            v[u] = j < sh.nv ? load16(row + sh.head + j * V) : Pack<T>::minus_inf();
        }
        const uint4 none = Pack<T>::minus_inf();
#pragma unroll
        for (int u = 0; u < U; ++u)
            some |= v[u].x != none.x || v[u].y != none.y || v[u].z != none.z || v[u].w != none.w;
    }
    return !__any_sync(0xffffffffu, some);
}

// A block's sum of weights; the first block clears the losses' block count and the mark
// of empty rows.
__device__ __forceinline__ void weight_part(double a, double* part, unsigned* done, unsigned* empties) {
    __shared__ double sm[kNT / 32];
    a = block_sum(a, sm);
    if (threadIdx.x == 0) {
        part[blockIdx.x] = a;
        if (blockIdx.x == 0) *done = *empties = 0;
    }
}

// Partial sums of the weights of the tokens with a label.
template <class A>
__global__ void __launch_bounds__(kNT)
    weight_kernel(Labels labels, int64_t c, const A* __restrict__ weight, int64_t n,
                  double* __restrict__ part, unsigned* __restrict__ done, unsigned* __restrict__ empties) {
    let_next();  // the rows' kernel needs the weights only once it has its first rows
    double a = 0.0;
    constexpr int U = 8;  // tokens in flight per thread
    for (int64_t t0 = (int64_t)blockIdx.x * kNT * U + threadIdx.x; t0 < n; t0 += (int64_t)gridDim.x * kNT * U) {
        int y[U];
        A w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + u * kNT;
            y[u] = t < n ? labels.in(t, c) : -1;
            w[u] = weight && t < n ? weight[t] : A(1);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (y[u] >= 0) a += (double)w[u];
    }
    weight_part(a, part, done, empties);
}

// The same without rows of -infinity: a row is looked at at its label's score, and read,
// up to the first score that is not -infinity, only where that one is. A warp takes
// `per` neighbouring tokens.
template <class T, class A>
__global__ void __launch_bounds__(kNT)
    weight_look_kernel(const T* __restrict__ x, int64_t ld, Labels labels, int64_t c,
                       const A* __restrict__ weight, int64_t n, int per, double* __restrict__ part,
                       unsigned* __restrict__ done, unsigned* __restrict__ empties) {
    let_next();
    double a = 0.0;
    const int lane = threadIdx.x & 31;
    const int64_t lo = ((int64_t)blockIdx.x * (kNT / 32) + threadIdx.x / 32) * per;
    const int64_t hi = lo + per < n ? lo + per : n;
    for (int64_t t0 = lo; t0 < hi; t0 += 32) {
        const int64_t t = t0 + lane;
        const int y = t < hi ? labels.in(t, c) : -1;
        const A w = weight && t < hi ? weight[t] : A(1);
        bool live = y >= 0;
        const bool low = live && widen<A>(x[t * ld + y]) == minus_inf<A>();
        for (unsigned m = __ballot_sync(0xffffffffu, low); m; m &= m - 1) {
            const int l = __ffs(m) - 1;
            if (empty_row(x + (t0 + l) * ld, (int)c) && l == lane) live = false;
        }
        if (live) a += (double)w;
    }
    weight_part(a, part, done, empties);
}

// Whether the weights are added up beside a look at the scores, or the rows' kernel is
// launched a second time in case that rows turn out empty. Small calls are bound by
// their launches (64 x 1000 bf16: 29 us a call with the look, 32 us with a second
// launch), large ones would read a sector of every row once more (1000003 x 10 float32:
// 44.7 us against 43.7 us; 16000 x 5000 float64: 635 us against 612 us).
inline bool looks_at_scores(int64_t n, int64_t c) { return n <= 65536 && n * c <= 1 << 22; }

// ------------------------------------------------------------- launchers --

// The most blocks of a policy kernel, each with its sums in the workspace (one wave is
// eight an SM at most).
constexpr unsigned kPolicyBlocks = 2048;

// A kernel over rows: the statistics start a chain of launches, the others go on in one.
template <Mode M, class K, class... Args>
void launch_rows(K kernel, unsigned grid, unsigned block, size_t smem, cudaStream_t s, Args... args) {
    if (M == POLICY) grid = std::min(grid, kPolicyBlocks);
    if (M == STATS)
        kernel<<<grid, block, smem, s>>>(args...);
    else
        launch_next(kernel, grid, block, smem, s, args...);
}

// Few classes: persistent warps over the tiles, whatever the mode.
template <class T, class A, Mode M>
void small_launch(int device, const T* x, int64_t ld, T* out, int64_t ld_out, const RowArgs<A>& a,
                  cudaStream_t s) {
    const size_t bytes = (size_t)(kSmallNT / 32) * 2 * kTileRows * a.c * sizeof(T);
    // one wave: the blocks an SM holds, by registers or by shared memory
    const int64_t fit = std::min<int64_t>(kSmallPerSm, (int64_t)(227 * 1024 / (bytes + 1280)));
    const int64_t blocks = ceil_div(a.n, kTileRows * (kSmallNT / 32)), most = (int64_t)sm_count(device) * fit;
    auto go = [&](auto w, auto turn) {
        auto k = small_rows_kernel<T, A, decltype(w)::value, decltype(turn)::value, M>;
        static bool asked[64];
        // the kernel's own arrays count towards the 48 KB that need no asking
        if (bytes + 1024 > 48 * 1024) allow_smem(k, device, 64 * 1024, asked, "class tile shared memory");
        launch_rows<M>(
            k, (unsigned)std::min(blocks, most), kSmallNT, bytes, s, x, ld, out, ld_out, a, ld == a.c && (uintptr_t)x % 16 == 0, ld_out == a.c && (uintptr_t)out % 16 == 0);
    };
    auto width = [&](auto turn) {
        if (a.c <= 4)
            go(std::integral_constant<int, 4>{}, turn);
        else if (a.c <= 8)
            go(std::integral_constant<int, 8>{}, turn);
        else if (a.c <= 12)
            go(std::integral_constant<int, 12>{}, turn);
        else if (a.c <= 16)
            go(std::integral_constant<int, 16>{}, turn);
        else
            go(std::integral_constant<int, kSmallC>{}, turn);
    };
    if (a.c % 4 == 0)
        width(std::true_type{});
    else
        width(std::false_type{});
}

// Rows of up to kCachedVecs vectors: the fewest lanes that hold one. Sixteen vectors a
// lane of a warp are the most that registers hold, and beat the ring and the elementwise
// gradient (60000 x 4096 bf16: policy 199 us against 268 us, gradient 159 us against
// 207 us; 100000 x 2049: 215 us against 303 us). The statistics alone stop at half of
// it: float32 rows of 2000 take 88 us by the scan, 96 us held (60000 rows), bf16 rows of
// 4096 the other way round 111 us and 100 us.
constexpr int64_t kCachedVecs = 512;

template <class T, class A, Mode M>
void cached_launch(int device, const T* x, int64_t ld, T* out, int64_t ld_out, const RowArgs<A>& a,
                   cudaStream_t s) {
    const int64_t nv = a.c / Pack<T>::N;
    auto go = [&](auto l, auto k) {
        constexpr int L = decltype(l)::value, K = decltype(k)::value;
        const int64_t blocks = ceil_div(a.n, (int64_t)kNT / L), most = (int64_t)sm_count(device) * cached_blocks<A>(K);
        launch_rows<M>(cached_rows_kernel<T, A, L, K, M>, (unsigned)std::min(blocks, most), kNT, 0, s, x, ld, out, ld_out, a);
    };
    using std::integral_constant;
    if (nv <= 16)
        go(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else if (nv <= 32)
        go(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    else if (nv <= 64)
        go(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    else if (nv <= 128)
        go(integral_constant<int, 32>{}, integral_constant<int, 4>{});
    else if (nv <= 256)
        go(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else
        go(integral_constant<int, 32>{}, integral_constant<int, 16>{});
}

// Launches the row kernel for c classes of type T: by the row's bytes, the fewest
// lanes that hold it in registers.
template <class T, class A, Mode M>
void rows_launch(int device, const T* x, int64_t ld, T* out, int64_t ld_out, const RowArgs<A>& a,
                 cudaStream_t s) {
    const int64_t n = a.n, nv = a.c / Pack<T>::N;  // a row's vectors, at most
    auto ring = [&](auto l) {
        constexpr int L = decltype(l)::value, bytes = ring_slots(L) * L * kRingVecs * 16;
        auto k = ring_rows_kernel<T, A, L>;
        static bool asked[64];
        allow_smem(k, device, bytes, asked, "row ring shared memory");
        const int64_t grid = (int64_t)sm_count(device) * ring_blocks(L);
        launch_rows<M>(k, (unsigned)(n < grid ? n : grid), L + 32, bytes, s, x, ld, out, ld_out, a);
    };
    auto scan = [&]() {
        const int64_t warps = (int64_t)sm_count(device) * 32;  // resident at once
        auto go = [&](auto l) {
            constexpr int L = decltype(l)::value;
            scan_rows_kernel<T, A, L><<<(unsigned)ceil_div(n, kNT / L), kNT, 0, s>>>(x, ld, a);
        };
        if (n * 4 < warps)
            go(std::integral_constant<int, kNT>{});
        else if (nv >= 1024)
            go(std::integral_constant<int, 128>{});
        else if (nv >= 512)
            go(std::integral_constant<int, 64>{});
        else
            go(std::integral_constant<int, 32>{});
    };
    using std::integral_constant;
    if (a.c <= kSmallC)
        small_launch<T, A, M>(device, x, ld, out, ld_out, a, s);
    else if (nv <= (M == STATS ? kCachedVecs / 2 : kCachedVecs))
        cached_launch<T, A, M>(device, x, ld, out, ld_out, a, s);
    else if constexpr (M == STATS)
        scan();
    else if (nv <= 2560)
        ring(integral_constant<int, kRingLanes / 8>{});
    else if (nv <= 5120)
        ring(integral_constant<int, kRingLanes / 4>{});
    else
        ring(integral_constant<int, kRingLanes / 2>{});
}

template <class T, class A>
void stats_launch(int device, const T* x, int64_t ld, int64_t n, int64_t c, Labels labels, A* lp,
                  double* lp64, A* lse, A* zero, unsigned* counter, cudaStream_t s) {
    if (n == 0) return;
    RowArgs<A> a{};
    a.labels = labels;
    a.n = n;
    a.c = c;
    a.lp = lp;
    a.lp64 = lp64;
    a.lse = lse;
    a.zero = zero;
    a.counter = counter;
    rows_launch<T, A, STATS>(device, x, ld, nullptr, 0, a, s);
    MFM_CHECK_LAUNCH("label log-probabilities launch");
}

// The gradient for given g and lse: elementwise. lse comes in the arithmetic type, as the
// forward returns it: in 32 bits a probability is off by |lse| 2^-24 of itself by that.
template <class T, class A>
void grad_launch(int device, const T* x, int64_t ld, int64_t n, int64_t c, Labels labels,
                 const A* g, const double* scale, const A* lse, T* out, int64_t ld_out,
                 cudaStream_t s) {
    if (n == 0) return;
    RowArgs<A> a{};
    a.labels = labels;
    a.n = n;
    a.c = c;
    a.g = g;
    a.scale = scale;
    a.lse_in = lse;
    if (c <= kSmallC)
        small_launch<T, A, GRAD>(device, x, ld, out, ld_out, a, s);
    else if (c / Pack<T>::N <= kCachedVecs)
        cached_launch<T, A, GRAD>(device, x, ld, out, ld_out, a, s);
    else
        launch_rows<GRAD>(label_grad_kernel<T, A, kNT>, (unsigned)n, kNT, 0, s, x, ld, out, ld_out, a);
    MFM_CHECK_LAUNCH("label gradient launch");
}

}  // namespace
}  // namespace mfm

using namespace mfm;

extern "C" int mfm_label_logprobs_device(int dtype, int device, const void* logits, int64_t ld,
                                         int64_t n_tokens, int64_t n_classes, int labels64,
                                         const void* labels, const int64_t* indptr, int64_t n_seq,
                                         void* logprobs, void* lse, void* sums, void* stream) {
    return guarded([&] {
        check_scores(dtype, logits, ld, n_tokens, n_classes, labels);
        if (n_tokens > 0 && (!logprobs || !lse)) fail(MFM_ERR_INVALID, "logprobs and lse must be provided");
        if (sums && (!indptr || n_seq < 0)) fail(MFM_ERR_INVALID, "sums need indptr and n_seq >= 0");
        if (sums && n_seq > INT32_MAX) fail(MFM_ERR_UNSUPPORTED, "n_seq exceeds the engine's 2^31-1 limit");
        DeviceGuard g(device);
        cudaStream_t s = (cudaStream_t)stream;
        with_score_types(dtype, [&](auto* t) {
            using T = Elem<decltype(t)>;
            using A = typename Arith<T>::type;
            stats_launch<T, A>(device, (const T*)logits, ld, n_tokens, n_classes, Labels{labels, labels64},
                               (A*)logprobs, nullptr, (A*)lse, nullptr, nullptr, s);
            if (sums && n_seq > 0) {
                seq_sums_kernel<A><<<(unsigned)ceil_div(n_seq, kNT / 32), kNT, 0, s>>>(
                    (const A*)logprobs, n_tokens, indptr, n_seq, (A*)sums);
                MFM_CHECK_LAUNCH("sequence sums launch");
            }
        });
    });
}

extern "C" int mfm_label_logprobs_grad_device(int dtype, int device, const void* logits,
                                              int64_t ld, int64_t n_tokens, int64_t n_classes,
                                              int labels64, const void* labels, const void* grad,
                                              const void* lse, void* d_logits, int64_t ld_out,
                                              void* stream) {
    return guarded([&] {
        check_scores(dtype, logits, ld, n_tokens, n_classes, labels);
        if (n_tokens == 0) return;
        if (!grad || !lse || !d_logits) fail(MFM_ERR_INVALID, "grad, lse and d_logits must be provided");
        check_out(d_logits, ld_out, n_tokens, n_classes);
        DeviceGuard g(device);
        with_score_types(dtype, [&](auto* t) {
            using T = Elem<decltype(t)>;
            using A = typename Arith<T>::type;
            grad_launch<T, A>(device, (const T*)logits, ld, n_tokens, n_classes,
                              Labels{labels, labels64}, (const A*)grad, nullptr, (const A*)lse,
                              (T*)d_logits, ld_out, (cudaStream_t)stream);
        });
    });
}

namespace {
struct PrefWs {  // log-probabilities, lse, token coefficients, pair losses, 1 / sum of weights and a block count
    size_t lse, g, pair, scale, bytes;
    PrefWs(int dtype, int64_t n, int64_t pairs) {
        const size_t a = up256((size_t)n * arith_size(dtype));
        lse = up256((size_t)n * 8);
        g = lse + a;
        pair = g + a;
        scale = pair + up256((size_t)pairs * 8);
        bytes = scale + 256;
    }
};
}  // namespace

extern "C" int64_t mfm_preference_workspace_bytes(int dtype, int64_t n_tokens, int64_t n_pairs) {
    if (n_tokens < 0 || n_pairs < 0) return 0;
    return (int64_t)PrefWs(dtype, n_tokens, n_pairs).bytes;
}

extern "C" int mfm_preference_loss_device(int dtype, int device, const void* logits, int64_t ld,
                                          int64_t n_tokens, int64_t n_classes, int labels64,
                                          const void* labels, const int64_t* indptr,
                                          int64_t n_pairs, const void* reference, double beta,
                                          double label_smoothing, const void* sample_weight,
                                          void* loss, void* margins, void* seq_logprobs,
                                          void* d_logits, int64_t ld_out, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_scores(dtype, logits, ld, n_tokens, n_classes, labels);
        if (n_pairs < 0) fail(MFM_ERR_INVALID, "n_pairs must be >= 0");
        if (n_pairs > INT32_MAX / 2) fail(MFM_ERR_UNSUPPORTED, "n_pairs exceeds the engine's 2^30-1 limit");
        if (!(label_smoothing >= 0.0 && label_smoothing <= 1.0))
            fail(MFM_ERR_INVALID, "label_smoothing must be in [0, 1]");
        if (!indptr || !loss) fail(MFM_ERR_INVALID, "indptr and loss must be provided");
        if (n_pairs > 0 && (!reference || !margins || !seq_logprobs))
            fail(MFM_ERR_INVALID, "reference, margins and seq_logprobs must be provided");
        check_out(d_logits, ld_out, n_tokens, n_classes);
        const PrefWs W(dtype, n_tokens, n_pairs);
        check_workspace(workspace, workspace_bytes, (int64_t)W.bytes);
        DeviceGuard g(device);
        cudaStream_t s = (cudaStream_t)stream;
        char* ws = (char*)workspace;
        double* pair = (double*)(ws + W.pair);
        double* scale = (double*)(ws + W.scale);
        unsigned* done = (unsigned*)(ws + W.scale + 8);
        with_score_types(dtype, [&](auto* t) {
            using T = Elem<decltype(t)>;
            using A = typename Arith<T>::type;
            double* lp = (double*)ws;
            A *lse = (A*)(ws + W.lse), *coef = d_logits ? (A*)(ws + W.g) : nullptr;
            const Labels y{labels, labels64};
            if (n_pairs == 0) zero_loss_kernel<A><<<1, 32, 0, s>>>((A*)loss, 1);
            if (n_pairs == 0 || n_tokens == 0)
                MFM_CUDA(cudaMemsetAsync(ws + W.scale, 0, 16, s), "memset");
            stats_launch<T, A>(device, (const T*)logits, ld, n_tokens, n_classes, y, nullptr, lp, lse, coef, done, s);
            if (n_pairs > 0) {
                auto pairs = [&](auto w) {
                    constexpr int PW = decltype(w)::value;
                    launch_next(pair_kernel<A, PW>, (unsigned)ceil_div(n_pairs, kNT / PW), kNT, 0, s,
                        lp, n_tokens, indptr, n_pairs, (const A*)reference, beta, label_smoothing,
                        (const A*)sample_weight, (A*)margins, (A*)seq_logprobs, pair, coef, done,
                        (A*)loss, scale);
                };
                if (n_tokens / (2 * n_pairs) >= 64)  // a block only where a warp would loop
                    pairs(std::integral_constant<int, kNT>{});
                else
                    pairs(std::integral_constant<int, 32>{});
            }
            MFM_CHECK_LAUNCH("preference loss launch");
            if (d_logits)
                grad_launch<T, A>(device, (const T*)logits, ld, n_tokens, n_classes, y, coef, scale,
                                  lse, (T*)d_logits, ld_out, s);
        });
    });
}

namespace {
struct PolicyWs {  // partial weights, a block count, the mark and the sum of empty rows, partial loss terms
    size_t part, bytes;
    explicit PolicyWs(int64_t n) {
        part = up256(kWeightBlocks * 8 + 16);
        bytes = part + up256((size_t)std::min<int64_t>(n, kPolicyBlocks) * 32);
    }
};
}  // namespace

extern "C" int64_t mfm_policy_workspace_bytes(int dtype, int64_t n_tokens) {
    (void)dtype;
    if (n_tokens < 0) return 0;
    return (int64_t)PolicyWs(n_tokens).bytes;
}

extern "C" int mfm_policy_loss_device(int dtype, int device, const void* logits, int64_t ld,
                                      int64_t n_tokens, int64_t n_classes, int labels64,
                                      const void* labels, const void* old_logprobs,
                                      const void* advantages, const void* reference,
                                      double clip_low, double clip_high, double kl_coef,
                                      const void* sample_weight, void* stats, void* logprobs,
                                      void* d_logits, int64_t ld_out, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_scores(dtype, logits, ld, n_tokens, n_classes, labels);
        if (!(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0))
            fail(MFM_ERR_INVALID, "clip_low must be in [0, 1] and clip_high >= 0");
        if (kl_coef != 0.0 && !reference) fail(MFM_ERR_INVALID, "kl_coef needs reference");
        if (!stats) fail(MFM_ERR_INVALID, "stats must be provided");
        if (n_tokens > 0 && (!old_logprobs || !advantages || !logprobs))
            fail(MFM_ERR_INVALID, "old_logprobs, advantages and logprobs must be provided");
        check_out(d_logits, ld_out, n_tokens, n_classes);
        const PolicyWs W(n_tokens);
        check_workspace(workspace, workspace_bytes, (int64_t)W.bytes);
        DeviceGuard g(device);
        cudaStream_t s = (cudaStream_t)stream;
        char* ws = (char*)workspace;
        double *wpart = (double*)ws, *part = (double*)(ws + W.part);
        unsigned *done = (unsigned*)(wpart + kWeightBlocks), *empties = done + 1;
        const bool look = looks_at_scores(n_tokens, n_classes);
        // eight tokens a warp that looks, eight a thread otherwise, more beyond the most blocks
        const int nw = (int)std::min<int64_t>(kWeightBlocks, ceil_div(n_tokens, look ? 8 * (kNT / 32) : 8 * kNT));
        with_score_types(dtype, [&](auto* t) {
            using T = Elem<decltype(t)>;
            using A = typename Arith<T>::type;
            if (n_tokens == 0) {
                zero_loss_kernel<A><<<1, 32, 0, s>>>((A*)stats, 3);
            } else {
                RowArgs<A> a{};
                a.labels = Labels{labels, labels64};
                a.n = n_tokens;
                a.c = n_classes;
                a.lp = (A*)logprobs;
                a.old = (const A*)old_logprobs;
                a.adv = (const A*)advantages;
                a.ref = (const A*)reference;
                a.weight = (const A*)sample_weight;
                a.clip_lo = (A)(1.0 - clip_low);
                a.clip_hi = (A)(1.0 + clip_high);
                a.kl_coef = (A)kl_coef;
                a.wpart = wpart;
                a.n_wpart = nw;
                a.part = part;
                a.stats = (A*)stats;
                a.done = done;
                a.empties = empties;
                a.live_total = wpart + kWeightBlocks + 1;
                if (look)
                    weight_look_kernel<T, A><<<nw, kNT, 0, s>>>((const T*)logits, ld, a.labels, n_classes, a.weight, n_tokens,
                                                                (int)ceil_div(n_tokens, (int64_t)nw * (kNT / 32)), wpart, done, empties);
                else
                    weight_kernel<A><<<nw, kNT, 0, s>>>(a.labels, n_classes, a.weight, n_tokens, wpart, done, empties);
                rows_launch<T, A, POLICY>(device, (const T*)logits, ld, (T*)d_logits, ld_out, a, s);
                if (d_logits && !look) {
                    a.wpart = a.live_total;
                    a.n_wpart = 1;
                    a.only_if = empties;
                    rows_launch<T, A, POLICY>(device, (const T*)logits, ld, (T*)d_logits, ld_out, a, s);
                }
            }
            MFM_CHECK_LAUNCH("policy loss launch");
        });
    });
}
