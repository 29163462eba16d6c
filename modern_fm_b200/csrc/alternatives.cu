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
// The scores are read once (the gradient reads and writes them once), one exponential a
// value: bound by HBM where rows are long (4096 x 65536 bf16: statistics 95 us, 5.7 TB/s;
// gradient 165 us, 6.1 TB/s), by issue slots where they are short, since what a row needs once
// (reductions, logarithm, the order of its best) costs its warp some 500 instructions. Rows are
// worked on in three ways:
//  * up to kSmallC classes: a thread per row (small_kernel, small_grad_kernel);
//  * rows of up to 256 vectors of 16 bytes: 4 to 32 lanes hold the row in registers
//    (held_kernel);
//  * longer ones: 32 to 256 threads scan the row with a running maximum, eight blocks of a
//    cluster where rows are few (scan_kernel); the gradient is elementwise (grad_kernel).
// The best classes come from a bound that at least `top` values of the row reach, known from
// the lanes' largest values: the few values that reach it are listed and ranked by
// counting. Where more reach it than the list holds (ties, masked classes), those above it are
// listed and the first of its equals follow.
#include "score_rows.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace mfm {
namespace {

constexpr int kNT = 256;
constexpr int kSmallC = 32;    // classes that a thread takes by itself
constexpr int kSmallNT = 128;
constexpr int kMany = 64;      // candidates that a few lanes rank
constexpr int kTop = 32;       // the most classes that are listed
constexpr int kFew = 9;        // candidates a lane of a group within a warp
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

// A thread per row over tiles of 32 rows, of which the next is copied through shared memory
// while one is worked on; bound by issue slots (333333 x 10 float32, the three best: 16 us, 1000
// instructions a row, a fifth of them the places). Every class's place is counted against every other, c (c - 1) / 2
// comparisons; the places name the classes in shared memory, from where the warp
// writes the tile's lists as they lie.
template <class T, class A, int CW>
struct SmallWarp {  // behind it: the warp's two tiles
    A off[kTileRows], ls[kTileRows];
    uint8_t order[kTileRows][CW];  // the classes in their order, kNone in a row without
};
constexpr unsigned kNone = 255;

template <class T, class A, int CW>
__host__ __device__ constexpr size_t small_bytes(int c) {
    return (sizeof(SmallWarp<T, A, CW>) + 15) / 16 * 16 + 2 * kTileRows * c * sizeof(T);
}

template <class T, class A, int CW>
__global__ void __launch_bounds__(kSmallNT, IsF64<A>::value || CW > 16 ? 4 : 8)
    small_kernel(const T* __restrict__ x, int64_t ld, Args<A> a, bool whole, unsigned by_top) {
    extern __shared__ uint4 small_smem[];
    const int c = (int)a.c, lane = threadIdx.x & 31, top = a.top;
    char* const mine = reinterpret_cast<char*>(small_smem) + (threadIdx.x / 32) * small_bytes<T, A, CW>(c);
    SmallWarp<T, A, CW>& w = *reinterpret_cast<SmallWarp<T, A, CW>*>(mine);
    T* const tiles = reinterpret_cast<T*>(mine + (sizeof(SmallWarp<T, A, CW>) + 15) / 16 * 16);
    const int64_t n_tiles = ceil_div(a.n, (int64_t)kTileRows), step = (int64_t)gridDim.x * (kSmallNT / 32);
    auto rows_of = [&](int64_t t0) { return (int)(a.n - t0 < kTileRows ? a.n - t0 : kTileRows); };
    int64_t i = (int64_t)blockIdx.x * (kSmallNT / 32) + threadIdx.x / 32;
    int y = -1;
    if (i < n_tiles) {
        tile_fetch(x, ld, i * kTileRows, rows_of(i * kTileRows), c, whole, tiles);
        if (lane < rows_of(i * kTileRows)) y = a.label(i * kTileRows + lane);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int buf = 0; i < n_tiles; i += step, buf ^= 1) {
        const int64_t t0 = i * kTileRows, t = t0 + lane, next = (i + step) * kTileRows;
        const int rows = rows_of(t0), y_now = y;
        const T* const tile = tiles + buf * (kTileRows * c);
        if (i + step < n_tiles) {
            tile_fetch(x, ld, next, rows_of(next), c, whole, tiles + (buf ^ 1) * (kTileRows * c));
            if (lane < rows_of(next)) y = a.label(next + lane);
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        if (lane < rows) {
            const T* row = tile + lane * c;
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
                const A z = v[j] - off, e = exp_of(z);
                s += e;
                d += e * floor_of(z);
            }
            const A xy = widen<A>(row[y_now < 0 ? 0 : y_now]);
            int rank = 0;
#pragma unroll
            for (int j = 0; j < CW; ++j) rank += j < c && (j < y_now ? v[j] >= xy : v[j] > xy) ? 1 : 0;
            const bool empty = m == minus_inf<A>() && s == A(0);
            const A ls = log_of(s);
            if (y_now < 0 || empty || s != s) {
                const A v0 = y_now >= 0 && !empty ? s : A(0);
                a.nothing(t, y_now < 0 ? A(0) : empty ? minus_inf<A>() : s, v0);
                w.off[lane] = v0;
                for (int j = 0; j < top; ++j) w.order[lane][j] = kNone;
            } else {
                a.lse[t] = off + ls;
                a.entropy[t] = entropy_of(ls, s, d);
                if (a.lp) a.lp[t] = (xy - off) - ls;
                if (a.ranks) a.id(a.ranks, t, rank);
                w.off[lane] = off;
                w.ls[lane] = ls;
                if (top) {
                    int place[CW];
#pragma unroll
                    for (int j = 0; j < CW; ++j) place[j] = 0;
#pragma unroll
                    for (int j = 1; j < CW; ++j)
#pragma unroll
                        for (int q = 0; q < j; ++q) {
                            const int up = v[j] > v[q] ? 1 : 0;
                            place[q] += up;
                            place[j] += 1 - up;
                        }
#pragma unroll
                    for (int j = 0; j < CW; ++j) w.order[lane][place[j]] = (uint8_t)j;  // padding comes last: below -infinity's ties
                }
            }
        }
        __syncwarp();
        for (int e = lane; e < rows * top; e += 32) {
            const int r = (int)(e * by_top >> 16), j = w.order[r][e - r * top];
            const int64_t to = t0 * top + e;
            if (a.ids64)
                static_cast<int64_t*>(a.top_ids)[to] = j == kNone ? -1 : j;
            else
                static_cast<int32_t*>(a.top_ids)[to] = j == kNone ? -1 : j;
            a.top_lp[to] = j == kNone ? w.off[r] : (widen<A>(tile[r * c + j]) - w.off[r]) - w.ls[r];
        }
        __syncwarp();  // the tile and the order are filled again
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ------------------------------------------------------------ longer rows --

// A row's, or a part of a row's, group of L threads within a block.
template <int L>
__device__ __forceinline__ void group_sync() {
    if (L <= 32)
        __syncwarp();
    else if (L == kNT)
        __syncthreads();
    else
        asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.x / L), "n"(L) : "memory");
}

// Sums of e = exp(v - off) and of e (v - off). In 32 bits as powers of two, two values an
// instruction, the second sum in units of log 2: 16-bit scores are otherwise bound by issue slots.
template <class A>
struct Terms {
    uint64_t s = 0, d = 0, minus_off;
    __device__ __forceinline__ explicit Terms(float off) : minus_off(pair_of(-off, -off)) {}
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N]) {
#pragma unroll
        for (int q = 0; q < N; q += 2) {
            float a, b, ea, eb;
            pair_to(pair_mul(pair_add(pair_of(v[q], v[q + 1]), minus_off), pair_of(1.4426950408889634f, 1.4426950408889634f)), a, b);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ea) : "f"(a));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(eb) : "f"(b));
            const uint64_t e = pair_of(ea, eb);
            s = pair_add(s, e);
            // an exponential of 0 times -infinity would be NaN; NaN is in e already
            asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(e), "l"(pair_of(fmaxf(a, -200.0f), fmaxf(b, -200.0f))));
        }
    }
    __device__ __forceinline__ void to(float& sum, float& moved) const {
        float a, b;
        pair_to(s, a, b);
        sum += a + b;
        pair_to(d, a, b);
        moved += (a + b) * 0.6931471805599453f;
    }
};
template <>
struct Terms<double> {
    double s = 0.0, d = 0.0, off;
    __device__ __forceinline__ explicit Terms(double o) : off(o) {}
    template <int N>
    __device__ __forceinline__ void add(const double (&v)[N]) {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const double z = v[q] - off, e = exp_of(z);
            s += e;
            d += e * floor_of(z);
        }
    }
    __device__ __forceinline__ void to(double& sum, double& moved) const {
        sum += s;
        moved += d;
    }
};

// Which of a vector's values are above `bound`, or (!STRICT) reach it: a bit each.
template <class T, bool STRICT>
struct Bits {
    template <class A>
    static __device__ __forceinline__ unsigned of(const uint4& r, A bound) {
        A p[Pack<T>::N];
        Pack<T>::unpack(r, p);
        unsigned bits = 0;
#pragma unroll
        for (int q = 0; q < Pack<T>::N; ++q) bits |= (STRICT ? p[q] > bound : p[q] >= bound) ? 1u << q : 0u;
        return bits;
    }
};
template <class P, bool STRICT>
__device__ __forceinline__ unsigned pair_bits(const uint4& r, P bound) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned m = STRICT ? __hgt2_mask(as_pair<P>(w[i]), bound) : __hge2_mask(as_pair<P>(w[i]), bound);
        bits |= m & (0x00020001u << (2 * i));
    }
    return (bits | bits >> 16) & 0xffu;
}
template <bool STRICT>
struct Bits<__nv_bfloat16, STRICT> {  // the bound is one of the values: exact in their type
    static __device__ __forceinline__ unsigned of(const uint4& r, float bound) {
        return pair_bits<__nv_bfloat162, STRICT>(r, __float2bfloat162_rn(bound));
    }
};
template <bool STRICT>
struct Bits<__half, STRICT> {
    static __device__ __forceinline__ unsigned of(const uint4& r, float bound) {
        return pair_bits<__half2, STRICT>(r, __float2half2_rn(bound));
    }
};

// How many of a row's values come before its label's: those above it, and of the ones
// equal to it those before its index, which are above the next lower value of the type. The
// vector that the label is in counts as one behind it; `fix` adds what that leaves out.
template <class T>
struct Before {
    T own, lower;     // lower: NaN below -infinity, where everything counts
    int y, vector;    // the label, which may lie outside the values that are looked at, and its vector;
                      // vectors from the last one on, which are -infinity, are behind it
    __device__ __forceinline__ Before(T xy, int label, const RowShape<T>& sh)
        : own(xy), lower(below(xy)), y(label), vector(label < sh.head ? -1 : min((label - sh.head) / RowShape<T>::V, sh.nv)) {}
    __device__ __forceinline__ T bound(int j) const { return j < vector ? lower : own; }
    static __device__ __forceinline__ float below(float v) {
        const int b = __float_as_int(v);
        return v == 0.0f ? __int_as_float((int)0x80000001) : v == minus_inf<float>() ? NAN : __int_as_float(v > 0.0f ? b - 1 : b + 1);
    }
    static __device__ __forceinline__ double below(double v) {
        const long long b = __double_as_longlong(v);
        return v == 0.0 ? __longlong_as_double((long long)0x8000000000000001ull)
                        : v == minus_inf<double>() ? (double)NAN : __longlong_as_double(v > 0.0 ? b - 1 : b + 1);
    }
    static __device__ __forceinline__ __nv_bfloat16 below(__nv_bfloat16 v) {
        const unsigned short b = __bfloat16_as_ushort(v);
        return __ushort_as_bfloat16((b & 0x7fff) == 0 ? 0x8001 : b == 0xff80 ? 0x7fff : b & 0x8000 ? b + 1 : b - 1);
    }
    static __device__ __forceinline__ __half below(__half v) {
        const unsigned short b = __half_as_ushort(v);
        return __ushort_as_half((b & 0x7fff) == 0 ? 0x8001 : b == 0xfc00 ? 0x7fff : b & 0x8000 ? b + 1 : b - 1);
    }
    template <class A>
    static __device__ __forceinline__ bool above(A v, A bound) { return !(v <= bound); }  // NaN: everything
    __device__ __forceinline__ int one(T v, int i) const {
        using A = typename Arith<T>::type;
        return above<A>(widen<A>(v), widen<A>(i < y ? lower : own)) ? 1 : 0;
    }
    // of the label's vector's values before the label that are equal to it, by one thread
    __device__ __forceinline__ int fix(const T* row, const RowShape<T>& sh) const {
        using A = typename Arith<T>::type;
        if (vector < 0 || vector >= sh.nv) return 0;
        const int first = sh.head + vector * RowShape<T>::V;
        const uint4 v = load16(row + first);
        const A own_wide = widen<A>(own);
        const unsigned equal = Bits<T, false>::of(v, own_wide) & ~Bits<T, true>::of(v, own_wide);
        return __popc(equal & ((1u << (y - first)) - 1));
    }
};
// Counts over a few vectors; total() at most once each 64 of them (16-bit counters hold 256).
template <class T>
struct Count {
    int n = 0;
    template <class A, int N>
    __device__ __forceinline__ void add(const uint4&, const A (&v)[N], T bound) {
        const A b = widen<A>(bound);
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (!(v[q] <= b)) ++n;
    }
    __device__ __forceinline__ int total() const { return n; }
};
template <class P, class T>
struct PairCount {
    P n;
    __device__ __forceinline__ void four(const uint4& r, P bound) {
        n = __hadd2(n, __hgtu2(as_pair<P>(r.x), bound));
        n = __hadd2(n, __hgtu2(as_pair<P>(r.y), bound));
        n = __hadd2(n, __hgtu2(as_pair<P>(r.z), bound));
        n = __hadd2(n, __hgtu2(as_pair<P>(r.w), bound));
    }
    __device__ __forceinline__ int total() const { return (int)(__low2float(n) + __high2float(n)); }
};
template <>
struct Count<__nv_bfloat16> : PairCount<__nv_bfloat162, __nv_bfloat16> {
    __device__ __forceinline__ Count() { n = __float2bfloat162_rn(0.0f); }
    template <int N>
    __device__ __forceinline__ void add(const uint4& r, const float (&)[N], __nv_bfloat16 bound) { four(r, __bfloat162bfloat162(bound)); }
};
template <>
struct Count<__half> : PairCount<__half2, __half> {
    __device__ __forceinline__ Count() { n = __float2half2_rn(0.0f); }
    template <int N>
    __device__ __forceinline__ void add(const uint4& r, const float (&)[N], __half bound) { four(r, __half2half2(bound)); }
};

// The largest of a few vectors' values: in 16 bits two at a time up to the last step.
template <class T, class A, int U>
__device__ __forceinline__ A top_of(const uint4 (&v)[U]) {
    A best = Pack<T>::top(v[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) best = fmax(best, Pack<T>::top(v[u]));
    return best;
}
template <class P, int U>
__device__ __forceinline__ float top_of_pairs(const uint4 (&v)[U]) {
    P m = as_pair<P>(v[0].x);
#pragma unroll
    for (int u = 0; u < U; ++u)
        m = __hmax2(__hmax2(__hmax2(m, as_pair<P>(v[u].x)), __hmax2(as_pair<P>(v[u].y), as_pair<P>(v[u].z))), as_pair<P>(v[u].w));
    return fmaxf(__low2float(m), __high2float(m));
}
template <>
__device__ __forceinline__ float top_of<__nv_bfloat16, float, 8>(const uint4 (&v)[8]) { return top_of_pairs<__nv_bfloat162>(v); }
template <>
__device__ __forceinline__ float top_of<__half, float, 8>(const uint4 (&v)[8]) { return top_of_pairs<__half2>(v); }

// A value with its index, as a number that grows in the order of the classes. In 32 bits one word: the
// value's bits in the order of values above the complement of the index.
template <class A>
struct Key;
template <>
struct Key<float> {
    uint64_t k;
    Key() = default;
    __device__ __forceinline__ Key(float v, int i) {
        const int b = __float_as_int(v + 0.0f);  // -0 is 0
        k = (uint64_t)(unsigned)(b ^ (b >> 31 | (int)0x80000000)) << 32 | (unsigned)~i;
    }
    static __device__ __forceinline__ Key none() {
        Key r;
        r.k = 0;
        return r;
    }
    __device__ __forceinline__ bool before(const Key& o) const { return k > o.k; }
    __device__ __forceinline__ bool is_none() const { return k == 0; }
    __device__ __forceinline__ float value() const {
        const int b = (int)(k >> 32);
        return __int_as_float(b ^ (~(b >> 31) | (int)0x80000000));
    }
    __device__ __forceinline__ int index() const { return (int)~(unsigned)k; }
    __device__ __forceinline__ void move(int by) { k -= by; }  // the index goes up
    __device__ __forceinline__ Key across(int lanes) const {
        Key r;
        r.k = __shfl_xor_sync(0xffffffffu, k, lanes);
        return r;
    }
};
template <>
struct Key<double> {
    double v;
    int64_t i;
    Key() = default;
    __device__ __forceinline__ Key(double value, int index) : v(value), i(index) {}
    static __device__ __forceinline__ Key none() {
        Key r;
        r.v = minus_inf<double>();
        r.i = INT64_MAX;
        return r;
    }
    __device__ __forceinline__ bool before(const Key& o) const { return v > o.v || (v == o.v && i < o.i); }
    __device__ __forceinline__ bool is_none() const { return i == INT64_MAX; }
    __device__ __forceinline__ double value() const { return v; }
    __device__ __forceinline__ int index() const { return (int)i; }
    __device__ __forceinline__ void move(int by) {
        if (!is_none()) i += by;
    }
    __device__ __forceinline__ Key across(int lanes) const {
        Key r;
        r.v = __shfl_xor_sync(0xffffffffu, v, lanes);
        r.i = __shfl_xor_sync(0xffffffffu, i, lanes);
        return r;
    }
};
// The same of a 16-bit value of a row of at most 2^16, in half the bits.
template <class T>
struct ShortKey {
    unsigned k;
    ShortKey() = default;
    __device__ __forceinline__ ShortKey(float v, int i) {
        const T t = narrow<T>(v + 0.0f);  // -0 is 0; exact
        const unsigned b = *reinterpret_cast<const unsigned short*>(&t);
        k = (b & 0x8000u ? ~b << 16 : (b | 0x8000u) << 16) | (0xffffu - (unsigned)i);
    }
    static __device__ __forceinline__ ShortKey none() {
        ShortKey r;
        r.k = 0;
        return r;
    }
    __device__ __forceinline__ bool before(const ShortKey& o) const { return k > o.k; }
    __device__ __forceinline__ float value() const {
        const unsigned h = k >> 16;
        const unsigned short b = (unsigned short)(h & 0x8000u ? h & 0x7fffu : ~h);
        return widen<float>(*reinterpret_cast<const T*>(&b));
    }
    __device__ __forceinline__ int index() const { return (int)(0xffffu - (k & 0xffffu)); }
    __device__ __forceinline__ ShortKey across(int lanes) const {
        ShortKey r;
        r.k = __shfl_xor_sync(0xffffffffu, k, lanes);
        return r;
    }
};

// How many of the keys of a list come before `me`: `n` of them, and up to kPad that are none behind
// them, so that whole vectors can be read.
constexpr int kPad = 4;
template <class KT>
__device__ __forceinline__ int place_of(const KT* keys, int n, const KT& me) {
    int place = 0;
    if constexpr (sizeof(KT) == 4) {
        for (int o = 0; o < n; o += 4) {
            const uint4 k = *reinterpret_cast<const uint4*>(keys + o);
            place += (k.x > me.k ? 1 : 0) + (k.y > me.k ? 1 : 0) + (k.z > me.k ? 1 : 0) + (k.w > me.k ? 1 : 0);
        }
    } else if constexpr (sizeof(KT) == 8) {
        for (int o = 0; o < n; o += 4) {
            const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(keys + o), b = *reinterpret_cast<const ulonglong2*>(keys + o + 2);
            place += (a.x > me.k ? 1 : 0) + (a.y > me.k ? 1 : 0) + (b.x > me.k ? 1 : 0) + (b.y > me.k ? 1 : 0);
        }
    } else {
        for (int o = 0; o < n; ++o) place += keys[o].before(me) ? 1 : 0;
    }
    return place;
}

constexpr int kSegments = 16;  // of a thread's vectors, each with its largest value

// What a group shares.
template <class KT, int CAP>
struct Lists {
    alignas(16) KT cand[CAP + kPad];
    KT best[kTop];  // the answer
    int count, listed;
};
template <class A, int L>
struct Shared : Lists<Key<A>, kCand> {
    A m[L / 32], s[L / 32], d[L / 32];
    A one[L / 32], every[L / 32];
    int rank[L / 32];
    A most[kSegments][L];  // of each of a thread's segments
};

// The values of each group of L lanes in falling order.
template <class A, int L = 32>
__device__ __forceinline__ A sorted_lanes(A v) {
    const int lane = threadIdx.x % L;
#pragma unroll
    for (int k = 2; k <= L; k *= 2)
#pragma unroll
        for (int j = k / 2; j > 0; j /= 2) {
            const A o = __shfl_xor_sync(0xffffffffu, v, j);
            const bool first = (lane & j) == 0, falling = (lane & k) == 0;
            v = first == falling ? fmax(v, o) : fmin(v, o);
        }
    return v;
}

// Values that at least a and b of the 32 lanes' values reach (b <= a): the a-th and b-th
// largest, or below. Few of them by so many maxima of the warp (of distinct values: what is
// found may be lower), more by sorting.
__device__ __forceinline__ void reached(float v, int a, int b, float& at_a, float& at_b) {
    if (a <= 8) {
        const int bits = __float_as_int(v);
        unsigned u = (unsigned)(bits ^ (bits >> 31 | (int)0x80000000));
        for (int i = 1;; ++i) {
            const unsigned top = __reduce_max_sync(0xffffffffu, u);
            const int back = (int)top < 0 ? (int)(top & 0x7fffffffu) : (int)~top;
            at_a = top ? __int_as_float(back) : minus_inf<float>();  // 0: every lane has been passed
            if (i == b) at_b = at_a;
            if (i == a) return;
            if (u == top) u = 0;
        }
    }
    v = sorted_lanes(v);
    at_a = __shfl_sync(0xffffffffu, v, a - 1);
    at_b = __shfl_sync(0xffffffffu, v, b - 1);
}
__device__ __forceinline__ void reached(double v, int a, int b, double& at_a, double& at_b) {
    v = sorted_lanes(v);
    at_a = __shfl_sync(0xffffffffu, v, a - 1);
    at_b = __shfl_sync(0xffffffffu, v, b - 1);
}
// The same of each group of L lanes.
template <class A, int L>
__device__ __forceinline__ A reached_in_group(A v, int a) {
    A at;
    if constexpr (L == 32)
        reached(v, a, a, at, at);
    else
        at = __shfl_sync(0xffffffffu, sorted_lanes<A, L>(v), a - 1, L);
    return at;
}

// What k <= kTop of a group's 2 L values reach, two a lane: the k-th largest, which is the least of
// the larger ones of the i-th of the one half and the (k - 1 - i)-th of the other.
template <class A, int L>
__device__ __forceinline__ A reached_of_two(A a, A b, int k) {
    const int lane = threadIdx.x % L, j = k - 1 - lane;
    a = sorted_lanes<A, L>(a);
    b = sorted_lanes<A, L>(b);
    const A other = __shfl_sync(0xffffffffu, b, j & (L - 1), L);
    A least = j < 0 ? (A)INFINITY : j < L ? fmax(a, other) : a;
    if (L < 32) {
        const A behind = __shfl_sync(0xffffffffu, b, (k - 1 - L) & (L - 1), L);  // beside none of the one half
        if (k > L) least = fmin(least, behind);
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) least = fmin(least, __shfl_xor_sync(0xffffffffu, least, o));
    return least;
}

// The vectors of a row of c values of which it has at least so many, wherever it begins.
template <int V>
__host__ __device__ constexpr int fewest_vectors(int64_t c) {
    return (int)(c - (V - 1)) / V;
}

// The least value of the type above v.
template <class T>
__device__ __forceinline__ float above(float v) {
    if constexpr (sizeof(T) == 4) {
        const int b = __float_as_int(v);
        return v == 0.0f ? __int_as_float(1) : __int_as_float(b < 0 ? b - 1 : b + 1);
    } else {
        const T t = narrow<T>(v);
        const unsigned short b = *reinterpret_cast<const unsigned short*>(&t);
        const unsigned short up = v == 0.0f ? 1 : b & 0x8000 ? b - 1 : b + 1;
        return widen<float>(*reinterpret_cast<const T*>(&up));
    }
}
template <class T>
__device__ __forceinline__ double above(double v) {
    const long long b = __double_as_longlong(v);
    return v == 0.0 ? __longlong_as_double(1) : __longlong_as_double(b < 0 ? b - 1 : b + 1);
}

// The k-th largest of a warp's values, N and one more a lane, by its bits from the highest on:
// for rows of few vectors beside the places that are asked for, where the lanes' largest say
// little. BITS: the upper bits in which the values differ.
template <int BITS, int N>
__device__ __forceinline__ float kth_of_warp(const float (&v)[N], float one, int k) {
    unsigned u = 0;
    for (int b = 31; b > 31 - BITS; --b) {
        const unsigned with = u | 1u << b;
        const float f = __int_as_float((int)with < 0 ? (int)(with & 0x7fffffffu) : (int)~with);  // NaN: reached by none
        int count = one >= f ? 1 : 0;
#pragma unroll
        for (int q = 0; q < N; ++q) count += v[q] >= f ? 1 : 0;
        if (__reduce_add_sync(0xffffffffu, count) >= k) u = with;
    }
    if (u < 0x00800000u) return minus_inf<float>();
    if ((int)u >= 0) u |= (unsigned)((1ull << (32 - BITS)) - 1);  // a negative value's lower bits are 0 in itself
    return __int_as_float((int)u < 0 ? (int)(u & 0x7fffffffu) : (int)~u);
}

// The first `want` values of the row that equal v, in index order, by one warp.
template <class T, class A, class KT>
__device__ __noinline__ void first_equal(const T* row, int c, A v, int want, KT* to) {
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
                if (before < want) to[before] = KT(v, (int)(j0 + lane * 8 + q));
                ++before;
            }
        found += all;
    }
}

// The first `top` values one at a time, each the first behind the one before, by a group: for
// rows of which a few threads hold most of the large values.
template <class T, class A, int L, class KT>
__device__ __noinline__ void one_by_one(const T* row, int c, int top, KT* parts, KT* to) {
    const int lane = threadIdx.x % L;
    KT last;
    for (int place = 0; place < top; ++place) {
        KT best = KT::none();
        for (int64_t j = lane; j < c; j += L) {
            const KT o(widen<A>(row[j]), (int)j);
            if ((place == 0 || last.before(o)) && o.before(best)) best = o;
        }
#pragma unroll
        for (int s = min(L, 32) / 2; s > 0; s >>= 1) {
            const KT o = best.across(s);
            if (o.before(best)) best = o;
        }
        if (L > 32) {
            group_sync<L>();
            if ((lane & 31) == 0) parts[lane / 32] = best;
            group_sync<L>();
            for (int w = 0; w < L / 32; ++w)
                if (parts[w].before(best)) best = parts[w];
        }
        last = best;
        if (lane == 0) to[place] = best;
    }
}

// The places of a group's candidates among each other: the first `top` to g.best. A warp sorts
// short keys that its lanes hold; others are counted against each other, n comparisons a key
// (200000 x 1003 float16, 32 best of which 110 candidates: 1085 us with 64-bit keys, 795 with short).
template <int L, class KT, int CAP>
__device__ __forceinline__ void places(Lists<KT, CAP>& g, int count, int top) {
    const int lane = threadIdx.x % L;
    if constexpr (L == 32 && sizeof(KT) == 4) {
        if (count <= 32) {
            unsigned k = lane < count ? g.cand[lane].k : 0;
            auto stage = [&](int size) {
#pragma unroll
                for (int j = size / 2; j > 0; j /= 2) {
                    const unsigned o = __shfl_xor_sync(0xffffffffu, k, j);
                    k = ((lane & j) == 0) == ((lane & size) == 0) ? max(k, o) : min(k, o);
                }
            };
            stage(2);
            stage(4);
            stage(8);
            if (count > 8) stage(16);
            if (count > 16) stage(32);
            if (lane < min(top, count)) g.best[lane].k = k;
            return;
        }
    }
    for (int j = lane; j < kPad; j += L) g.cand[count + j] = KT::none();
    group_sync<L>();
    for (int q = lane; q < count; q += L) {
        const KT me = g.cand[q];
        const int place = place_of(g.cand, count, me);
        if (place < top) g.best[place] = me;
    }
}

// The first `top` of a row's c values in their order to g.best, by the group. `bound`: what at
// least `top` of them reach. `walk(strict)` lists the values that reach it (strict: that are above it) as
// candidates and says how many there are, or, where that is more than fit, that it is.
template <class T, class A, int L, class KT, class W>
__device__ __forceinline__ void choose(Lists<KT, kCand>& g, const T* row, int c, int top, A bound, W&& walk) {
    if (bound != minus_inf<A>()) {
        const int count = walk(std::false_type{});
        if (count <= kCand) {
            places<L>(g, count, top);
            return;
        }
    }
    // Too many reach it: mostly ties, as of masked classes. Those above it, and the first
    // of those that are equal.
    const int count = walk(std::true_type{});
    if (count <= kCand) {
        places<L>(g, count, top);
        if (count < top && threadIdx.x % L < 32) first_equal(row, c, bound, top - count, g.best + count);
        return;
    }
    one_by_one<T, A, L>(row, c, top, g.cand, g.best);
}

// What a row's finished statistics say, by one thread; false where there is no more to say.
template <class A>
__device__ __forceinline__ bool finish(const Args<A>& a, int64_t t, A xy, const Stats<A>& r, int rank, A& off, A& ls, bool write) {
    off = offset_of(r.m);
    ls = log_of(r.s);
    const bool empty = r.m == minus_inf<A>() && r.s == A(0);
    if (empty || r.s != r.s) {
        if (write) a.nothing(t, empty ? minus_inf<A>() : r.s, empty ? A(0) : r.s);
        return false;
    }
    if (write) {
        if (a.lp) a.lp[t] = (xy - off) - ls;
        a.lse[t] = off + ls;
        a.entropy[t] = entropy_of(ls, r.s, r.d);
        if (a.ranks) a.id(a.ranks, t, rank);
    }
    return true;
}

// Rows of up to L K vectors: L lanes each, the row in their registers. Bound by issue slots, most of
// them what a row costs its warp once: 200000 x 1003 float16 131, 208, 258 us without, with 5 and
// with 16 best by a warp a row, 107, 172, 229 by half a warp (401 MB: 61 us). The row behind one
// prefetched by persistent warps: 148, 235, 296 us instead of 131, 208, 258, for a block an SM less.
template <class T, class A, int L, int K>
__global__ void __launch_bounds__(kNT, IsF64<A>::value ? 2 : K > 4 ? 3 : 4)
    held_kernel(const T* __restrict__ x, int64_t ld, Args<A> a) {
    constexpr int V = 16 / sizeof(T), E = (2 * (V - 1) + L - 1) / L;
    constexpr int ALL = L * K * V + 2 * (V - 1), CAP = ALL < kFew * L ? ALL : kFew * L;  // values, candidates
    static_assert(kFew * 32 == kCand, "a warp's list is that of the longer rows");
    static_assert(K * V <= 64, "a bit a value");
    using KT = std::conditional_t<sizeof(T) == 2, ShortKey<T>, Key<A>>;
    __shared__ Lists<KT, CAP> shared[kNT / L];
    Lists<KT, CAP>& g = shared[threadIdx.x / L];
    const int lane = threadIdx.x % L, top = a.top;
    const int64_t t = (int64_t)blockIdx.x * (kNT / L) + threadIdx.x / L;
    const int y = t < a.n ? a.label(t) : -1;
    if (t < a.n && y < 0) {
        if (lane == 0) a.nothing(t, A(0), A(0));
        for (int j = lane; j < top; j += L) a.no_class(t, j, A(0));
    }
    if (L == 32 ? y < 0 : __all_sync(0xffffffffu, y < 0)) return;  // the whole warp
    const bool in = y >= 0;
    const T* row = x + (in ? t : 0) * ld;
    const RowShape<T> sh(row, in ? (int)a.c : 0);
    uint4 v[K];
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] = lane + i * L < sh.nv ? load16(row + sh.head + (lane + i * L) * V) : Pack<T>::minus_inf();
    const T low = narrow<T>(minus_inf<A>());
    T last[E];
    A mine = minus_inf<A>();
#pragma unroll
    for (int i = 0; i < E; ++i) {
        last[i] = lane + i * L < sh.edges ? row[sh.edge(lane + i * L)] : low;
        mine = fmax(mine, widen<A>(last[i]));
    }
    const Before<T> before(row[in ? y : 0], y, sh);
#pragma unroll
    for (int i = 0; i < K; ++i) mine = fmax(mine, Pack<T>::top(v[i]));
    Stats<A> r{mine, A(0), A(0)};
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) r.m = fmax(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
    A off = offset_of(r.m), ls;
    Terms<A> terms(off);
    Count<T> counted;
    int rank = lane == 0 ? before.fix(row, sh) : 0;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        A p[V];
        Pack<T>::unpack(v[i], p);
        terms.add(p);
        counted.add(v[i], p, before.bound(lane + i * L));
    }
    terms.to(r.s, r.d);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const A z = widen<A>(last[i]) - off, e = exp_of(z);
        r.s += e;
        r.d += e * floor_of(z);
        if (lane + i * L < sh.edges) rank += before.one(last[i], sh.edge(lane + i * L));
    }
    rank += counted.total();
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
        r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
        r.d += __shfl_xor_sync(0xffffffffu, r.d, o);
        rank += __shfl_xor_sync(0xffffffffu, rank, o);
    }
    const bool go = in && finish(a, t, widen<A>(before.own), r, rank, off, ls, lane == 0);
    if (in && !go)
        for (int j = lane; j < top; j += L) a.no_class(t, j, r.s != r.s ? r.s : A(0));
    if (top == 0 || (L == 32 ? !go : __all_sync(0xffffffffu, !go))) return;
    // Of the largest values of the lanes (up to half as many places as lanes), or of two a lane: with
    // as many places as lanes one a lane reaches far down (200000 x 1003 float16, 32 best: 795 us by
    // one, 331 by two; 16 best: 257 and 266). Where the row may have fewer than that, or hardly more,
    // by bits in a warp (400000 x 128 bfloat16, 32 best: 650 us, by two a lane 850), and in fewer lanes not
    // at all: its values are few enough to be listed. The warp's rows go one way, whose vectors may
    // differ by one: `fewest` of them.
    A bound = minus_inf<A>();
    const int fewest = fewest_vectors<V>(a.c);
    if (L == 32 && K > 1 ? top <= 16 : L < 32 && top <= L / 2 && top <= fewest) {
        bound = reached_in_group<A, L>(mine, top);
    } else if (L == 32 && K > 1 || top <= (L < 32 ? 2 * min(fewest, L) : fewest * 3 / 2)) {
        A first = minus_inf<A>(), second = minus_inf<A>();
#pragma unroll
        for (int i = 0; i < K; ++i) {
            if constexpr (L == 32 && K > 1) {
                if (i < K / 2)
                    first = fmax(first, Pack<T>::top(v[i]));
                else
                    second = fmax(second, Pack<T>::top(v[i]));
            } else {
                first = fmax(first, Pack<T>::top(make_uint4(v[i].x, v[i].y, v[i].x, v[i].y)));
                second = fmax(second, Pack<T>::top(make_uint4(v[i].z, v[i].w, v[i].z, v[i].w)));
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) second = fmax(second, widen<A>(last[i]));
        bound = reached_of_two<A, L>(first, second, top);
    } else if constexpr (L == 32 && K == 1 && !IsF64<A>::value) {
        A p[V];
        Pack<T>::unpack(v[0], p);
        bound = kth_of_warp<sizeof(T) == 4 ? 32 : 19>(p, widen<A>(last[0]), top);
    }
    // A bit for each value that is listed; then they are taken one a lane at a time.
    auto walk = [&](auto strict) {
        constexpr bool S = decltype(strict)::value;
        const unsigned group = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1) << (threadIdx.x & 31 & ~(L - 1));
        const unsigned before_me = group & ((1u << (threadIdx.x & 31)) - 1);
        uint64_t bits = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) bits |= (uint64_t)Bits<T, S>::of(v[i], bound) << (i * V);
        int count = 0;
        if (!go) bits = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const A e = widen<A>(last[i]);
            const bool hit = go && lane + i * L < sh.edges && (S ? e > bound : e >= bound);
            const unsigned hits = __ballot_sync(0xffffffffu, hit) & group;
            if (hit) g.cand[count + __popc(hits & before_me)] = KT(e, sh.edge(lane + i * L));
            count += __popc(hits);
        }
        for (;;) {
            const unsigned all = __ballot_sync(0xffffffffu, bits != 0 && count <= CAP), hits = all & group;
            if (all == 0) break;
            if (hits >> (threadIdx.x & 31) & 1) {
                const int q = __ffsll((long long)bits) - 1, i = sh.head + (lane + q / V * L) * V + q % V;
                const int to = count + __popc(hits & before_me);
                if (to < CAP) g.cand[to] = KT(widen<A>(row[i]), i);
                bits &= bits - 1;
            }
            count += __popc(hits);
        }
        __syncwarp();
        return count;
    };
    if constexpr (L < 32 || CAP == ALL) {
        // Where many reach the bound (ties), and where it is -infinity, those above it are listed,
        // and the first of its equals; where these do not fit, one is found at a time.
        const A equal = bound;
        bool over = bound == minus_inf<A>();
        if (over) bound = above<T>(bound);
        int count = walk(std::false_type{});
        const bool many = !over && count > min(kMany, CAP);
        if (__any_sync(0xffffffffu, many)) {
            if (many) bound = above<T>(bound);
            over |= many;
            count = walk(std::false_type{});
        }
        places<L>(g, min(count, CAP), top);
        if constexpr (CAP < ALL) {
            const bool beyond = go && count > CAP;
            if (__any_sync(0xffffffffu, beyond)) {
                __syncwarp();
                one_by_one<T, A, L>(row, (int)a.c, top, g.cand, beyond ? g.best : g.cand);
            }
        }
        const int more = go && over && count < top ? top - count : 0;
        if (__any_sync(0xffffffffu, more > 0))
            for (int o = 0; o < 32; o += L) {
                const int want = __shfl_sync(0xffffffffu, more, o), from = __shfl_sync(0xffffffffu, count, o);
                const A v = __shfl_sync(0xffffffffu, equal, o);
                const int64_t of = __shfl_sync(0xffffffffu, t, o);
                if (want > 0)
                    first_equal(x + of * ld, (int)a.c, v, want, shared[threadIdx.x / 32 * (32 / L) + o / L].best + from);
            }
    } else {
        choose<T, A, L>(g, row, (int)a.c, top, bound, walk);
    }
    __syncwarp();
    if (go)
        for (int j = lane; j < top; j += L) {
            a.id(a.top_ids, t * top + j, g.best[j].index());
            a.top_lp[t * top + j] = (g.best[j].value() - off) - ls;
        }
}

// Longer rows, read once with a running maximum: L threads a row, or a cluster of CL blocks
// of L threads where rows are few, each block on a part of the row and the first one on
// what the others found, in distributed shared memory. A row's own work (reductions, the
// bound, the candidates) costs each of its warps several hundred instructions, so short rows
// take few lanes. 32, 64, 128, 256 lanes a row, the five best of bf16 rows: 30000 x 5000 92, 131,
// 172, 329 us; 8195 x 32000 119, 116, 121, 142; 4096 x 65536 117, 115, 112, 117; 300 x 65536
// 45, 27, 23, 23.
template <class T, class A, int L, int CL>
__global__ void __launch_bounds__(kNT, IsF64<A>::value ? 2 : 4)
    scan_kernel(const T* __restrict__ x, int64_t ld, Args<A> a) {
    constexpr int V = 16 / sizeof(T), U = 8, W = L / 32;
    using G = Shared<A, L>;
    extern __shared__ uint4 rows_smem[];
    G& g = reinterpret_cast<G*>(rows_smem)[threadIdx.x / L];
    const int lane = threadIdx.x % L, warp = lane / 32, top = a.top;
    const int64_t t = CL > 1 ? blockIdx.x / CL : (int64_t)blockIdx.x * (kNT / L) + threadIdx.x / L;
    if (t >= a.n) return;  // the whole group, the whole cluster
    const int y_row = a.label(t);
    if (y_row < 0) {
        const bool first = CL == 1 || blockIdx.x % CL == 0;
        if (first && lane == 0) a.nothing(t, A(0), A(0));
        if (first && lane < top) a.no_class(t, lane, A(0));
        return;
    }
    // this block's part of the row: columns [begin, begin + c)
    int begin = 0, c = (int)a.c;
    if (CL > 1) {
        const int64_t share = ceil_div(a.c, (int64_t)CL * 64) * 64, part = blockIdx.x % CL;
        begin = (int)min(part * share, a.c);
        c = (int)(min((part + 1) * share, a.c) - begin);
    }
    const T* row = x + t * ld + begin;
    const RowShape<T> sh(row, c);
    const T xy = x[t * ld + y_row];
    const Before<T> before(xy, y_row - begin, sh);
    const T last = lane < sh.edges ? row[sh.edge(lane)] : narrow<T>(minus_inf<A>());
    const A edge = widen<A>(last);
    const int per = (sh.nv + L * U * kSegments - 1) / (L * U * kSegments);  // batches a segment
    int rank = lane < sh.edges ? before.one(last, sh.edge(lane)) : 0;
    if (lane == 0) rank += before.fix(row, sh);
    Stats<A> r{edge, A(0), A(0)};
    r.s = exp_of(edge - offset_of(edge));  // 1, 0 for -infinity, NaN
    A part_most = minus_inf<A>();
    int in_part = 0, segment = 0;
    // U vectors a thread; `full`: there are as many
    auto batch = [&](int j0, auto full) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] = decltype(full)::value || j0 + u * L < sh.nv ? load16(row + sh.head + (int64_t)(j0 + u * L) * V) : Pack<T>::minus_inf();
        const A best = top_of<T, A>(v);
        if (top) {
            part_most = fmax(part_most, best);
            if (++in_part == per || j0 - lane + L * U >= sh.nv) {
                g.most[segment++][lane] = part_most;
                part_most = minus_inf<A>();
                in_part = 0;
            }
        }
        if (best > r.m) r.raise(best);
        Terms<A> terms(offset_of(r.m));
        Count<T> counted;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            A p[V];
            Pack<T>::unpack(v[u], p);
            terms.add(p);
            counted.add(v[u], p, before.bound(j0 + u * L));
        }
        terms.to(r.s, r.d);
        rank += counted.total();
    };
    int j0 = lane;
    for (; j0 - lane + L * U <= sh.nv; j0 += L * U) batch(j0, std::true_type{});
    if (j0 - lane < sh.nv) batch(j0, std::false_type{});
    const A mine = r.m;
    join(r, 32);
    rank = __reduce_add_sync(0xffffffffu, rank);
    if (top) {
        // what ceil(top / W) threads of every warp reach, top values of the row do; and what
        // top threads of one warp do
        A one, every;
        reached(mine, top, (top + W - 1) / W, one, every);
        if ((lane & 31) == 0) {
            g.one[warp] = one;
            g.every[warp] = every;
        }
    }
    if ((lane & 31) == 0) {
        g.m[warp] = r.m;
        g.s[warp] = r.s;
        g.d[warp] = r.d;
        g.rank[warp] = rank;
    }
    if (lane == 0) g.count = 0;
    if (CL > 1 && lane < kTop) g.best[lane] = Key<A>::none();
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
    A off, ls;
    if (CL == 1 && !finish(a, t, widen<A>(xy), r, rank, off, ls, lane == 0)) {
        if (lane < top) a.no_class(t, lane, r.s != r.s ? r.s : A(0));
        return;
    }
    // a part with a NaN or without a value has no order, and none is asked for
    if (top && r.s == r.s && c > 0) {
        A one = g.one[0], every = g.every[0];
#pragma unroll
        for (int w = 1; w < W; ++w) {
            one = fmax(one, g.one[w]);
            every = fmin(every, g.every[w]);
        }
        const A bound = fmax(one, every);
        const int wanted = CL > 1 && c < top ? c : top;
        // A segment of a thread's whose largest reaches the bound is read again by eight lanes,
        // a vector each, four of them at a time.
        choose<T, A, L>(g, row, c, wanted, bound, [&](auto strict) {
            constexpr bool S = decltype(strict)::value;
            auto reaches = [&](A v) { return S ? v > bound : v >= bound; };
            auto take = [&](A v, int i) {
                const int at = atomicAdd(&g.count, 1);
                if (at < kCand) g.cand[at] = Key<A>(v, i);
            };
            if (lane < sh.edges && reaches(edge)) take(edge, sh.edge(lane));
            for (int s = 0; __any_sync(0xffffffffu, reaches(mine)) && s * per * L * U < sh.nv; ++s) {
                unsigned hits = __ballot_sync(0xffffffffu, reaches(g.most[s][lane]));
                while (hits && __all_sync(0xffffffffu, *(volatile int*)&g.count <= kCand)) {
                    int owner = -1;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if ((lane & 31) / 8 == q && hits) owner = __ffs(hits) - 1;
                        hits &= hits - 1;
                    }
                    for (int b = s * per; b < (s + 1) * per; ++b) {
                        const int j = (b * U + (lane & 7)) * L + warp * 32 + owner;
                        if (owner < 0 || j >= sh.nv) continue;
                        for (unsigned bits = Bits<T, S>::of(load16(row + sh.head + (int64_t)j * V), bound); bits; bits &= bits - 1) {
                            const int i = sh.head + j * V + __ffs((int)bits) - 1;
                            take(widen<A>(row[i]), i);
                        }
                    }
                }
            }
            group_sync<L>();
            const int count = g.count;
            group_sync<L>();
            if (lane == 0) g.count = 0;  // for a second walk, which begins behind the next barrier
            if (!S) group_sync<L>();
            return count;
        });
        group_sync<L>();
    }
    if constexpr (CL > 1) {
        namespace cg = cooperative_groups;
        auto cluster = cg::this_cluster();
        if (lane == 0) {
            g.m[0] = r.m;
            g.s[0] = r.s;
            g.d[0] = r.d;
            g.rank[0] = rank;
            g.listed = begin;
        }
        cluster.sync();
        if (cluster.block_rank() == 0) {
            // the parts' statistics, one a lane of each warp, and their candidates
            G* other = cluster.map_shared_rank(&g, (lane & 31) % CL);
            const bool in = (lane & 31) < CL;
            r.m = in ? other->m[0] : minus_inf<A>();
            r.s = in ? other->s[0] : A(0);
            r.d = in ? other->d[0] : A(0);
            rank = __reduce_add_sync(0xffffffffu, in ? other->rank[0] : 0);
            join(r, 32);
            const bool go = finish(a, t, widen<A>(xy), r, rank, off, ls, lane == 0);
            if (!go && lane < top) a.no_class(t, lane, r.s != r.s ? r.s : A(0));
            if (go && top) {
                const int count = top * CL;
                for (int q = lane; q < count; q += L) {
                    const G* o = cluster.map_shared_rank(&g, q / top);
                    Key<A> k = o->best[q % top];
                    if (!k.is_none()) k.move(o->listed);
                    g.cand[q] = k;
                }
                group_sync<L>();
                for (int q = lane; q < count; q += L) {
                    const Key<A> me = g.cand[q];
                    const int place = place_of(g.cand, count, me);  // eight times as many: whole vectors
                    if (place < top && !me.is_none()) {
                        a.id(a.top_ids, t * top + place, me.index());
                        a.top_lp[t * top + place] = (me.value() - off) - ls;
                    }
                }
            }
        }
        cluster.sync();  // the others' shared memory is read until here
    } else if (lane < top) {
        a.id(a.top_ids, t * top + lane, g.best[lane].index());
        a.top_lp[t * top + lane] = (g.best[lane].value() - off) - ls;
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

// A row's gradient by p alone: -p (sum + gh (x - lse + h)).
template <class A>
struct Slope {
    A l, whole, gh;  // whole = sum + gh h
    __device__ __forceinline__ A of(A v) const {
        const A z = v - l;
        return -exp_of(z) * (whole + gh * floor_of(z));
    }
    template <int N>
    __device__ __forceinline__ void all(double (&v)[N]) const {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = of(v[q]);
    }
    // two at a time, the difference in units of log 2
    template <int N>
    __device__ __forceinline__ void all(float (&v)[N]) const {
        const uint64_t ml = pair_of(-l, -l), w = pair_of(-whole, -whole), k = pair_of(gh * -0.6931471805599453f, gh * -0.6931471805599453f);
#pragma unroll
        for (int q = 0; q < N; q += 2) {
            float a, b, ea, eb;
            pair_to(pair_mul(pair_add(pair_of(v[q], v[q + 1]), ml), pair_of(1.4426950408889634f, 1.4426950408889634f)), a, b);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ea) : "f"(a));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(eb) : "f"(b));
            uint64_t t;
            asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t) : "l"(pair_of(fmaxf(a, -200.0f), fmaxf(b, -200.0f))), "l"(k), "l"(w));
            pair_to(pair_mul(pair_of(ea, eb), t), v[q], v[q + 1]);
        }
    }
};

// Few classes: a thread per row as in small_kernel, the gradient written in its row's place
// (333333 x 10 float32: 12 us, 520 instructions a row).
template <class T, class A, int CW>
__global__ void __launch_bounds__(kSmallNT, IsF64<A>::value || CW > 16 ? 4 : 8)
    small_grad_kernel(const T* __restrict__ x, int64_t ld, T* __restrict__ out, int64_t ld_out, GradArgs<A> a,
                      bool whole_in, bool whole_out) {
    extern __shared__ uint4 small_smem[];
    const int c = (int)a.c, lane = threadIdx.x & 31;
    T* const tiles = reinterpret_cast<T*>(small_smem) + (threadIdx.x / 32) * (2 * kTileRows * c);
    const int64_t n_tiles = ceil_div(a.n, (int64_t)kTileRows), step = (int64_t)gridDim.x * (kSmallNT / 32);
    // from the last row to the first: the forward left the last ones in L2
    auto begin = [&](int64_t i) { return (n_tiles - 1 - i) * kTileRows; };
    auto rows_of = [&](int64_t t0) { return (int)(a.n - t0 < kTileRows ? a.n - t0 : kTileRows); };
    int64_t i = (int64_t)blockIdx.x * (kSmallNT / 32) + threadIdx.x / 32;
    int y = -1;
    A l = A(0), g_lp = A(0), g_h = A(0), h = A(0);
    auto inputs = [&](int64_t t0) {
        const int64_t t = t0 + lane;
        if (lane >= rows_of(t0)) return;
        y = a.labels.p ? a.labels.in(t, a.c) : 0;
        l = a.lse[t];
        g_lp = a.g_lp ? a.g_lp[t] : A(0);
        g_h = a.g_entropy ? a.g_entropy[t] : A(0);
        h = a.g_entropy ? a.entropy[t] : A(0);
    };
    if (i < n_tiles) {
        tile_fetch(x, ld, begin(i), rows_of(begin(i)), c, whole_in, tiles);
        inputs(begin(i));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int buf = 0; i < n_tiles; i += step, buf ^= 1) {
        const int64_t t0 = begin(i), t = t0 + lane;
        const int rows = rows_of(t0), y_now = y;
        const A l_now = l, lp_now = g_lp, h_now = h;
        A gh = g_h;
        T* const tile = tiles + buf * (kTileRows * c);
        if (i + step < n_tiles) {
            const int64_t next = begin(i + step);
            tile_fetch(x, ld, next, rows_of(next), c, whole_in, tiles + (buf ^ 1) * (kTileRows * c));
            inputs(next);
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        if (lane < rows) {
            T* row = tile + lane * c;
            const bool dead = y_now < 0 || l_now == minus_inf<A>();
            A sum = A(0), v[CW];
            if (!dead) {
                for (int j = 0; j < a.top; ++j) {
                    const int64_t id = a.id(t * a.top + j);
                    if (id >= 0 && id < a.c) sum += a.g_top[t * a.top + j];
                }
                sum += lp_now;
            } else {
                gh = A(0);
            }
            const bool none = sum == A(0) && gh == A(0);
            const Slope<A> slope{l_now, gh == A(0) ? sum : sum + gh * h_now, gh};
#pragma unroll
            for (int j = 0; j < CW; ++j)
                if (j < c) v[j] = none ? A(0) : slope.of(widen<A>(row[j]));
            if (!dead) {
                auto name = [&](int64_t id, A g) {
#pragma unroll
                    for (int j = 0; j < CW; ++j)
                        if (j == id) v[j] += g;
                };
                if (a.g_lp) name(y_now, lp_now);
                for (int j = 0; j < a.top; ++j) name(a.id(t * a.top + j), a.g_top[t * a.top + j]);
            }
#pragma unroll
            for (int j = 0; j < CW; ++j)
                if (j < c) row[j] = narrow<T>(v[j]);
        }
        __syncwarp();
        tile_put(out, ld_out, t0, rows, c, whole_out, tile);
        __syncwarp();  // the tile's buffer is filled again
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// L threads a row: every value by p alone, then again those of the label and the best
// classes with their gradients, summed over all places that name the class. Bound by HBM for
// long rows, for short ones by the dependent loads before a row is read (its label, lse and
// places say whether it is): few lanes a row, many rows in flight.
template <class T, class A, int L>
__global__ void __launch_bounds__(kNT, IsF64<A>::value ? 2 : 4)
    grad_kernel(const T* __restrict__ x, int64_t ld, T* __restrict__ out, int64_t ld_out, GradArgs<A> a) {
    constexpr int V = 16 / sizeof(T), U = 4, S = L < 32 ? L : 32;
    __shared__ A own[kNT / L][kTop + 1];
    __shared__ int at[kNT / L][kTop + 1];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    // from the last row to the first: the forward left the last ones in L2
    const int64_t back = (int64_t)blockIdx.x * (kNT / L) + group;
    if (L >= 32 && back >= a.n) return;  // the whole group
    const bool in = back < a.n;
    const int64_t t = in ? a.n - 1 - back : 0;
    const T* row = x + t * ld;
    T* to = out + t * ld_out;
    const RowShape<T> sh(row, in ? (int)a.c : 0);
    const bool whole = alike(row, to);
    const int y = a.labels.p ? a.labels.in(t, a.c) : 0;
    const A l = a.lse[t], g_lp = a.g_lp ? a.g_lp[t] : A(0);
    A gh = a.g_entropy ? a.g_entropy[t] : A(0), h = a.g_entropy ? a.entropy[t] : A(0);
    const bool dead = !in || y < 0 || l == minus_inf<A>();
    const int top = dead ? 0 : a.top, named = dead ? 0 : a.top + (a.g_lp ? 1 : 0);
    A sum = top || dead ? A(0) : g_lp;
    if (a.top) {
        for (int j = lane; j < named; j += L) {
            const int64_t i = j < top ? a.id(t * top + j) : (int64_t)y;
            const bool is = i >= 0 && i < a.c;
            at[group][j] = is ? (int)i : -1;
            own[group][j] = is ? (j < top ? a.g_top[t * top + j] : g_lp) : A(0);
        }
        group_sync<L>();
        if (top) {
            sum = A(0);
            for (int j = threadIdx.x % S; j < named; j += S) sum += own[group][j];
        }
        __syncwarp();
#pragma unroll
        for (int o = S / 2; o > 0; o >>= 1) {
            const A other = __shfl_xor_sync(0xffffffffu, sum, o);
            if (top) sum += other;
        }
    }
    if (dead) gh = A(0);
    const bool none = sum == A(0) && gh == A(0);
    const Slope<A> slope{l, gh == A(0) ? sum : sum + gh * h, gh};
    for (int i = lane; i < sh.edges; i += L) {
        const int j = sh.edge(i);
        to[j] = narrow<T>(none ? A(0) : slope.of(widen<A>(row[j])));
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
                    slope.all(p);
                }
                store16<T, A>(to + sh.head + (int64_t)(j0 + u * L) * V, p, whole);
            }
    }
    group_sync<L>();  // the places' values come after all others
    if (named == 0) return;
    if (top == 0) {
        if (lane == 0) to[y] = narrow<T>(g_lp + (none ? A(0) : slope.of(widen<A>(row[y]))));
        return;
    }
    for (int j = lane; j < named; j += L) {
        const int i = at[group][j];
        if (i < 0) continue;
        const T v = row[i];
        A mine = A(0);
#pragma unroll 4
        for (int o = 0; o < named; ++o) mine += at[group][o] == i ? own[group][o] : A(0);
        to[i] = narrow<T>(mine + (none ? A(0) : slope.of(widen<A>(v))));
    }
}

// ------------------------------------------------------------- launchers --

// The width of the registers that hold c classes.
template <class F>
void small_widths(int c, F&& f) {
    using std::integral_constant;
    if (c <= 4)
        f(integral_constant<int, 4>{});
    else if (c <= 8)
        f(integral_constant<int, 8>{});
    else if (c <= 12)
        f(integral_constant<int, 12>{});
    else if (c <= 16)
        f(integral_constant<int, 16>{});
    else if (c <= 24)
        f(integral_constant<int, 24>{});
    else
        f(integral_constant<int, 32>{});
}

// One wave of blocks of a kernel over tiles, with the shared memory it asks for.
template <auto Kernel>
unsigned small_grid(int device, int64_t n, int c, size_t bytes) {
    static bool asked[64];
    allow_smem(Kernel, device, 128 * 1024, asked, "class tile shared memory");
    static int per_sm[64][kSmallC + 1];  // the answer stays
    int per = per_sm[device & 63][c];
    if (per == 0) {
        MFM_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, Kernel, kSmallNT, bytes), "occupancy");
        per_sm[device & 63][c] = per = std::max(per, 1);
    }
    return (unsigned)std::min(ceil_div(n, kTileRows * (kSmallNT / 32)), (int64_t)sm_count(device) * per);
}

template <class T, class A>
void rows_launch(int device, const T* x, int64_t ld, const Args<A>& a, cudaStream_t s) {
    if (a.c <= kSmallC) {
        const bool whole = ld == a.c && (uintptr_t)x % 16 == 0;
        small_widths((int)a.c, [&](auto w) {
            constexpr int CW = decltype(w)::value;
            constexpr auto k = small_kernel<T, A, CW>;
            const size_t bytes = (kSmallNT / 32) * small_bytes<T, A, CW>((int)a.c);
            // e / top for e < 32 top as a product: exact, since 1024 / 65536 < 1 / 32
            k<<<small_grid<k>(device, a.n, (int)a.c, bytes), kSmallNT, bytes, s>>>(x, ld, a, whole, a.top ? 65536u / a.top + 1 : 0);
        });
        return;
    }
    const int64_t nv = a.c / Pack<T>::N, sms = sm_count(device);
    using std::integral_constant;
    auto held = [&](auto l, auto k) {
        constexpr int L = decltype(l)::value;
        held_kernel<T, A, L, decltype(k)::value><<<(unsigned)ceil_div(a.n, kNT / L), kNT, 0, s>>>(x, ld, a);
    };
    auto scan = [&](auto l) {
        constexpr int L = decltype(l)::value, bytes = (int)sizeof(Shared<A, L>) * (kNT / L);
        auto k = scan_kernel<T, A, L, 1>;
        static bool asked[64];
        allow_smem(k, device, bytes, asked, "row shared memory");
        k<<<(unsigned)ceil_div(a.n, kNT / L), kNT, bytes, s>>>(x, ld, a);
    };
    // As few lanes a row as are enough for the bound, two values each, or for ranking the values of a
    // short row without one (of double values as few as shared memory has lists for). By lanes, us
    // without best classes, with 5, 10, 16, 24:
    //   400000 x 100 bfloat16   4: 38, 92, 379   8: 55, 119, 162, 489   16: 10 best 238, 16 285, 24 795   32: 428, 465, 640
    //   200000 x 250 bfloat16   8: 38, 74, 95, 475   16: 58, 105, 121, 144, 198   32: 16 best 207, 24 228
    //   200000 x 500 float16    8: 61, 103, 131   16: 68, 119, 139, 162, 223   32: 111, 180, 207, 225, 248
    //   200000 x 1003 float16   16: 107, 172, 199, 229, 304   32: 131, 208, 238, 258, 287
    constexpr int kFour = IsF64<A>::value ? 8 : 4, kEight = IsF64<A>::value ? 16 : 8;
    const int top = a.top, two = 2 * fewest_vectors<Pack<T>::N>(a.c);
    if (nv <= 16 && top <= 5)
        held(integral_constant<int, kFour>{}, integral_constant<int, 16 / kFour>{});
    else if (nv <= 16 && (top <= 12 || a.c <= 64))
        held(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else if (nv <= 32 && top <= 12)
        held(integral_constant<int, kEight>{}, integral_constant<int, 32 / kEight>{});
    else if (nv <= 32 && (top <= min(24, two) || a.c <= 64))
        held(integral_constant<int, 16>{}, integral_constant<int, 2>{});
    else if (nv > 32 && nv <= 64 && top <= 10)
        held(integral_constant<int, kEight>{}, integral_constant<int, 64 / kEight>{});
    else if (nv > 32 && nv <= 64 && top <= 24)
        held(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    else if (nv > 64 && nv <= 128 && top <= 20)
        held(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else if (nv <= 32)
        held(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (nv <= 64)
        held(integral_constant<int, 32>{}, integral_constant<int, 2>{});
    else if (nv <= 128)
        held(integral_constant<int, 32>{}, integral_constant<int, 4>{});
    else if (nv <= 256)
        held(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if (nv >= 1024 && a.n <= sms / 2) {
        // so few rows that a cluster of eight blocks each fits at once
        constexpr int bytes = (int)sizeof(Shared<A, kNT>);
        auto k = scan_kernel<T, A, kNT, 8>;
        static bool asked[64];
        allow_smem(k, device, bytes, asked, "row shared memory");
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)a.n * 8);
        cfg.blockDim = dim3(kNT);
        cfg.dynamicSmemBytes = bytes;
        cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 8;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        MFM_CUDA(cudaLaunchKernelEx(&cfg, k, x, ld, a), "kernel launch");
    } else if (nv >= 1024 && a.n <= 2 * sms)
        scan(integral_constant<int, kNT>{});
    else if (nv >= 6144)
        scan(integral_constant<int, 128>{});
    else if (nv >= 1024)
        scan(integral_constant<int, 64>{});
    else
        scan(integral_constant<int, 32>{});
}

template <class T, class A>
void grad_launch(int device, const T* x, int64_t ld, T* out, int64_t ld_out, const GradArgs<A>& a, cudaStream_t s) {
    if (a.c <= kSmallC) {
        small_widths((int)a.c, [&](auto w) {
            constexpr auto k = small_grad_kernel<T, A, decltype(w)::value>;
            const size_t bytes = (size_t)(kSmallNT / 32) * 2 * kTileRows * a.c * sizeof(T);
            k<<<small_grid<k>(device, a.n, (int)a.c, bytes), kSmallNT, bytes, s>>>(
                x, ld, out, ld_out, a, ld == a.c && (uintptr_t)x % 16 == 0, ld_out == a.c && (uintptr_t)out % 16 == 0);
        });
        return;
    }
    auto go = [&](auto l) {
        constexpr int L = decltype(l)::value;
        grad_kernel<T, A, L><<<(unsigned)ceil_div(a.n, kNT / L), kNT, 0, s>>>(x, ld, out, ld_out, a);
    };
    const int64_t nv = a.c / Pack<T>::N;
    // 4, 8, 16, 32, 64 lanes a row, with five best classes: 400000 x 100 bf16 68, 102, 180, 365, 686 us
    // (160 MB: 24), 200000 x 250 59, 66; 200000 x 500 95, 92, 200000 x 1003 192, 158, 174, 248, 407;
    // 100000 x 2000 by 8 154, 145, 165, 218
    if (nv <= 32)
        go(std::integral_constant<int, 4>{});
    else if (nv <= 160)
        go(std::integral_constant<int, 8>{});
    else if (nv <= 512)
        go(std::integral_constant<int, 16>{});
    else if (nv < 1024)
        go(std::integral_constant<int, 32>{});
    else
        go(std::integral_constant<int, kNT>{});
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
            grad_launch<T, A>(device, (const T*)logits, ld, (T*)d_logits, ld_out, a, (cudaStream_t)stream);
        });
        MFM_CHECK_LAUNCH("label alternatives gradient launch");
    });
}
