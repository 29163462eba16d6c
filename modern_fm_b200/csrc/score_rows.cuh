// score_rows.cuh — rows of class scores, for the kernels that take their softmax: the
// exponentials and their sums, labels, the vectors of a row that begins anywhere, tiles
// of short rows in shared memory, and the entry points' checks.
#pragma once

#include "vecio.cuh"

namespace mfm {
namespace {

// exp(d). The 32-bit form, one multiply and ex2, is exact at 0 and off by at most
// (4 + 2 |d|) 2^-24 of the value (ex2.approx 2^-22; the product's and the constant's
// roundings), 0 below 2^-126. It is taken for the values of a row, where d <= 0: a value
// e^d of a sum of 1 or more is off by less than 2^-22 of 1, whatever d is. expf there
// takes 123 us instead of 100 us (log-probabilities, 8195 x 32000 bf16), 313 us instead
// of 229 us (policy, 4096 x 65536 bf16), 96 us instead of 84 us (400000 x 100 bf16).
__device__ __forceinline__ float exp_of(float d) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
    return r;
}
// a call: its code is long, and unrolled loops hold many
__device__ __noinline__ double exp_call(double d) { return exp(d); }
__device__ __forceinline__ double exp_of(double d) { return exp_call(d); }
__device__ __forceinline__ float log_of(float v) { return logf(v); }
__device__ __forceinline__ double log_of(double v) { return log(v); }

// Sums of exp(v - off), and k exp(v - off) for each value: two 32-bit lanes an
// instruction (the f32x2 forms round each lane as the scalar ones do), since
// 16-bit scores are otherwise bound by issue slots, not by bytes.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void pair_to(uint64_t r, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t pair_exp(float a, float b, uint64_t minus_off) {
    const uint64_t d = pair_mul(pair_add(pair_of(a, b), minus_off), pair_of(1.4426950408889634f, 1.4426950408889634f));
    float p, q;
    pair_to(d, p, q);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(p));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(q));
    return pair_of(p, q);
}
// Adds N values' exponentials to `acc`, a pair of partial sums.
template <int N>
__device__ __forceinline__ void add_exp(uint64_t& acc, const float (&v)[N], uint64_t minus_off) {
#pragma unroll
    for (int q = 0; q < N; q += 2) acc = pair_add(acc, pair_exp(v[q], v[q + 1], minus_off));
}
template <int N>
__device__ __forceinline__ void scaled_exp(float (&v)[N], float k, uint64_t minus_off) {
    const uint64_t kk = pair_of(k, k);
#pragma unroll
    for (int q = 0; q < N; q += 2) pair_to(pair_mul(pair_exp(v[q], v[q + 1], minus_off), kk), v[q], v[q + 1]);
}
template <class A>
struct ExpSum {  // running sum of exp(v - off)
    uint64_t acc = 0, moff;
    __device__ __forceinline__ explicit ExpSum(float off) : moff(pair_of(-off, -off)) {}
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N]) { add_exp(acc, v, moff); }
    __device__ __forceinline__ float sum() const {
        float a, b;
        pair_to(acc, a, b);
        return a + b;
    }
    template <int N>
    __device__ __forceinline__ void scaled(float (&v)[N], float k) const { scaled_exp(v, k, moff); }
};
template <>
struct ExpSum<double> {
    double acc = 0.0, off;
    __device__ __forceinline__ explicit ExpSum(double o) : off(o) {}
    template <int N>
    __device__ __forceinline__ void add(const double (&v)[N]) {
#pragma unroll
        for (int q = 0; q < N; ++q) acc += exp_of(v[q] - off);
    }
    __device__ __forceinline__ double sum() const { return acc; }
    template <int N>
    __device__ __forceinline__ void scaled(double (&v)[N], double k) const {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = k * exp_of(v[q] - off);
    }
};

template <class A>
__device__ __forceinline__ A minus_inf() { return (A)(-INFINITY); }

// Labels are int32 or int64 (one load per row: no type of its own in the kernels).
struct Labels {
    const void* p;
    int is64;
    // the label of token t, -1 for one outside [0, c)
    __device__ __forceinline__ int in(int64_t t, int64_t c) const {
        const int64_t y = is64 ? static_cast<const int64_t*>(p)[t] : (int64_t)static_cast<const int32_t*>(p)[t];
        return y >= 0 && y < c ? (int)y : -1;
    }
};

// The offset subtracted before exp: the maximum, or 0 for a row of -inf, so that
// such rows sum to 0 and NaN stays NaN.
template <class A>
__device__ __forceinline__ A offset_of(A m) { return m == minus_inf<A>() ? A(0) : m; }

template <class A>
struct RowStats {
    A m, s;  // maximum, sum of exp(x - offset_of(m))
};

// The statistics of `width` neighbouring lanes joined, on each of them.
template <class A>
__device__ __forceinline__ void across(RowStats<A>& r, int width) {
    const A was = r.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < width) r.m = fmax(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
    if (r.m != minus_inf<A>()) r.s *= exp_of(was - r.m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < width) r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
}

__device__ __forceinline__ uint4 load16(const void* p) { return *static_cast<const uint4*>(p); }

// A warp works on tiles of 32 rows, a thread per row, and copies the next tile into
// shared memory while it works on one. Tiles keep the scores' type and layout, so
// whole 16-byte pieces come and go; the result takes its row's place there.
constexpr int kTileRows = 32;

// Copies a tile's elements: asynchronously where the rows are contiguous and
// aligned (`whole`), one by one otherwise. The caller commits the group.
template <class T>
__device__ __forceinline__ void tile_fetch(const T* x, int64_t ld, int64_t t0, int rows, int c,
                                           bool whole, T* tile) {
    const int lane = threadIdx.x & 31, total = rows * c;
    const T* at = x + t0 * ld;
    if (whole) {
        constexpr int V = Pack<T>::N;
        const int vecs = total / V;
        for (int i = lane; i < vecs; i += 32)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                             (uint32_t)__cvta_generic_to_shared(tile + i * V)),
                         "l"(at + i * V)
                         : "memory");
        for (int i = vecs * V + lane; i < total; i += 32) tile[i] = at[i];
    } else {
        for (int i = lane; i < total; i += 32) tile[i] = at[(i / c) * ld + i % c];
    }
}

template <class T>
__device__ __forceinline__ void tile_put(T* out, int64_t ld, int64_t t0, int rows, int c, bool whole,
                                         const T* tile) {
    const int lane = threadIdx.x & 31, total = rows * c;
    T* at = out + t0 * ld;
    if (whole) {
        constexpr int V = Pack<T>::N;
        const int vecs = total / V;
        for (int i = lane; i < vecs; i += 32) *reinterpret_cast<uint4*>(at + i * V) = load16(tile + i * V);
        for (int i = vecs * V + lane; i < total; i += 32) at[i] = tile[i];
    } else {
        for (int i = lane; i < total; i += 32) at[(i / c) * ld + i % c] = tile[i];
    }
}

// The column at which a thread begins its row, where c is a multiple of 4 (two
// rows at most meet in a bank otherwise). Rows of c elements meet in the same
// banks after 32 / gcd(c, 32) rows (64-bit values: of 16 lanes; 16-bit ones:
// pairs); each such round of rows begins one column further on.
template <class T>
__device__ __forceinline__ int first_column(int c) {
    const int lane = threadIdx.x & 31, g = c & -c;
    if (sizeof(T) == 8) return (lane & 15) * (g < 16 ? g : 16) / 16 % c;
    if (sizeof(T) == 2) return g == 1 ? 0 : 2 * (lane * (g / 2 < 32 ? g / 2 : 32) / 32) % c;
    return lane * (g < 32 ? g : 32) / 32 % c;
}

// Where a row's 16-byte vectors begin, how many there are, and the single
// elements before and behind them (at most 2 (V - 1): one per lane).
template <class T>
struct RowShape {
    static constexpr int V = 16 / sizeof(T);
    int head, nv, edges;
    __device__ __forceinline__ RowShape(const T* x, int c) {
        const int h = (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T));
        head = h < c ? h : c;
        nv = (c - head) / V;
        edges = c - nv * V;
    }
    __device__ __forceinline__ int edge(int i) const { return i < head ? i : i + nv * V; }
};

// Whether two rows have the same place within 16 bytes, so that their vectors do.
__device__ __forceinline__ bool alike(const void* a, const void* b) {
    return ((uintptr_t)a - (uintptr_t)b) % 16 == 0;
}

// The lane that writes the vector with column y of a row (-1: an edge element or
// none). It writes the label's element once more, by itself, behind its vectors:
// the loops over vectors then carry no test for it.
template <class T, int L>
__device__ __forceinline__ int label_lane(const RowShape<T>& sh, int y) {
    const unsigned j = (unsigned)(y - sh.head) / (unsigned)RowShape<T>::V;
    return y >= sh.head && j < (unsigned)sh.nv ? (int)(j % (unsigned)L) : -1;
}

// N values to `at`: as one vector, or one by one where the rows of scores and
// gradient are not alike.
template <class T, class A>
__device__ __forceinline__ void store16(T* at, const A (&v)[Pack<T>::N], bool whole) {
    if (whole) {
        *reinterpret_cast<uint4*>(at) = Pack<T>::pack(v);
    } else {
#pragma unroll
        for (int q = 0; q < Pack<T>::N; ++q) at[q] = narrow<T>(v[q]);
    }
}

// ---------------------------------------------------------------- checks --

void check_scores(int dtype, const void* logits, int64_t ld, int64_t n, int64_t c,
                  const void* labels) {
    if (dtype != MFM_DTYPE_F64 && dtype != MFM_DTYPE_F32 && dtype != MFM_DTYPE_BF16 && dtype != MFM_DTYPE_F16)
        fail(MFM_ERR_INVALID, fmt("unknown dtype %d", dtype));
    if (n < 0 || c < 1) fail(MFM_ERR_INVALID, "n_tokens must be >= 0 and n_classes >= 1");
    if (n > 0 && (!logits || !labels)) fail(MFM_ERR_INVALID, "logits and labels must be provided");
    if (n > 0 && ld < c) fail(MFM_ERR_INVALID, fmt("row pitch of logits %lld < %lld", (long long)ld, (long long)c));
    if (n > INT32_MAX || c > INT32_MAX)
        fail(MFM_ERR_UNSUPPORTED, "n_tokens and n_classes exceed the engine's 2^31-1 limit");
}

template <class P>
using Elem = std::remove_const_t<std::remove_pointer_t<std::remove_reference_t<P>>>;

template <class F>
void with_score_types(int dtype, F&& f) {
    switch (dtype) {
        case MFM_DTYPE_F64: f((double*)nullptr); break;
        case MFM_DTYPE_F32: f((float*)nullptr); break;
        case MFM_DTYPE_BF16: f((__nv_bfloat16*)nullptr); break;
        default: f((__half*)nullptr); break;
    }
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }
size_t arith_size(int dtype) { return dtype == MFM_DTYPE_F64 ? 8 : 4; }

void check_out(const void* out, int64_t ld_out, int64_t n, int64_t c) {
    if (out && n > 0 && ld_out < c)
        fail(MFM_ERR_INVALID, fmt("row pitch of d_logits %lld < %lld", (long long)ld_out, (long long)c));
}

void check_workspace(const void* ws, int64_t have, int64_t need) {
    if (need > 0 && (!ws || have < need))
        fail(MFM_ERR_INVALID, fmt("workspace of %lld bytes, %lld needed", (long long)have, (long long)need));
    if ((uintptr_t)ws % 256) fail(MFM_ERR_INVALID, "workspace must be 256-byte aligned");
}

}  // namespace
}  // namespace mfm
