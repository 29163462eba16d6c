// preference.cu — losses of class scores by label log-probabilities: the
// log-probabilities themselves, the paired preference loss and the clipped
// policy loss with a KL term, each with the gradient of the scores.
//
// Per token row x of C scores with label y: lse = m + log sum exp(x - m), m = max x;
// lp = x[y] - lse; a loss with derivative g in lp has d/dx[c] = g ([c = y] - exp(x[c] - lse)).
#include "vecio.cuh"

#include <algorithm>

namespace mfm {
namespace {

constexpr int kNT = 256;

__device__ __forceinline__ float exp_of(float d) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
    return r;
}
__device__ __forceinline__ double exp_of(double d) { return exp(d); }
__device__ __forceinline__ float log_of(float v) { return logf(v); }
__device__ __forceinline__ double log_of(double v) { return log(v); }

template <class A>
__device__ __forceinline__ A minus_inf() { return (A)(-INFINITY); }

// A running maximum m and s = sum of exp(x - m); m = -inf stands for an offset of 0
// so that rows of -inf stay 0 and NaN stays NaN.
template <class A>
struct Softmax {
    A m = minus_inf<A>(), s = A(0);
    __device__ __forceinline__ A off() const { return m == minus_inf<A>() ? A(0) : m; }
    template <int N>
    __device__ __forceinline__ void add(const A (&x)[N]) {
        A top = m;
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmax(top, x[j]);
        if (top > m) {
            s *= exp_of(m - top);
            m = top;
        }
        const A o = off();
#pragma unroll
        for (int j = 0; j < N; ++j) s += exp_of(x[j] - o);
    }
    __device__ __forceinline__ void join(A m2, A s2) {
        const A top = fmax(m, m2);
        if (top == minus_inf<A>()) {
            s += s2;
        } else {
            s = s * exp_of(m - top) + s2 * exp_of(m2 - top);
            m = top;
        }
    }
};

// Group of L lanes working on one row; L = kNT is the whole block.
template <class A, int L>
__device__ __forceinline__ void group_join(Softmax<A>& r, A* sm) {
    constexpr int W = L < 32 ? L : 32;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        const A m2 = __shfl_xor_sync(0xffffffffu, r.m, o);
        const A s2 = __shfl_xor_sync(0xffffffffu, r.s, o);
        r.join(m2, s2);
    }
    if (L > 32) {
        const int warp = threadIdx.x / 32;
        if ((threadIdx.x & 31) == 0) {
            sm[2 * warp] = r.m;
            sm[2 * warp + 1] = r.s;
        }
        __syncthreads();
        Softmax<A> t;
#pragma unroll
        for (int w = 0; w < L / 32; ++w) t.join(sm[2 * w], sm[2 * w + 1]);
        r = t;
        __syncthreads();
    }
}

// Elements before the first 16-byte boundary of a row (all of them when the row is short).
template <class T, int VEC>
__device__ __forceinline__ int64_t head_of(const T* x, int64_t c) {
    if (VEC == 1) return 0;
    const int64_t h = (int64_t)((16 - (uintptr_t)x % 16) % 16 / sizeof(T));
    return h < c ? h : c;
}

template <class T, class A, int VEC, int L>
__device__ __forceinline__ Softmax<A> row_softmax(const T* x, int64_t c, int lane, A* sm) {
    Softmax<A> r;
    const int64_t h = head_of<T, VEC>(x, c), nv = (c - h) / VEC;
    for (int64_t j = lane; j < h; j += L) {
        const A v[1] = {widen<A>(x[j])};
        r.add(v);
    }
    for (int64_t j = lane; j < nv; j += L) {
        const Vec<T, VEC> p = ldg_vec<T, VEC>(x + h + j * VEC);
        A v[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[q] = widen<A>(p.v[q]);
        r.add(v);
    }
    for (int64_t j = h + nv * VEC + lane; j < c; j += L) {
        const A v[1] = {widen<A>(x[j])};
        r.add(v);
    }
    group_join<A, L>(r, sm);
    return r;
}

// out = g ([c = y] - exp(x - lse)); x and out have the same place within 16 bytes when VEC > 1.
template <class T, class A, int VEC, int L>
__device__ __forceinline__ void row_grad(const T* x, T* out, int64_t c, int64_t y, A g, A lse,
                                         int lane) {
    const int64_t h = head_of<T, VEC>(x, c), nv = (c - h) / VEC;
    auto one = [&](T v, int64_t j) {
        return g == A(0) ? narrow<T>(A(0))
                         : narrow<T>(g * ((j == y ? A(1) : A(0)) - exp_of(widen<A>(v) - lse)));
    };
    for (int64_t j = lane; j < h; j += L) out[j] = one(x[j], j);
    for (int64_t j = lane; j < nv; j += L) {
        const int64_t at = h + j * VEC;
        Vec<T, VEC> p = ldg_vec<T, VEC>(x + at);
#pragma unroll
        for (int q = 0; q < VEC; ++q) p.v[q] = one(p.v[q], at + q);
        *reinterpret_cast<Vec<T, VEC>*>(out + at) = p;
    }
    for (int64_t j = h + nv * VEC + lane; j < c; j += L) out[j] = one(x[j], j);
}

// (lse, label's log-probability, unmasked) of a finished row.
template <class T, class A>
__device__ __forceinline__ void finish_row(const Softmax<A>& r, const T* x, int64_t c, int64_t y,
                                           A& lse, A& lp, bool& live) {
    const bool empty = r.m == minus_inf<A>() && r.s == A(0);
    const A ls = log_of(r.s);
    lse = empty ? minus_inf<A>() : r.off() + ls;
    live = y >= 0 && y < c && !empty;
    lp = live ? (widen<A>(x[y]) - r.off()) - ls : A(0);
}

template <class T, class A, class I, int VEC, int L>
__global__ void __launch_bounds__(kNT)
    label_stats_kernel(const T* __restrict__ x, int64_t ld, int64_t n, int64_t c,
                       const I* __restrict__ labels, A* __restrict__ lp, A* __restrict__ lse,
                       A* __restrict__ zero) {
    __shared__ A sm[2 * kNT / 32];
    const int lane = threadIdx.x % L;
    const int64_t t = (int64_t)blockIdx.x * (kNT / L) + threadIdx.x / L;
    const bool in = t < n;
    const T* row = x + (in ? t : 0) * ld;
    const Softmax<A> r = row_softmax<T, A, VEC, L>(row, in ? c : 0, lane, sm);
    if (in && lane == 0) {
        A s, p;
        bool live;
        finish_row(r, row, c, (int64_t)labels[t], s, p, live);
        lp[t] = p;
        if (lse) lse[t] = s;
        if (zero) zero[t] = A(0);
    }
}

// scale: factor of every g (NULL = 1), on the device.
template <class T, class A, class I, int VEC, int L>
__global__ void __launch_bounds__(kNT)
    label_grad_kernel(const T* __restrict__ x, int64_t ld, int64_t n, int64_t c,
                      const I* __restrict__ labels, const A* __restrict__ g,
                      const double* __restrict__ scale, const A* __restrict__ lse,
                      T* __restrict__ out, int64_t ld_out) {
    const int lane = threadIdx.x % L;
    const int64_t t = (int64_t)blockIdx.x * (kNT / L) + threadIdx.x / L;
    if (t >= n) return;
    const int64_t y = (int64_t)labels[t];
    A f = y >= 0 && y < c && lse[t] != minus_inf<A>() ? g[t] : A(0);
    if (scale) f = (A)((double)f * *scale);
    row_grad<T, A, VEC, L>(x + t * ld, out + t * ld_out, c, y, f, lse[t], lane);
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

// One warp per pair: sums, margin, the pair's weighted loss and its unnormalised
// derivative, written to every token of the two sequences.
template <class A>
__global__ void __launch_bounds__(kNT)
    pair_kernel(const A* __restrict__ lp, int64_t n, const int64_t* __restrict__ indptr,
                int64_t n_pairs, const A* __restrict__ reference, double beta, double eps,
                const A* __restrict__ weight, A* __restrict__ margins, A* __restrict__ sums,
                double* __restrict__ pair_loss, A* __restrict__ g) {
    const int64_t p = (int64_t)blockIdx.x * (kNT / 32) + threadIdx.x / 32;
    const int lane = threadIdx.x & 31;
    if (p >= n_pairs) return;
    int64_t lo[2], hi[2];
    double s[2];
    for (int i = 0; i < 2; ++i) {
        seq_bounds(indptr, p + i * n_pairs, n, lo[i], hi[i]);
        s[i] = warp_seq_sum(lp, lo[i], hi[i]);
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
        pair_loss[p] = w == 0.0 ? 0.0 : w * (soft + (1.0 - eps) * fmax(-z, 0.0) + eps * fmax(z, 0.0));
    }
    if (g)
        for (int i = 0; i < 2; ++i)
            for (int64_t t = lo[i] + lane; t < hi[i]; t += 32) g[t] = (A)(i ? -slope : slope);
}

// Sums of `width` interleaved columns and of the weights by one block in a fixed order.
__device__ __forceinline__ double block_sum(double v, double* sm) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x / 32] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) t += sm[w];
    __syncthreads();
    return t;
}

template <class A>
__global__ void __launch_bounds__(1024)
    pair_finish_kernel(const double* __restrict__ pair_loss, const A* __restrict__ weight,
                       int64_t n_pairs, A* __restrict__ loss, double* __restrict__ scale) {
    __shared__ double sm[32];
    double a = 0.0, b = 0.0;
    for (int64_t p = threadIdx.x; p < n_pairs; p += 1024) {
        a += pair_loss[p];
        b += weight ? (double)weight[p] : 1.0;
    }
    a = block_sum(a, sm);
    b = block_sum(b, sm);
    if (threadIdx.x == 0) {
        *loss = b != 0.0 ? (A)(a / b) : A(0);
        *scale = b != 0.0 ? 1.0 / b : 0.0;
    }
}

constexpr int kWeightBlocks = 128;

template <class A, class I>
__global__ void __launch_bounds__(kNT)
    weight_kernel(const I* __restrict__ labels, int64_t c, const A* __restrict__ weight, int64_t n,
                  double* __restrict__ part) {
    __shared__ double sm[kNT / 32];
    double a = 0.0;
    for (int64_t t = (int64_t)blockIdx.x * kNT + threadIdx.x; t < n; t += (int64_t)gridDim.x * kNT) {
        const int64_t y = (int64_t)labels[t];
        if (y >= 0 && y < c) a += weight ? (double)weight[t] : 1.0;
    }
    a = block_sum(a, sm);
    if (threadIdx.x == 0) part[blockIdx.x] = a;
}

struct PolicyArgs {
    double clip_low, clip_high, kl_coef;
};

// One group per token: statistics, the token's loss terms and its gradient row.
template <class T, class A, class I, int VEC, int L>
__global__ void __launch_bounds__(kNT)
    policy_kernel(const T* __restrict__ x, int64_t ld, int64_t n, int64_t c,
                  const I* __restrict__ labels, const A* __restrict__ old,
                  const A* __restrict__ adv, const A* __restrict__ ref, PolicyArgs k,
                  const A* __restrict__ weight, const double* __restrict__ wpart, int n_wpart,
                  double* __restrict__ part, A* __restrict__ lps, T* __restrict__ out,
                  int64_t ld_out) {
    __shared__ A sm[2 * kNT / 32];
    __shared__ double terms[3][kNT / L];
    const int lane = threadIdx.x % L, row_in = threadIdx.x / L;
    const int64_t t = (int64_t)blockIdx.x * (kNT / L) + row_in;
    const bool in = t < n;
    const T* row = x + (in ? t : 0) * ld;
    double total = 0.0;
    for (int i = threadIdx.x & 31; i < n_wpart; i += 32) total += wpart[i];
    total = warp_sum(total);
    const Softmax<A> r = row_softmax<T, A, VEC, L>(row, in ? c : 0, lane, sm);
    double e[3] = {0.0, 0.0, 0.0};
    if (in) {
        const int64_t y = (int64_t)labels[t];
        A lse, lp;
        bool live;
        finish_row(r, row, c, y, lse, lp, live);
        A g = A(0);
        const double w = live && weight ? (double)weight[t] : 1.0;
        if (live && w != 0.0) {  // a token of weight 0 is left out, whatever its ratio
            const double a = (double)adv[t];
            const double ratio = exp((double)lp - (double)old[t]);
            const double bent = fmin(fmax(ratio, 1.0 - k.clip_low), 1.0 + k.clip_high);
            const bool cut = ratio * a > bent * a;
            double slope = cut ? 0.0 : -ratio * a, kl = 0.0;
            if (ref) {
                const double u = (double)ref[t] - (double)lp, eu = expm1(u);
                kl = eu - u;
                slope -= k.kl_coef * eu;
            }
            e[0] = w * (-(cut ? bent * a : ratio * a) + k.kl_coef * kl);
            e[1] = w * kl;
            e[2] = cut ? w : 0.0;
            g = total != 0.0 ? (A)(w * slope / total) : A(0);
        }
        if (lane == 0) lps[t] = lp;
        if (out) row_grad<T, A, VEC, L>(row, out + t * ld_out, c, y, g, lse, lane);
    }
    if (lane == 0)
        for (int i = 0; i < 3; ++i) terms[i][row_in] = e[i];
    __syncthreads();
    if (threadIdx.x < 3) {
        double a = 0.0;
        for (int i = 0; i < kNT / L; ++i) a += terms[threadIdx.x][i];
        part[3 * (int64_t)blockIdx.x + threadIdx.x] = a;
    }
}

template <class A>
__global__ void __launch_bounds__(1024)
    policy_finish_kernel(const double* __restrict__ part, int64_t n_part,
                         const double* __restrict__ wpart, int n_wpart, A* __restrict__ stats) {
    __shared__ double sm[32];
    double e[3] = {0.0, 0.0, 0.0}, w = 0.0;
    for (int64_t p = threadIdx.x; p < n_part; p += 1024)
        for (int i = 0; i < 3; ++i) e[i] += part[3 * p + i];
    for (int i = 0; i < 3; ++i) e[i] = block_sum(e[i], sm);
    for (int i = threadIdx.x; i < n_wpart; i += 1024) w += wpart[i];
    w = block_sum(w, sm);
    if (threadIdx.x < 3) stats[threadIdx.x] = w != 0.0 ? (A)(e[threadIdx.x] / w) : A(0);
}

// ------------------------------------------------------------- launchers --

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

// f(VEC, L): 16-byte vectors where rows of scores and gradient have the same place
// within 16 bytes; lanes per row by the number of classes.
template <class T, class F>
void with_shape(const void* x, int64_t ld, const void* out, int64_t ld_out, int64_t c, F&& f) {
    constexpr int V = 16 / sizeof(T);
    const bool alike = !out || (((uintptr_t)x - (uintptr_t)out) % 16 == 0 && (ld - ld_out) % V == 0);
    auto lanes = [&](auto vec) {
        if (c <= 32)
            f(vec, std::integral_constant<int, 8>{});
        else if (c <= 2048)
            f(vec, std::integral_constant<int, 32>{});
        else
            f(vec, std::integral_constant<int, kNT>{});
    };
    if (alike && c > 32)
        lanes(std::integral_constant<int, V>{});
    else
        lanes(std::integral_constant<int, 1>{});
}

template <int L>
unsigned row_blocks(int64_t n) { return (unsigned)ceil_div(n, kNT / L); }

template <class T, class A, class I>
void stats_launch(const T* x, int64_t ld, int64_t n, int64_t c, const I* labels, A* lp, A* lse,
                  A* zero, cudaStream_t s) {
    if (n == 0) return;
    with_shape<T>(x, ld, nullptr, 0, c, [&](auto v, auto l) {
        constexpr int V = decltype(v)::value, L = decltype(l)::value;
        label_stats_kernel<T, A, I, V, L><<<row_blocks<L>(n), kNT, 0, s>>>(x, ld, n, c, labels, lp, lse, zero);
    });
    MFM_CHECK_LAUNCH("label log-probabilities launch");
}

template <class T, class A, class I>
void grad_launch(const T* x, int64_t ld, int64_t n, int64_t c, const I* labels, const A* g,
                 const double* scale, const A* lse, T* out, int64_t ld_out, cudaStream_t s) {
    if (n == 0) return;
    with_shape<T>(x, ld, out, ld_out, c, [&](auto v, auto l) {
        constexpr int V = decltype(v)::value, L = decltype(l)::value;
        label_grad_kernel<T, A, I, V, L><<<row_blocks<L>(n), kNT, 0, s>>>(x, ld, n, c, labels, g, scale, lse, out, ld_out);
    });
    MFM_CHECK_LAUNCH("label gradient launch");
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
            with_index_type(labels64, [&](auto* i) {
                using I = Elem<decltype(i)>;
                stats_launch<T, A, I>((const T*)logits, ld, n_tokens, n_classes, (const I*)labels,
                                      (A*)logprobs, (A*)lse, nullptr, s);
            });
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
            with_index_type(labels64, [&](auto* i) {
                using I = Elem<decltype(i)>;
                grad_launch<T, A, I>((const T*)logits, ld, n_tokens, n_classes, (const I*)labels,
                                     (const A*)grad, nullptr, (const A*)lse, (T*)d_logits, ld_out,
                                     (cudaStream_t)stream);
            });
        });
    });
}

namespace {
struct PrefWs {  // log-probabilities, lse, token coefficients, pair losses, 1 / sum of weights
    size_t lse, g, pair, scale, bytes;
    PrefWs(int dtype, int64_t n, int64_t pairs) {
        const size_t a = up256((size_t)n * arith_size(dtype));
        lse = a;
        g = 2 * a;
        pair = 3 * a;
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
        with_score_types(dtype, [&](auto* t) {
            using T = Elem<decltype(t)>;
            using A = typename Arith<T>::type;
            A *lp = (A*)ws, *lse = (A*)(ws + W.lse), *coef = d_logits ? (A*)(ws + W.g) : nullptr;
            with_index_type(labels64, [&](auto* i) {
                using I = Elem<decltype(i)>;
                stats_launch<T, A, I>((const T*)logits, ld, n_tokens, n_classes, (const I*)labels,
                                      lp, lse, coef, s);
                if (n_pairs > 0)
                    pair_kernel<A><<<(unsigned)ceil_div(n_pairs, kNT / 32), kNT, 0, s>>>(
                        lp, n_tokens, indptr, n_pairs, (const A*)reference, beta, label_smoothing,
                        (const A*)sample_weight, (A*)margins, (A*)seq_logprobs, pair, coef);
                pair_finish_kernel<A><<<1, 1024, 0, s>>>(pair, (const A*)sample_weight, n_pairs, (A*)loss, scale);
                MFM_CHECK_LAUNCH("preference loss launch");
                if (d_logits)
                    grad_launch<T, A, I>((const T*)logits, ld, n_tokens, n_classes,
                                         (const I*)labels, coef, scale, lse, (T*)d_logits, ld_out, s);
            });
        });
    });
}

namespace {
struct PolicyWs {  // partial weights, partial loss terms
    size_t part, bytes;
    explicit PolicyWs(int64_t n) {
        part = up256(kWeightBlocks * 8);
        bytes = part + up256((size_t)n * 24);
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
        const int nw = (int)std::min<int64_t>(kWeightBlocks, ceil_div(n_tokens, kNT));
        with_score_types(dtype, [&](auto* t) {
            using T = Elem<decltype(t)>;
            using A = typename Arith<T>::type;
            int64_t n_part = 0;
            if (n_tokens > 0)
                with_index_type(labels64, [&](auto* i) {
                    using I = Elem<decltype(i)>;
                    weight_kernel<A, I><<<nw, kNT, 0, s>>>((const I*)labels, n_classes, (const A*)sample_weight, n_tokens, wpart);
                    with_shape<T>(logits, ld, d_logits, ld_out, n_classes, [&](auto v, auto l) {
                        constexpr int V = decltype(v)::value, L = decltype(l)::value;
                        n_part = row_blocks<L>(n_tokens);
                        policy_kernel<T, A, I, V, L><<<(unsigned)n_part, kNT, 0, s>>>(
                            (const T*)logits, ld, n_tokens, n_classes, (const I*)labels,
                            (const A*)old_logprobs, (const A*)advantages, (const A*)reference,
                            PolicyArgs{clip_low, clip_high, kl_coef}, (const A*)sample_weight,
                            wpart, nw, part, (A*)logprobs, (T*)d_logits, ld_out);
                    });
                });
            policy_finish_kernel<A><<<1, 1024, 0, s>>>(part, n_part, wpart, nw, (A*)stats);
            MFM_CHECK_LAUNCH("policy loss launch");
        });
    });
}
