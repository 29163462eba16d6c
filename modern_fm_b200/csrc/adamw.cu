// adamw.cu — the AdamW step over many tensors at once: moments in 32 or 64 bits or in
// 8, master weights, a clip of the gradients' norm, and tables stepped by touched rows.
//
//   g = s grad,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p -= lr wd p + lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
// with s = grad_scale min(1, max_norm / norm). t is the device's own count, so that a
// captured step goes on; a table's rows have one each (the engine's lazy Adam).
//
// One pass over p, g, m, v: bound by HBM (28 bytes a value with float32 everything: 332 M values
// 1.49 ms, 6.2 TB/s), but for 8-bit moments (10 bytes a value of 16 bits): those are bound by the
// integer pipe, which decodes and encodes (184 M values 444 us, 4.2 TB/s; 68 instructions a
// value, half of them its). All tensors of one kind of types are one launch: their
// descriptions travel in the kernel's parameters, and persistent blocks walk chunks across
// them. A norm is one launch more, whose last block leaves the factor s.
#include "vecio.cuh"

#include <algorithm>
#include <cmath>

namespace mfm {
namespace {

constexpr int kNT = 256;
constexpr int kPer = 8;                     // values a thread and chunk
constexpr int64_t kChunk = kNT * kPer;      // values a block takes at once
constexpr int kFew = 40, kMany = 400;       // descriptions a launch carries (4 or 32 KB of parameters)
constexpr int kNormFew = 100, kNormMany = 800;
constexpr unsigned kNormBlocks = 1024;      // the most, each with its sum in the workspace

// ------------------------------------------------------------ 8-bit moments --

// Blocks of 32 neighbouring values share an exponent byte X. Code k > 0 stands for the
// float32 whose upper 11 bits (exponent and 3 bits of mantissa) are the number 8 X + k.
// m has a sign and 7 bits (15 octaves), v 8 bits (31 octaves: it holds squares). Scales
// are powers of two, so a value that stays is encoded as itself whatever its block's
// largest does.
constexpr unsigned kHalfStep = (1u << 19) + 64;  // what `code` adds to m, of which it says why
template <bool SIGNED>
struct Code {
    static constexpr unsigned kMost = SIGNED ? 127 : 255, kReach = SIGNED ? 15 : 31;
    static __device__ __forceinline__ float value(unsigned code, unsigned x) {
        const unsigned k = code & kMost, bits = k ? (8 * x + k) << 20 : 0;
        return __uint_as_float(SIGNED ? bits | (code & 128) << 24 : bits);
    }
    // The number of a magnitude's bits after `add` below it; finite values stay finite,
    // infinity and NaN stay what they are (whose bits could wrap).
    static __device__ __forceinline__ unsigned number(unsigned bits, unsigned add) {
        return bits < 0x7f800000u ? min((bits + add) >> 20, 0x7f7u) : bits == 0x7f800000u ? 0x7f8u : 0x7fcu;
    }
    // The shared exponent by the block's largest magnitude, as it rounds (v: as it may).
    static __device__ __forceinline__ unsigned shared(unsigned largest) {
        const unsigned top = number(largest, SIGNED ? kHalfStep : (1u << 20) - 1) >> 3;
        return top > kReach ? top - kReach : 0;
    }
    // `add`: for m half a step and 64 units of the last place, so that ties, which 0.9 m +
    // 0.1 g of values of few bits often is, go up whatever the sum's last bits are; for v 20
    // random bits: b2 = 0.999 moves v by a thousandth of itself, and rounded to nearest it
    // would stand still until g^2 is some 50 times v. What is above 0 stays above 0 in v,
    // where 0 would leave m / eps.
    static __device__ __forceinline__ unsigned code(float v, unsigned add, unsigned x) {
        const unsigned bits = __float_as_uint(v) & 0x7fffffffu, n = number(bits, add), base = 8 * x;
        if (bits == 0) return 0;
        const unsigned k = n > base ? min(n - base, kMost) : SIGNED ? 0u : 1u;
        return SIGNED ? k | (__float_as_uint(v) >> 31) << 7 : k;
    }
};
using MCode = Code<true>;
using VCode = Code<false>;

// Two codes, one in each half of a word, as the bfloat16 values that they stand for: a number's bits
// are the float32's upper ones. base: x << 7 in each half.
template <bool SIGNED>
__device__ __forceinline__ unsigned halves_of(unsigned pair, unsigned base) {
    const unsigned k = SIGNED ? pair & 0x007f007fu : pair;
    const unsigned some = ((k + 0x00ff00ffu) >> 8 & 0x00010001u) * 0xffffu;  // of codes that are not 0
    const unsigned bits = (k * 16 + base) & some;
    return SIGNED ? bits | (pair & 0x00800080u) << 8 : bits;
}
// Four codes of a word as float32.
template <bool SIGNED>
__device__ __forceinline__ void four_of(unsigned word, unsigned base, float* v) {
    const unsigned low = halves_of<SIGNED>(__byte_perm(word, 0, 0x4140), base);
    const unsigned high = halves_of<SIGNED>(__byte_perm(word, 0, 0x4342), base);
    v[0] = __uint_as_float(low << 16);
    v[1] = __uint_as_float(low & 0xffff0000u);
    v[2] = __uint_as_float(high << 16);
    v[3] = __uint_as_float(high & 0xffff0000u);
}

// 32 bits that depend on each bit of x: two rounds of shift, xor and product (the
// finaliser of MurmurHash3, A. Appleby).
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x85ebca6bu;
    x = (x ^ (x >> 13)) * 0xc2b2ae35u;
    return x ^ (x >> 16);
}
// The rounding of value e of a tensor, 20 bits; key: of seed, tensor and step.
__device__ __forceinline__ uint32_t round_from(int64_t e, uint32_t key) {
    return (uint32_t)e ^ (key + 0x9e3779b9u * (uint32_t)(e >> 32));
}
__device__ __forceinline__ uint32_t round_bits(uint32_t key, int64_t e) { return mix(round_from(e, key)) >> 12; }
// The same of value e + i, e a multiple of 8 and i below 8, by folded = x ^ (x >> 16) of e's
// x = round_from: mix begins with this, and i changes only its lowest bits.
__device__ __forceinline__ uint32_t round_bits_near(uint32_t folded, uint32_t i) {
    uint32_t x = (folded ^ i) * 0x85ebca6bu;
    x = (x ^ (x >> 13)) * 0xc2b2ae35u;
    return (x ^ (x >> 16)) >> 12;
}

// ------------------------------------------------------------------- norm --

struct Summand {
    const void* p;
    int64_t n;             // values, or with `count`: rows at most
    const int64_t* count;  // rows in use, NULL = a dense tensor
    int first, d, dtype;   // its first chunk, row width
};
template <int N>
struct Summands {
    Summand of[N];
};

struct Hyper {
    double lr, b1, b2, eps, ln_b1, ln_b2, grad_scale, max_norm;
    const double *lr_at, *grad_scale_at;  // on the device, NULL = the numbers above
    int64_t* step;
    uint32_t seed;
};

// What a call keeps on the device between its launches, and the count of finished blocks, which is
// 0 between launches.
struct Work {
    unsigned done;
    double factor;  // of every gradient
    double part[kNormBlocks];
};

// The block that finishes last: on every thread whether this is it; the count is left at 0.
__device__ __forceinline__ bool last_block(unsigned* done) {
    __shared__ unsigned last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(done, 1u) == gridDim.x - 1 ? 1u : 0u;
        if (last) *done = 0;
    }
    __syncthreads();
    if (!last) return false;
    __threadfence();
    return true;
}

// Squares are added in 32 bits over a thread's values of a chunk, and in 64 bits from
// there; values whose squares leave the 32-bit range are squared in 64. `bits`: not 0 where
// any value is not.
template <class A>
__device__ __forceinline__ double square_sum(const A (&v)[kPer], unsigned bits) {
    A s = A(0);
#pragma unroll
    for (int j = 0; j < kPer; ++j) s += v[j] * v[j];
    if (!IsF64<A>::value && (!(s < A(1e37)) || (s < A(1e-25) && bits != 0))) {
        double w = 0.0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) w += (double)v[j] * (double)v[j];
        return w;
    }
    return (double)s;
}
// A thread's share of the values [base, n) of a chunk of R kChunk: R times eight neighbouring ones,
// all on their way at once, where the array begins at a vector and the chunk is whole; else every
// kNT-th.
template <class G, int R>
__device__ __forceinline__ double square_sum(const G* g, int64_t n, int64_t base) {
    using A = typename Arith<G>::type;
    constexpr int V = Pack<G>::N, W = kPer / V;
    double sum = 0.0;
    if ((uintptr_t)g % 16 == 0 && base + R * kChunk <= n) {
        uint4 r[R][W];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int q = 0; q < W; ++q) r[i][q] = *reinterpret_cast<const uint4*>(g + base + i * kChunk + threadIdx.x * kPer + q * V);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            A v[kPer];
            unsigned bits = 0;
#pragma unroll
            for (int q = 0; q < W; ++q) {
                A p[V];
                Pack<G>::unpack(r[i][q], p);
                bits |= r[i][q].x | r[i][q].y | r[i][q].z | r[i][q].w;
#pragma unroll
                for (int c = 0; c < V; ++c) v[q * V + c] = p[c];
            }
            sum += square_sum(v, bits);
        }
        return sum;
    }
    for (int64_t b = base; b < n && b < base + R * kChunk; b += kChunk) {
        A v[kPer];
        unsigned bits = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int64_t e = b + threadIdx.x + j * kNT;
            v[j] = e < n ? widen<A>(g[e]) : A(0);
            bits |= v[j] != A(0);
        }
        sum += square_sum(v, bits);
    }
    return sum;
}

// Sums of squares by block, R chunks at a time where there are many, bound by HBM (184 M float32
// values 110 us, 6.7 TB/s; bfloat16 60 us, 97 with R = 1); the last block of the last launch (`finish`) adds them, in
// block order, to the norm and the gradients' factor. A norm that is not finite leaves
// NaN there, and the step does nothing.
template <int N, int R>
__global__ void __launch_bounds__(kNT)
    norm_kernel(const __grid_constant__ Summands<N> list, int n_of, int64_t chunks, Work* work,
                int part_at, bool finish, const __grid_constant__ Hyper h, int norm64, void* norm) {
    __shared__ double sm[kNT / 32];
    after_previous();
    double a = 0.0;
    int i = 0;
    for (int64_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        while (i + 1 < n_of && c >= list.of[i + 1].first) ++i;
        const Summand& s = list.of[i];
        int64_t n = s.n;
        if (s.count) {
            const int64_t used = *s.count;
            n = (used < 0 ? 0 : used > n ? n : used) * s.d;
        }
        const int64_t base = (c - s.first) * (R * kChunk);
        if (base >= n) continue;
        if (s.dtype == MFM_DTYPE_F64)
            a += square_sum<double, R>((const double*)s.p, n, base);
        else if (s.dtype == MFM_DTYPE_F32)
            a += square_sum<float, R>((const float*)s.p, n, base);
        else if (s.dtype == MFM_DTYPE_BF16)
            a += square_sum<__nv_bfloat16, R>((const __nv_bfloat16*)s.p, n, base);
        else
            a += square_sum<__half, R>((const __half*)s.p, n, base);
    }
    a = block_sum(a, sm);
    if (threadIdx.x == 0) work->part[part_at + blockIdx.x] = a;
    if (!last_block(&work->done) || !finish) return;
    double t = 0.0;
    for (int b = threadIdx.x; b < part_at + (int)gridDim.x; b += kNT) t += __ldcg(work->part + b);
    t = block_sum(t, sm);
    if (threadIdx.x != 0) return;
    const double scale = h.grad_scale_at ? *h.grad_scale_at : h.grad_scale;
    const double whole = sqrt(t) * fabs(scale);
    if (norm64)
        *(double*)norm = whole;
    else
        *(float*)norm = (float)whole;
    // whole = 0: nothing to scale
    work->factor = !isfinite(whole) ? (double)NAN : whole > h.max_norm ? scale * (h.max_norm / whole) : scale;
}

// ------------------------------------------------------------------- step --

// What every value of a launch shares.
template <class A>
struct Shared {
    A lr, b1, c1, b2, c2, eps, scale;  // c = 1 - b
    A i1, i2;                          // lr / (1 - b1^t), 1 / (1 - b2^t)
    A root_scale, unscale;             // i2 comes times the first, the root times the second
    __device__ __forceinline__ void corrections(A one, A two) {
        i1 = lr * one;
        i2 = two * root_scale;
    }
};

// 1 / (sqrt(b) + eps), in 32 bits off by at most 5 units of 2^-24 of itself (root 2, sum 1,
// reciprocal 2: the approximate forms of one instruction; the denominator is at least eps, a
// normal number). A root flushes what is below 2^-126 to 0, which an eps of 1e-11 or more
// does not notice; beside a smaller one b comes 2^24 times as large (then a move is 0 from
// b = 2^104 on).
__device__ __forceinline__ float over_root(float b, float eps, float unscale) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(b));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(r * unscale + eps));
    return r;
}
__device__ __forceinline__ double over_root(double b, double eps, double) { return 1.0 / (sqrt(b) + eps); }

template <class A>
__device__ __forceinline__ A step_one(const Shared<A>& k, A p, A g, A& m, A& v, A decay) {
    g *= k.scale;
    m = k.b1 * m + k.c1 * g;
    v = k.b2 * v + k.c2 * (g * g);
    // lr wd p by itself: 1 - lr wd would lose most of its digits
    return (p - decay * p) - (m * k.i1) * over_root(v * k.i2, k.eps, k.unscale);
}

// 1 / (1 - b^t) by t log b
__device__ __forceinline__ float inverse_left(double t_ln_b, float) { return 1.0f / -expm1f((float)t_ln_b); }
__device__ __forceinline__ double inverse_left(double t_ln_b, double) { return 1.0 / -expm1(t_ln_b); }

template <class A>
__device__ __forceinline__ Shared<A> shared_of(const Hyper& h, const Work* work, bool clipped, double& lr) {
    Shared<A> k;
    lr = h.lr_at ? *h.lr_at : h.lr;
    k.lr = (A)lr;
    k.b1 = (A)h.b1;
    k.c1 = (A)(1.0 - h.b1);
    k.b2 = (A)h.b2;
    k.c2 = (A)(1.0 - h.b2);
    k.eps = (A)h.eps;
    k.scale = (A)(clipped ? work->factor : h.grad_scale_at ? *h.grad_scale_at : h.grad_scale);
    const bool small = !IsF64<A>::value && h.eps < 1e-11;
    k.root_scale = small ? A(16777216) : A(1);
    k.unscale = small ? A(1.0 / 4096) : A(1);
    return k;
}

struct Tensor {
    void* param;
    const void* grad;
    void *m, *v;
    uint8_t *m_exp, *v_exp;
    float* master;
    int64_t n;  // values
    double decay;
    int first, number;  // its first chunk, its place in the caller's list
};
template <int N>
struct Tensors {
    Tensor of[N];
};

// One value of the arrays of a tensor or a table row. e: in the moments; ep: in p.
template <class P, class G, class A, bool MASTER, int BITS>
struct Values {
    A p, g, m, v;
    __device__ __forceinline__ void load(const P* param, const G* grad, const void* ms, const void* vs,
                                         const float* master, int64_t ep, int64_t eg, int64_t e) {
        p = MASTER ? (A)master[e] : widen<A>(param[ep]);
        g = widen<A>(grad[eg]);
        if constexpr (BITS != 8) {
            m = ((const A*)ms)[e];
            v = ((const A*)vs)[e];
        }
    }
    __device__ __forceinline__ void store(P* param, void* ms, void* vs, float* master, int64_t ep, int64_t e) const {
        if (MASTER) master[e] = (float)p;
        param[ep] = narrow<P>(p);
        if constexpr (BITS != 8) {
            ((A*)ms)[e] = m;
            ((A*)vs)[e] = v;
        }
    }
};

// Lane `lane` of 32 neighbouring values: moments read from codes and written to them, the
// whole warp at once (a lane without a value takes part with 0).
__device__ __forceinline__ void moments_of(const uint8_t* m, const uint8_t* v, unsigned xm, unsigned xv, int64_t e,
                                           bool in, float& fm, float& fv) {
    fm = in ? MCode::value(m[e], xm) : 0.0f;
    fv = in ? VCode::value(v[e], xv) : 0.0f;
}
__device__ __forceinline__ void moments_to(uint8_t* m, uint8_t* v, uint8_t* m_exp, uint8_t* v_exp, int64_t block,
                                           int64_t e, bool in, float fm, float fv, uint32_t random) {
    const unsigned xm = MCode::shared(__reduce_max_sync(0xffffffffu, __float_as_uint(fm) & 0x7fffffffu));
    const unsigned xv = VCode::shared(__reduce_max_sync(0xffffffffu, __float_as_uint(fv) & 0x7fffffffu));
    if (in) {
        m[e] = (uint8_t)MCode::code(fm, kHalfStep, xm);
        v[e] = (uint8_t)VCode::code(fv, random, xv);
    }
    if ((threadIdx.x & 31) == 0) {
        m_exp[block] = (uint8_t)xm;
        v_exp[block] = (uint8_t)xv;
    }
}

// Eight neighbouring values as one access of 16 or 32 bytes.
template <class T>
struct Eight;
template <>
struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p) {
        asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "l"(p)
                     : "memory");
    }
    __device__ __forceinline__ float get(int i) const { return v[i]; }
    static __device__ __forceinline__ void store(float* p, const float (&o)[8]) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(o[0]), "f"(o[1]), "f"(o[2]),
                     "f"(o[3]), "f"(o[4]), "f"(o[5]), "f"(o[6]), "f"(o[7])
                     : "memory");
    }
};
template <class H>
struct EightHalves {
    uint4 r;
    __device__ __forceinline__ void load(const H* p) { r = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ float get(int i) const {
        float v[8];
        Pack<H>::unpack(r, v);
        return v[i];
    }
    static __device__ __forceinline__ void store(H* p, const float (&o)[8]) {
        *reinterpret_cast<uint4*>(p) = Pack<H>::pack(o);
    }
};
template <>
struct Eight<__nv_bfloat16> : EightHalves<__nv_bfloat16> {};
template <>
struct Eight<__half> : EightHalves<__half> {};

// Where eight neighbouring values lie. Bases that a block shares and offsets of 32 bits make
// addresses of one instruction.
template <class P, class G>
struct At {
    P* param;
    const G* grad;
    char *m, *v;  // float32, or codes
    uint8_t *m_exp, *v_exp;
    float* master;
    // of the tensor's or row's value `e`, a multiple of 32 for a dense tensor; p: of the parameter
    template <int BITS, class S>
    static __device__ __forceinline__ At of(const S& s, int64_t ep, int64_t eg, int64_t e) {
        constexpr int size = BITS == 8 ? 1 : 4;
        return At{(P*)s.param + ep, (const G*)s.grad + eg, (char*)s.m + e * size, (char*)s.v + e * size,
                  s.m_exp + e / 32, s.v_exp + e / 32, s.master + e};
    }
};

template <class P, class G, bool MASTER, int BITS>
struct Step8 {
    Eight<P> p;
    Eight<G> g;
    Eight<float> w, fm, fv;
    uint2 cm, cv;
    uint8_t xm, xv;
    // Whole warps take a step: four lanes share a block of 8-bit moments. A lane without
    // values (`in` false) takes part with those at offset 0, and stores nothing.
    __device__ __forceinline__ void load(const At<P, G>& at, unsigned off) {
        if (MASTER)
            w.load(at.master + off);
        else
            p.load(at.param + off);
        g.load(at.grad + off);
        if (BITS == 8) {
            cm = *reinterpret_cast<const uint2*>(at.m + off);
            cv = *reinterpret_cast<const uint2*>(at.v + off);
            xm = at.m_exp[off / 32];
            xv = at.v_exp[off / 32];
        } else {
            fm.load((const float*)at.m + off);
            fv.load((const float*)at.v + off);
        }
    }
    // e: the first value's place in the tensor, which its random bits go by
    __device__ __forceinline__ void step(const Shared<float>& k, float decay, const At<P, G>& at, unsigned off, int64_t e,
                                         uint32_t key, bool in) {
        float out[8], m[8], v[8];
        if (BITS == 8) {
            const unsigned was_m = (unsigned)xm * 0x00800080u, was_v = (unsigned)xv * 0x00800080u;
            four_of<true>(cm.x, was_m, m);
            four_of<true>(cm.y, was_m, m + 4);
            four_of<false>(cv.x, was_v, v);
            four_of<false>(cv.y, was_v, v + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m[i] = fm.get(i);
                v[i] = fv.get(i);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = step_one(k, MASTER ? w.get(i) : p.get(i), g.get(i), m[i], v[i], decay);
        unsigned cms[2], cvs[2], x_m = 0, x_v = 0;
        if (BITS == 8) {
            // twice m's bits: without the sign (v has none, or is NaN)
            unsigned twice[8], top_m = 0, top_v = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) twice[i] = __float_as_uint(m[i]) * 2;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                top_m = __vimax3_u32(top_m, twice[i], twice[i + 1]);
                top_v = __vimax3_u32(top_v, __float_as_uint(v[i]), __float_as_uint(v[i + 1]));
            }
            top_m = in ? top_m / 2 : 0;
            top_v = in ? top_v & 0x7fffffffu : 0;
#pragma unroll
            for (int o = 1; o < 4; o *= 2) {
                top_m = max(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
                top_v = max(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
            }
            x_m = MCode::shared(top_m);
            x_v = VCode::shared(top_v);
            // up to 61440 in m: twice a number's distance from the base then fits in 31 bits
            if (top_m < 0x47700000u && top_v < 0x7f700000u) {
                const uint32_t from = round_from(e, key), folded = from ^ (from >> 16);
                // No number is more than its code's most above the base, which the largest one gave;
                // m: 0 for what is below it, v: 1, but 0 stays 0 (other values are no less than 1).
                const unsigned add_m = 2 * (kHalfStep - (x_m << 23)), less_v = x_v << 23;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    unsigned km = 0, kv = 0;
#pragma unroll
                    for (int i = 3; i >= 0; --i) {
                        const unsigned bv = __float_as_uint(v[4 * w + i]), random = round_bits_near(folded, 4 * w + i);
                        km = km * 256 + (unsigned)(max((int)(twice[4 * w + i] + add_m), 0) >> 21);
                        kv = kv * 256 + min((unsigned)max((int)(bv + random - less_v), 1 << 20) >> 20, bv);
                    }
                    const unsigned low = __byte_perm(__float_as_uint(m[4 * w]), __float_as_uint(m[4 * w + 1]), 0x0073);
                    const unsigned high = __byte_perm(__float_as_uint(m[4 * w + 2]), __float_as_uint(m[4 * w + 3]), 0x0073);
                    cms[w] = km | (__byte_perm(low, high, 0x5410) & 0x80808080u);
                    cvs[w] = kv;
                }
            } else {  // an infinity, a NaN, or a value that would round to one, or a large m
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    cms[w] = cvs[w] = 0;
                    for (int i = 0; i < 4; ++i) {
                        cms[w] |= MCode::code(m[4 * w + i], kHalfStep, x_m) << (8 * i);
                        cvs[w] |= VCode::code(v[4 * w + i], round_bits(key, e + 4 * w + i), x_v) << (8 * i);
                    }
                }
            }
        }
        if (!in) return;
        if (MASTER) Eight<float>::store(at.master + off, out);
        Eight<P>::store(at.param + off, out);
        if (BITS == 8) {
            *reinterpret_cast<uint2*>(at.m + off) = make_uint2(cms[0], cms[1]);
            *reinterpret_cast<uint2*>(at.v + off) = make_uint2(cvs[0], cvs[1]);
            if (off % 32 == 0) {
                at.m_exp[off / 32] = (uint8_t)x_m;
                at.v_exp[off / 32] = (uint8_t)x_v;
            }
        } else {
            Eight<float>::store((float*)at.m + off, m);
            Eight<float>::store((float*)at.v + off, v);
        }
    }
};

// One value: of p at `ep`, of the gradient at `eg`, else at `e`. Whole warps call it: 32
// lanes share a block of 8-bit moments.
template <class P, class G, class A, bool MASTER, int BITS>
__device__ __forceinline__ void step_value(const Shared<A>& k, A decay, P* param, const G* grad, void* ms, void* vs,
                                           uint8_t* m_exp, uint8_t* v_exp, float* master, int64_t ep, int64_t eg,
                                           int64_t e, int64_t at, uint32_t key, bool in) {
    Values<P, G, A, MASTER, BITS> v;
    if (in) v.load(param, grad, ms, vs, master, ep, eg, e);
    if constexpr (BITS == 8) {
        const int64_t block = (e - (threadIdx.x & 31)) / 32;
        float fm, fv;
        moments_of((const uint8_t*)ms, (const uint8_t*)vs, m_exp[block], v_exp[block], e, in, fm, fv);
        if (in) v.p = step_one(k, v.p, v.g, fm, fv, decay);
        moments_to((uint8_t*)ms, (uint8_t*)vs, m_exp, v_exp, block, e, in, fm, fv, round_bits(key, at));
    } else if (in) {
        v.p = step_one(k, v.p, v.g, v.m, v.v, decay);
    }
    if (in) v.store(param, ms, vs, master, ep, e);
}

// Dense tensors of one kind. EIGHTS: they begin at whole vectors, and a thread takes eight
// neighbouring values, up to the last whole block of 32; elsewhere a warp's 32 lanes
// take 32 neighbouring values kPer times. Chunks are walked from the last to the first: the
// norm's pass left the last gradients in L2.
template <class P, class G, bool MASTER, int BITS, bool EIGHTS, int N>
__global__ void __launch_bounds__(kNT, IsF64<typename Arith<P>::type>::value ? 2 : 3)
    adamw_kernel(const __grid_constant__ Tensors<N> list, int n_of, int64_t chunks, int rounds, Work* work, bool clipped,
                 bool count, const __grid_constant__ Hyper h) {
    using A = typename Arith<P>::type;
    __shared__ double left[2];
    after_previous();
    const int64_t t = *h.step + 1;
    if (threadIdx.x == 0) left[0] = -1.0 / expm1((double)t * h.ln_b1);
    if (threadIdx.x == 32) left[1] = -1.0 / expm1((double)t * h.ln_b2);
    __syncthreads();
    double lr;
    Shared<A> k = shared_of<A>(h, work, clipped, lr);
    k.corrections((A)left[0], (A)left[1]);
    if (clipped && isnan(work->factor)) {
        last_block(&work->done);
        return;
    }
    int i = n_of - 1;
    if constexpr (EIGHTS) {
        // A thread's eights of a chunk, kChunk apart. 8-bit moments are bound by instructions:
        // there the loads of one are under way while the one before it is worked on (184 M values:
        // 532 us against 577 without). The others wait for memory whatever they do, and need
        // the registers for blocks.
        constexpr bool AHEAD = BITS == 8;
        const int64_t size = kChunk * rounds;
        for (int64_t c = chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
            while (c < list.of[i].first) --i;
            const Tensor& s = list.of[i];
            const A decay = (A)(lr * s.decay);
            const uint32_t key = mix(mix(mix(h.seed) + (uint32_t)s.number) + (uint32_t)t);
            const int64_t base = (c - s.first) * size, whole = s.n / 32 * 32 - base;
            // values of the chunk that vectors take: whole blocks of 32
            const unsigned n = (unsigned)(whole < 0 ? 0 : whole > size ? size : whole);
            const At<P, G> at = At<P, G>::template of<BITS>(s, base, base, base);
            unsigned off = threadIdx.x * kPer;
            Step8<P, G, MASTER, BITS> now, next;
            if (AHEAD && n) now.load(at, off < n ? off : 0);
#pragma unroll 1
            for (unsigned done = 0; done < n; done += kChunk, off += kChunk) {
                const unsigned coming = off + kChunk;
                if (!AHEAD)
                    now.load(at, off < n ? off : 0);
                else if (done + kChunk < n)
                    next.load(at, coming < n ? coming : 0);
                now.step(k, decay, at, off, base + off, key, off < n);
                if (AHEAD) now = next;
            }
            if (base + size > s.n && s.n % 32 && threadIdx.x < 32) {  // the tensor's last values
                const int64_t q = s.n / 32 * 32 + threadIdx.x;
                step_value<P, G, A, MASTER, BITS>(k, decay, (P*)s.param, (const G*)s.grad, s.m, s.v, s.m_exp, s.v_exp, s.master, q, q, q, q, key, q < s.n);
            }
        }
    } else {
        for (int64_t c = chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
            while (c < list.of[i].first) --i;
            const Tensor& s = list.of[i];
            P* param = (P*)s.param;
            const G* grad = (const G*)s.grad;
            const A decay = (A)(lr * s.decay);
            const uint32_t key = mix(mix(mix(h.seed) + (uint32_t)s.number) + (uint32_t)t);
            const int64_t e = (c - s.first) * kChunk + threadIdx.x;
            if constexpr (BITS == 8) {
                for (int j = 0; j < kPer; ++j) {
                    const int64_t q = e + j * kNT;
                    if (q - (threadIdx.x & 31) < s.n)  // uniform over the warp
                        step_value<P, G, A, MASTER, BITS>(k, decay, param, grad, s.m, s.v, s.m_exp, s.v_exp, s.master, q, q, q, q, key, q < s.n);
                }
            } else {
                Values<P, G, A, MASTER, BITS> v[kPer];
#pragma unroll
                for (int j = 0; j < kPer; ++j)
                    if (e + j * kNT < s.n) v[j].load(param + e, grad + e, (A*)s.m + e, (A*)s.v + e, s.master + e, j * kNT, j * kNT, j * kNT);
#pragma unroll
                for (int j = 0; j < kPer; ++j)
                    if (e + j * kNT < s.n) {
                        v[j].p = step_one(k, v[j].p, v[j].g, v[j].m, v[j].v, decay);
                        v[j].store(param + e, (A*)s.m + e, (A*)s.v + e, s.master + e, j * kNT, j * kNT);
                    }
            }
        }
    }
    // every block has read the step count when the last one finishes
    if (last_block(&work->done) && count && threadIdx.x == 0) *h.step = t;
}

// A table by touched rows.
struct Table {
    void* param;
    const void* grad;
    void *m, *v;
    uint8_t *m_exp, *v_exp;
    float* master;
    const void* keys;
    const int64_t* count;
    int32_t* row_steps;
    int64_t n_rows, d, ld, pitch, n_keys;
    double decay;
    int number;
};

// The row of slot `slot`, -1 for one that is left out: a key outside the table, or not above
// the one before it.
template <class K>
__device__ __forceinline__ int64_t row_of(const Table& s, int64_t slot, int64_t used) {
    if (slot >= used) return -1;
    const K* keys = (const K*)s.keys;
    const int64_t r = (int64_t)keys[slot], before = slot > 0 ? (int64_t)keys[slot - 1] : -1;
    return r < s.n_rows && r > before && r >= 0 ? r : -1;
}

// L lanes a row, a value a lane or (EIGHTS) eight neighbouring ones: gathers of a few sectors a
// row and array, bound by their latency where a batch touches few rows (55000 x 16 float32: 7.5 us
// of kernel against 3.9 us of bytes; 14500 x 1024 bfloat16 48 us with 8-bit moments against
// 27.5, 63 us with float32 ones against 54.5).
template <class P, class G, bool MASTER, int BITS, class K, bool EIGHTS, int L>
__global__ void __launch_bounds__(kNT, EIGHTS ? 3 : 4)
    adamw_rows_kernel(const __grid_constant__ Table s, Work* work, bool clipped, bool count,
                      const __grid_constant__ Hyper h) {
    using A = typename Arith<P>::type;
    after_previous();
    const int64_t t_all = *h.step + 1;
    double lr;
    Shared<A> k = shared_of<A>(h, work, clipped, lr);
    if (clipped && isnan(work->factor)) {
        last_block(&work->done);
        return;
    }
    P* param = (P*)s.param;
    const G* grad = (const G*)s.grad;
    const A decay = (A)(lr * s.decay);
    const uint32_t key32 = mix(mix(mix(h.seed) + (uint32_t)s.number) + (uint32_t)t_all);
    const int lane = threadIdx.x % L;
    int64_t used = *s.count;
    used = used < 0 ? 0 : used > s.n_keys ? s.n_keys : used;
    const int64_t groups = (int64_t)gridDim.x * (kNT / L);
    // uniform over the warp, whose rows go round together
    for (int64_t at = ((int64_t)blockIdx.x * kNT + threadIdx.x) / 32 * (32 / L); at < used; at += groups) {
        const int64_t slot = at + threadIdx.x % 32 / L;
        const int64_t r = row_of<K>(s, slot, used);
        int t = 0;
        if (r >= 0 && lane == 0) {
            t = s.row_steps[r] + 1;
            s.row_steps[r] = t;
        }
        t = __shfl_sync(0xffffffffu, t, 0, L);
        k.corrections(inverse_left((double)t * h.ln_b1, A(0)), inverse_left((double)t * h.ln_b2, A(0)));
        if constexpr (EIGHTS) {
            for (int64_t c0 = 0; c0 < s.pitch; c0 += L * 8) {
                const unsigned c = (unsigned)c0 + lane * 8;
                const bool in = r >= 0 && c < s.d;
                Step8<P, G, MASTER, BITS> now;
                const At<P, G> at = r < 0 ? At<P, G>::template of<BITS>(s, 0, 0, 0)
                                          : At<P, G>::template of<BITS>(s, r * s.ld, slot * s.d, r * s.pitch);
                now.load(at, in ? c : 0);
                now.step(k, decay, at, c, r * s.d + c, key32, in);
            }
        } else {
            for (int64_t c0 = 0; c0 < s.d; c0 += L) {
                const int64_t c = c0 + lane;
                if (BITS == 8 && r < 0) break;  // L = 32: uniform over the warp
                step_value<P, G, A, MASTER, BITS>(k, decay, param, grad, s.m, s.v, s.m_exp, s.v_exp, s.master, r * s.ld + c,
                                                  slot * s.d + c, r * s.pitch + c, r * s.d + c, key32, r >= 0 && c < s.d);
            }
        }
    }
    if (last_block(&work->done) && count && threadIdx.x == 0) *h.step = t_all;
}

// A step without a gradient still counts.
__global__ void count_kernel(Work* work, bool clipped, const __grid_constant__ Hyper h) {
    after_previous();
    if (threadIdx.x == 0 && (!clipped || !isnan(work->factor))) *h.step += 1;
}

// Codes as the values that they stand for (one code a time takes 235 us for both moments of
// 184 M values, two 208 us).
template <bool SIGNED>
__device__ __forceinline__ void decode(const uint8_t* code, const uint8_t* shared, int64_t n, unsigned short* out, bool whole,
                                       int64_t first, int64_t step) {
    const int64_t eights = whole ? n / 8 : 0;
    for (int64_t i = first; i < eights; i += step) {
        const uint2 c = *reinterpret_cast<const uint2*>(code + 8 * i);
        const unsigned base = (unsigned)shared[i / 4] * 0x00800080u;
        uint4 w;
        w.x = halves_of<SIGNED>(__byte_perm(c.x, 0, 0x4140), base);
        w.y = halves_of<SIGNED>(__byte_perm(c.x, 0, 0x4342), base);
        w.z = halves_of<SIGNED>(__byte_perm(c.y, 0, 0x4140), base);
        w.w = halves_of<SIGNED>(__byte_perm(c.y, 0, 0x4342), base);
        *reinterpret_cast<uint4*>(out + 8 * i) = w;
    }
    for (int64_t e = eights * 8 + first; e < n; e += step)
        out[e] = (unsigned short)halves_of<SIGNED>(code[e], (unsigned)shared[e / 32] * 128);
}
__global__ void __launch_bounds__(kNT)
    moments_kernel(const uint8_t* __restrict__ code, const uint8_t* __restrict__ shared, int64_t n,
                   unsigned short* __restrict__ out, bool is_signed, bool whole) {
    const int64_t step = (int64_t)gridDim.x * kNT, first = (int64_t)blockIdx.x * kNT + threadIdx.x;
    if (is_signed)
        decode<true>(code, shared, n, out, whole, first, step);
    else
        decode<false>(code, shared, n, out, whole, first, step);
}

// ------------------------------------------------------------- launchers --

size_t size_of(int dtype) { return dtype == MFM_DTYPE_F64 ? 8 : dtype == MFM_DTYPE_F32 ? 4 : 2; }

void check_tensor(const mfm_adamw_tensor& t, int64_t i, int bits) {
    auto bad = [&](const char* what) { fail(MFM_ERR_INVALID, fmt("tensor %lld: %s", (long long)i, what)); };
    if (t.dtype != MFM_DTYPE_F64 && t.dtype != MFM_DTYPE_F32 && t.dtype != MFM_DTYPE_BF16 && t.dtype != MFM_DTYPE_F16)
        fail(MFM_ERR_INVALID, fmt("tensor %lld: unknown dtype %d", (long long)i, t.dtype));
    const bool half = t.dtype == MFM_DTYPE_BF16 || t.dtype == MFM_DTYPE_F16;
    if (t.grad_dtype != t.dtype && !(half && t.grad_dtype == MFM_DTYPE_F32))
        bad("grad_dtype must be dtype, or MFM_DTYPE_F32 for 16-bit parameters");
    if (t.n_rows < 0 || t.d < 0) bad("n_rows and d must be >= 0");
    if (t.master && !half) bad("master weights are for 16-bit parameters");
    if (bits == 8 && t.dtype == MFM_DTYPE_F64) bad("8-bit moments are for parameters of at most 32 bits");
    const bool rows = t.keys != nullptr;
    if (!rows && t.n_rows != 1) bad("a tensor without keys has n_rows = 1");
    if (rows && (!t.count || !t.row_steps)) bad("keys need count and row_steps");
    if (rows && (t.n_keys < 0 || t.n_rows > INT32_MAX || t.n_keys > INT32_MAX || t.d > INT32_MAX))
        bad("n_rows, n_keys and d of a table must be in [0, 2^31)");
    if (rows && t.ld < t.d) bad("row pitch below d");
    if (t.d > 0 && t.n_rows > 0 && (!t.param || !t.m || !t.v || (bits == 8 && (!t.m_exp || !t.v_exp))))
        bad("param, m and v (and their exponents in 8 bits) must be provided");
    const size_t s = size_of(t.dtype), wide = bits == 8 ? 1 : t.dtype == MFM_DTYPE_F64 ? 8 : 4;
    if ((uintptr_t)t.param % s || (uintptr_t)t.grad % size_of(t.grad_dtype) || (uintptr_t)t.m % wide ||
        (uintptr_t)t.v % wide || (uintptr_t)t.master % 4 || (uintptr_t)t.keys % (t.keys64 ? 8 : 4))
        bad("an array does not begin at a multiple of its element's size");
}

// Whether eight neighbouring values are whole vectors in every array: they begin at them, and
// rows at multiples of `row` values (0: no rows).
bool eights(const mfm_adamw_tensor& t, int bits, int64_t row) {
    if (t.dtype == MFM_DTYPE_F64 || row % 8) return false;
    const uintptr_t p = t.dtype == MFM_DTYPE_F32 ? 32 : 16, g = t.grad_dtype == MFM_DTYPE_F32 ? 32 : 16;
    return (uintptr_t)t.param % p == 0 && (uintptr_t)t.grad % g == 0 && ((uintptr_t)t.m | (uintptr_t)t.v) % (bits == 8 ? 8 : 32) == 0 &&
           (uintptr_t)t.master % 32 == 0;
}

template <class F>
void with_kind(const mfm_adamw_tensor& t, int bits, F&& f) {
    using std::integral_constant;
    auto state = [&](auto* p, auto* g, auto master) {
        if (bits == 8)
            f(p, g, master, integral_constant<int, 8>{});
        else
            f(p, g, master, integral_constant<int, 32>{});
    };
    auto half = [&](auto* p) {
        auto grad = [&](auto* g) {
            if (t.master)
                state(p, g, std::true_type{});
            else
                state(p, g, std::false_type{});
        };
        if (t.grad_dtype == MFM_DTYPE_F32)
            grad((float*)nullptr);
        else
            grad(p);
    };
    switch (t.dtype) {
        case MFM_DTYPE_F64: f((double*)nullptr, (double*)nullptr, std::false_type{}, integral_constant<int, 32>{}); break;
        case MFM_DTYPE_F32: state((float*)nullptr, (float*)nullptr, std::false_type{}); break;
        case MFM_DTYPE_BF16: half((__nv_bfloat16*)nullptr); break;
        default: half((__half*)nullptr); break;
    }
}

int kind_of(const mfm_adamw_tensor& t, int bits) {
    return ((t.dtype * 8 + t.grad_dtype) * 2 + (t.master ? 1 : 0)) * 2 + (eights(t, bits, 0) ? 1 : 0);
}

template <class X>
using Bare = std::remove_pointer_t<X>;

// Blocks of a persistent kernel: one wave.
template <auto Kernel>
unsigned wave(int device, int64_t most) {
    static int per_sm[64];  // of this kernel: the answer stays
    int per = per_sm[device & 63];
    if (per == 0) {
        MFM_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, Kernel, kNT, 0), "occupancy");
        per_sm[device & 63] = per = std::max(per, 1);
    }
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)sm_count(device) * per));
}

}  // namespace
}  // namespace mfm

using namespace mfm;

extern "C" int64_t mfm_adamw_workspace_bytes(void) { return (int64_t)sizeof(Work); }

extern "C" int mfm_adamw_step_device(int device, const mfm_adamw_tensor* tensors, int64_t n_tensors,
                                     const mfm_adamw* hyper, int64_t* step, void* norm, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    return guarded([&] {
        if (!hyper || !step || n_tensors < 0 || (n_tensors > 0 && !tensors))
            fail(MFM_ERR_INVALID, "tensors, hyper and step must be provided");
        const mfm_adamw& o = *hyper;
        if (!(o.beta_1 >= 0.0 && o.beta_1 < 1.0 && o.beta_2 >= 0.0 && o.beta_2 < 1.0))
            fail(MFM_ERR_INVALID, "beta_1 and beta_2 must be in [0, 1)");
        if (!(o.epsilon >= 1.2e-38)) fail(MFM_ERR_INVALID, "epsilon must be at least 2^-126");
        if (o.state_bits != 32 && o.state_bits != 8) fail(MFM_ERR_INVALID, "state_bits must be 32 or 8");
        const bool clipped = o.max_norm >= 0.0;
        if (std::isnan(o.max_norm)) fail(MFM_ERR_INVALID, "max_norm must be a number");
        if (clipped && !norm) fail(MFM_ERR_INVALID, "max_norm needs norm");
        if (!workspace || workspace_bytes < (int64_t)sizeof(Work))
            fail(MFM_ERR_INVALID, fmt("workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)sizeof(Work)));
        if ((uintptr_t)workspace % 256) fail(MFM_ERR_INVALID, "workspace must be 256-byte aligned");
        bool wide = false;
        for (int64_t i = 0; i < n_tensors; ++i) {
            if (tensors[i].grad) check_tensor(tensors[i], i, o.state_bits);
            wide |= tensors[i].dtype == MFM_DTYPE_F64;
        }
        DeviceGuard guard(device);
        cudaStream_t s = (cudaStream_t)stream;
        Work* work = (Work*)workspace;
        Hyper h{o.learning_rate, o.beta_1, o.beta_2, o.epsilon, std::log(o.beta_1), std::log(o.beta_2),
                o.grad_scale, o.max_norm, o.learning_rate_at, o.grad_scale_at, step, o.seed};
        // the tensors with a gradient, tables apart, and the dense ones by kind
        std::vector<int64_t> dense, tables;
        for (int64_t i = 0; i < n_tensors; ++i) {
            const mfm_adamw_tensor& t = tensors[i];
            if (!t.grad || t.d == 0 || t.n_rows == 0 || (t.keys && t.n_keys == 0)) continue;
            (t.keys ? tables : dense).push_back(i);
        }
        auto kind = [&](int64_t i) { return kind_of(tensors[i], o.state_bits); };
        std::stable_sort(dense.begin(), dense.end(), [&](int64_t a, int64_t b) { return kind(a) < kind(b); });
        bool begun = false;  // the first launch of a call waits for all before it, the others go on in a chain
        auto launch = [&](auto kernel, unsigned grid, auto&&... args) {
            if (begun)
                launch_next(kernel, grid, kNT, 0, s, args...);
            else
                kernel<<<grid, kNT, 0, s>>>(args...);
            begun = true;
        };
        auto chunk = [](int64_t at) {
            if (at > INT32_MAX) fail(MFM_ERR_UNSUPPORTED, "tensors of one kind exceed the engine's 2^42 values");
            return (int)at;
        };
        if (clipped) {
            std::vector<int64_t> all = dense;
            all.insert(all.end(), tables.begin(), tables.end());
            const size_t launches = std::max<size_t>(1, (size_t)ceil_div((int64_t)all.size(), kNormMany));
            const unsigned share = kNormBlocks / (unsigned)std::min<size_t>(launches, kNormBlocks);
            if (launches > kNormBlocks) fail(MFM_ERR_UNSUPPORTED, "more tensors than a norm is taken of");
            int part = 0;
            for (size_t l = 0; l < launches; ++l) {
                const size_t lo = l * kNormMany, hi = std::min(all.size(), lo + kNormMany);
                int64_t values = 0;
                for (size_t q = lo; q < hi; ++q) values += (tensors[all[q]].keys ? tensors[all[q]].n_keys : 1) * tensors[all[q]].d;
                auto go = [&](auto most, auto rounds) {
                    constexpr int N = decltype(most)::value, R = decltype(rounds)::value;
                    static thread_local Summands<N> list;
                    int64_t chunks = 0;
                    for (size_t q = lo; q < hi; ++q) {
                        const mfm_adamw_tensor& t = tensors[all[q]];
                        const int64_t rows = t.keys ? t.n_keys : 1;
                        list.of[q - lo] = Summand{t.grad, t.keys ? t.n_keys : t.d, t.keys ? t.count : nullptr,
                                                  chunk(chunks), t.keys ? (int)t.d : 1, t.grad_dtype};
                        chunks += ceil_div(rows * t.d, R * kChunk);
                    }
                    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>({chunks, (int64_t)share, (int64_t)sm_count(device) * 6}));
                    launch(norm_kernel<N, R>, grid, list, (int)(hi - lo), chunks, work, part, l + 1 == launches, h, wide ? 1 : 0, norm);
                    part += (int)grid;
                };
                auto size = [&](auto rounds) {
                    if (hi - lo <= kNormFew)
                        go(std::integral_constant<int, kNormFew>{}, rounds);
                    else
                        go(std::integral_constant<int, kNormMany>{}, rounds);
                };
                if (values >= 4 * 6 * kChunk * sm_count(device))
                    size(std::integral_constant<int, 4>{});
                else
                    size(std::integral_constant<int, 1>{});
            }
        }
        // dense tensors: as many of one kind as a launch carries
        for (size_t lo = 0; lo < dense.size();) {
            size_t hi = lo;
            const int one = kind(dense[lo]);
            while (hi < dense.size() && hi - lo < kMany && kind(dense[hi]) == one) ++hi;
            const bool last = hi == dense.size() && tables.empty();
            with_kind(tensors[dense[lo]], o.state_bits, [&](auto* p, auto* g, auto master, auto bits) {
                using P = Bare<decltype(p)>;
                using G = Bare<decltype(g)>;
                auto go = [&](auto most, auto aligned) {
                    constexpr int N = decltype(most)::value;
                    static thread_local Tensors<N> list;
                    // chunks of 8-bit moments are larger where there are enough of them: what a chunk
                    // costs a thread is shared by more values (184 M values: 495 us with one round,
                    // 459 with four, 444 with eight)
                    int64_t chunks = 0, values = 0;
                    for (size_t q = lo; q < hi; ++q) values += tensors[dense[q]].d;
                    const int rounds = decltype(bits)::value == 8 && decltype(aligned)::value
                                           ? (int)std::clamp<int64_t>(values / (kChunk * 12 * sm_count(device)), 1, 8)
                                           : 1;
                    for (size_t q = lo; q < hi; ++q) {
                        const mfm_adamw_tensor& t = tensors[dense[q]];
                        list.of[q - lo] = Tensor{t.param, t.grad, t.m, t.v, t.m_exp, t.v_exp, t.master, t.d,
                                                 t.weight_decay, chunk(chunks), (int)dense[q]};
                        chunks += ceil_div(t.d, kChunk * rounds);
                    }
                    constexpr auto kernel = adamw_kernel<P, G, decltype(master)::value, decltype(bits)::value, decltype(aligned)::value, N>;
                    launch(kernel, wave<kernel>(device, chunks), list, (int)(hi - lo), chunks, rounds, work, clipped, last, h);
                };
                auto size = [&](auto aligned) {
                    if (hi - lo <= kFew)
                        go(std::integral_constant<int, kFew>{}, aligned);
                    else
                        go(std::integral_constant<int, kMany>{}, aligned);
                };
                if constexpr (!IsF64<P>::value) {
                    if (one & 1) return size(std::true_type{});
                }
                size(std::false_type{});
            });
            lo = hi;
        }
        for (size_t q = 0; q < tables.size(); ++q) {
            const mfm_adamw_tensor& t = tensors[tables[q]];
            with_kind(t, o.state_bits, [&](auto* p, auto* g, auto master, auto bits) {
                using P = Bare<decltype(p)>;
                using G = Bare<decltype(g)>;
                constexpr int B = decltype(bits)::value;
                const int64_t pitch = B == 8 ? ceil_div(t.d, 32) * 32 : t.d;
                const Table table{t.param, t.grad, t.m, t.v, t.m_exp, t.v_exp, t.master, t.keys, t.count, t.row_steps,
                                  t.n_rows, t.d, t.ld, pitch, t.n_keys, t.weight_decay, (int)tables[q]};
                with_index_type(t.keys64, [&](auto* kp) {
                    using K = std::remove_const_t<Bare<decltype(kp)>>;
                    auto go = [&](auto lanes, auto aligned) {
                        constexpr int L = decltype(lanes)::value;
                        constexpr auto kernel = adamw_rows_kernel<P, G, decltype(master)::value, B, K, decltype(aligned)::value, L>;
                        launch(kernel, wave<kernel>(device, ceil_div(t.n_keys, kNT / L)), table, work, clipped,
                               q + 1 == tables.size(), h);
                    };
                    using std::integral_constant;
                    if constexpr (!IsF64<P>::value) {
                        // in 8 bits every block of 32 has its four lanes, also where a row ends in it
                        if (eights(t, o.state_bits, t.d | t.ld)) {
                            if (B != 8 && t.d <= 16) return go(integral_constant<int, B == 8 ? 4 : 2>{}, std::true_type{});
                            if (t.d <= 32) return go(integral_constant<int, 4>{}, std::true_type{});
                            if (t.d <= 128) return go(integral_constant<int, 16>{}, std::true_type{});
                            return go(integral_constant<int, 32>{}, std::true_type{});
                        }
                    }
                    if constexpr (B != 8) {
                        if (t.d <= 16) return go(integral_constant<int, 16>{}, std::false_type{});
                    }
                    go(integral_constant<int, 32>{}, std::false_type{});
                });
            });
        }
        if (dense.empty() && tables.empty()) launch(count_kernel, 1, work, clipped, h);
        MFM_CHECK_LAUNCH("AdamW step launch");
    });
}

extern "C" int mfm_adamw_moments_device(int device, int is_signed, const uint8_t* code, const uint8_t* exponent,
                                        int64_t n, void* out, void* stream) {
    return guarded([&] {
        if (n < 0) fail(MFM_ERR_INVALID, "n must be >= 0");
        if (n == 0) return;
        if (!code || !exponent || !out) fail(MFM_ERR_INVALID, "code, exponent and out must be provided");
        DeviceGuard guard(device);
        const int64_t grid = std::min<int64_t>(ceil_div(n, 8 * kNT), (int64_t)sm_count(device) * 8);
        moments_kernel<<<(unsigned)grid, kNT, 0, (cudaStream_t)stream>>>(code, exponent, n, (unsigned short*)out, is_signed != 0,
                                                                 (uintptr_t)code % 8 == 0 && (uintptr_t)out % 16 == 0);
        MFM_CHECK_LAUNCH("moments launch");
    });
}
