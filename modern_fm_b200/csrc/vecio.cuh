// vecio.cuh — element types of the embedding and preference kernels: widening
// loads and once-rounding stores of vectors of float64, float32, bfloat16 and
// float16 values, and the arithmetic type each is computed in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mfm {

// Arithmetic type: float64 for float64 values, float32 for the others (sums
// and softmax statistics are never held in 16 bits).
template <class T>
struct Arith {
    using type = float;
};
template <>
struct Arith<double> {
    using type = double;
};

template <class A>
__device__ __forceinline__ A widen(double v) { return (A)v; }
template <class A>
__device__ __forceinline__ A widen(float v) { return (A)v; }
template <class A>
__device__ __forceinline__ A widen(__nv_bfloat16 v) { return (A)__bfloat162float(v); }
template <class A>
__device__ __forceinline__ A widen(__half v) { return (A)__half2float(v); }

template <class T>
__device__ __forceinline__ T narrow(double v) { return (T)v; }
template <class T>
__device__ __forceinline__ T narrow(float v) { return (T)v; }
// round to nearest even, the only rounding between the 32-bit arithmetic and
// a 16-bit result
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

template <class T>
struct IsF64 {
    static constexpr bool value = false;
};
template <>
struct IsF64<double> {
    static constexpr bool value = true;
};

// Sixteen bytes of T held as raw words: an array of 16-bit values would take a
// register each. N values; unpack widens them exactly, pack rounds them once.
template <class T>
struct Pack;
template <>
struct Pack<double> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void unpack(const uint4& r, double (&v)[2]) {
        v[0] = __hiloint2double((int)r.y, (int)r.x);
        v[1] = __hiloint2double((int)r.w, (int)r.z);
    }
    static __device__ __forceinline__ uint4 pack(const double (&v)[2]) {
        return make_uint4((unsigned)__double2loint(v[0]), (unsigned)__double2hiint(v[0]),
                          (unsigned)__double2loint(v[1]), (unsigned)__double2hiint(v[1]));
    }
    static __device__ __forceinline__ double top(const uint4& r) {
        double v[2];
        unpack(r, v);
        return fmax(v[0], v[1]);
    }
    static __device__ __forceinline__ uint4 minus_inf() { return make_uint4(0u, 0xfff00000u, 0u, 0xfff00000u); }
};
template <>
struct Pack<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& r, float (&v)[4]) {
        v[0] = __uint_as_float(r.x);
        v[1] = __uint_as_float(r.y);
        v[2] = __uint_as_float(r.z);
        v[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ float top(const uint4& r) {
        float v[4];
        unpack(r, v);
        return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
    }
    static __device__ __forceinline__ uint4 minus_inf() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
};
template <class P>
__device__ __forceinline__ P as_pair(unsigned w) { return *reinterpret_cast<const P*>(&w); }
template <class P>
__device__ __forceinline__ unsigned as_word(P p) { return *reinterpret_cast<const unsigned*>(&p); }
template <>
struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& r, float (&v)[8]) {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = as_word(__floats2bfloat162_rn(v[2 * i], v[2 * i + 1]));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // the largest value, compared as pairs: exact
    static __device__ __forceinline__ float top(const uint4& r) {
        using P = __nv_bfloat162;
        const P m = __hmax2(__hmax2(as_pair<P>(r.x), as_pair<P>(r.y)), __hmax2(as_pair<P>(r.z), as_pair<P>(r.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ uint4 minus_inf() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
};
template <>
struct Pack<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& r, float (&v)[8]) {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(as_pair<__half2>(w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = as_word(__floats2half2_rn(v[2 * i], v[2 * i + 1]));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float top(const uint4& r) {
        const __half2 m = __hmax2(__hmax2(as_pair<__half2>(r.x), as_pair<__half2>(r.y)),
                                  __hmax2(as_pair<__half2>(r.z), as_pair<__half2>(r.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ uint4 minus_inf() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
};

// The largest vector, in elements, that divides every row start: VEC * size
// bytes at most 16, the base addresses and the row pitches (in elements)
// multiples of it.
inline bool vec_ok(const void* p, int64_t ld, size_t size, int vec) {
    return ((uintptr_t)p % (size * vec)) == 0 && (ld % vec) == 0;
}

// Programmatic dependent launch: a kernel launched by launch_next may be scheduled
// while its predecessor in the stream drains. after_previous, its first
// statement, waits for the predecessor to be complete and visible, and lets the
// successor be scheduled in turn. A chain of four to eight short kernels is
// spent on launch gaps to a tenth. What the chain writes is no __restrict__ argument of a
// kernel that reads it: such a load may be issued as one of memory that is constant
// while the kernel runs, and the kernel runs before the wait.
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_previous() {
    wait_previous();
    let_next();
}

template <class... KArgs, class... Args>
void launch_next(void (*kernel)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t s,
                 Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    MFM_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...), "kernel launch");
}

// Sum over the block in a fixed order, on every thread.
__device__ __forceinline__ double block_sum(double v, double* sm) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x / 32] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) t += sm[w];
    return t;
}

template <class F>
void with_index_type(int ids64, F&& f) {
    if (ids64)
        f((const int64_t*)nullptr);
    else
        f((const int32_t*)nullptr);
}

}  // namespace mfm
