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

// Bytes per element of an MFM_DTYPE_* storage type.
inline size_t dtype_size(int dtype) {
    switch (dtype) {
        case MFM_DTYPE_F64: return 8;
        case MFM_DTYPE_BF16:
        case MFM_DTYPE_F16: return 2;
        default: return 4;
    }
}

// The largest vector, in elements, that divides every row start: VEC * size
// bytes at most 16, the base addresses and the row pitches (in elements)
// multiples of it.
inline bool vec_ok(const void* p, int64_t ld, size_t size, int vec) {
    return ((uintptr_t)p % (size * vec)) == 0 && (ld % vec) == 0;
}

template <class F>
void with_index_type(int ids64, F&& f) {
    if (ids64)
        f((const int64_t*)nullptr);
    else
        f((const int32_t*)nullptr);
}

}  // namespace mfm
