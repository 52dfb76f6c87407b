// elem.cuh -- element types of the training-step operators (fp16, bf16, fp32): conversion to and
// from fp32, and loads / stores of up to 16 bytes a thread.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/morpho_sm100.h"

namespace morpho {

// Wait until the kernels before this one on the stream have ended and their writes are visible; every
// CTA of a kernel launched by launch_after calls it before it touches global memory.  And let the next
// such kernel be set up from here on.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements, moved as one access (N * sizeof(T) a power of two up to 16, aligned).
template <class T, int N>
struct alignas(N * sizeof(T)) Pack {
    T v[N];
};

template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, N>*>(p);
}

template <class T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& x) {
    *reinterpret_cast<Pack<T, N>*>(p) = x;
}

// One element of a tensor whose type (MORPHO_DTYPE_*) is known at run time only.
__device__ __forceinline__ float load_as_f32(const void* p, int type, int64_t i) {
    if (type == MORPHO_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (type == MORPHO_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_from_f32(void* p, int type, int64_t i, float x) {
    if (type == MORPHO_DTYPE_F32)
        static_cast<float*>(p)[i] = x;
    else if (type == MORPHO_DTYPE_F16)
        static_cast<__half*>(p)[i] = __float2half_rn(x);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

__host__ __device__ constexpr int dtype_bytes(int type) { return type == MORPHO_DTYPE_F32 ? 4 : 2; }

}  // namespace morpho
