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

// N (4 or 8) consecutive elements of such a tensor from element i on, 16-byte aligned there if `whole`.
template <int N>
__device__ __forceinline__ void load_n_as_f32(const void* p, int type, int64_t i, bool whole, float* out) {
    if (!whole) {
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = load_as_f32(p, type, i + k);
    } else if (type == MORPHO_DTYPE_F32) {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + k);
            out[k] = x.x, out[k + 1] = x.y, out[k + 2] = x.z, out[k + 3] = x.w;
        }
    } else {
        uint32_t u[N / 2];
        const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
        if (N == 8) {
            const uint4 x = *reinterpret_cast<const uint4*>(q);
            u[0] = x.x, u[1] = x.y, u[N / 2 - 2] = x.z, u[N / 2 - 1] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(q);
            u[0] = x.x, u[1] = x.y;
        }
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            if (type == MORPHO_DTYPE_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
                out[2 * k] = f.x, out[2 * k + 1] = f.y;
            } else {
                out[2 * k] = __uint_as_float(u[k] << 16), out[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
            }
        }
    }
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
