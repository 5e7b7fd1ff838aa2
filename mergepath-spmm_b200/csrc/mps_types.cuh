// Element types of the routed operators: every sum is kept in fp32, a stored 16-bit value is one rounding of it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace mps {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of T as they come from one 128-bit load
template <typename T>
struct alignas(16) Pack {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

// What a kernel of the routed operators reports (mps_routed_check): bits of a per-device status word.
enum { kStatusTimeout = 1, kStatusBadIndex = 2 };

}  // namespace mps
