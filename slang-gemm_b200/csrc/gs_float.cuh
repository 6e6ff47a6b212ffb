// gs_float.cuh -- conversions between f32 and the 16- and 32-bit float types of
// the element-wise kernels, and 16-byte vectors of them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gs_internal.h"

namespace gs {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, loaded and stored as 16-byte words (N * sizeof(T) is 16 or 32).
template <typename T, int N>
struct alignas(16) Pack {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
    Pack<T, N> r;
    const uint4 *s = reinterpret_cast<const uint4 *>(p);
    uint4 *d = reinterpret_cast<uint4 *>(&r);
#pragma unroll
    for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i) d[i] = s[i];
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &r) {
    const uint4 *s = reinterpret_cast<const uint4 *>(&r);
    uint4 *d = reinterpret_cast<uint4 *>(p);
#pragma unroll
    for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i) d[i] = s[i];
}

// Calls f with a value of the element type that a GS_R_* float type names.
template <typename F>
cudaError_t with_float_type(int type, F f) {
    switch (type) {
    case GS_R_32F: return f(float{});
    case GS_R_16F: return f(__half{});
    case GS_R_16BF: return f(__nv_bfloat16{});
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace gs
