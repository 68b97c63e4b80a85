// Helpers of the row operators (norm, routing, grouped products): value types, 128-bit row accesses.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace fg {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_fp8_e4m3>(__nv_fp8_e4m3 v) { return static_cast<float>(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive values as one access of N * sizeof(T) bytes (4, 8 or 16; one value where N = 1).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& v) {
    *reinterpret_cast<Pack<T, N>*>(p) = v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = (w > v || w != w) ? w : v;  // a NaN wins
    }
    return v;
}

// Whether a wait of the norm, its 8-bit form or its gradient ever ran out on the current device (row_norm.cu), copied to *out on
// `s`.
int norm_stuck(cudaStream_t s, int* out);

// out[t] = sum over j of parts[position[t * k + j]], rounded once to `type` (routing.cu).
int sum_slots(const float* parts, const int32_t* position, void* out, int64_t n, int32_t k, int32_t d, int32_t type, cudaStream_t s);

inline int type_size(int32_t t) { return t == FG_F32 ? 4 : t == FG_E4M3 ? 1 : 2; }
inline bool float_type(int32_t t) { return t == FG_F32 || t == FG_F16 || t == FG_BF16; }

}  // namespace fg
