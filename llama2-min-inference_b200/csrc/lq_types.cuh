// Activation element types of the token-scaled products and the paged cache:
// loads widen to fp32, stores round once to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace lq {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// N consecutive elements as fp32; VEC: p is aligned to N elements (at most 16 bytes)
template <int N, bool VEC, typename T>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
    if constexpr (VEC) {
        struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
            T e[N];
        };
        const Pack k = *reinterpret_cast<const Pack*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_f32(k.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_f32(p[i]);
    }
}

template <int N, bool VEC, typename T>
__device__ __forceinline__ void store_n(T* p, const float (&v)[N]) {
    if constexpr (VEC) {
        struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
            T e[N];
        };
        Pack k;
#pragma unroll
        for (int i = 0; i < N; ++i) k.e[i] = from_f32<T>(v[i]);
        *reinterpret_cast<Pack*>(p) = k;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_f32<T>(v[i]);
    }
}

// max|.| of non-negative floats by their bit patterns: infinity and NaN win
constexpr uint32_t kInfBits = 0x7F800000u;
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// rint(x / s) of a value whose scale is max|x| / 127: within +-127
__device__ __forceinline__ int quant8(float x, float s) { return max(-127, min(127, __float2int_rn(x / s))); }

__device__ __forceinline__ uint32_t pack8(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
}

}  // namespace lq
