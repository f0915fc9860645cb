// Activation element types of the token-scaled products and the paged cache:
// loads widen to fp32, stores round once to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

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

// the elements of a 32-bit word as fp32
template <typename T>
__device__ __forceinline__ void unpack_word(uint32_t w, float* v) {
    if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(w);
    } else if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        v[0] = f.x;
        v[1] = f.y;
    } else {
        v[0] = __uint_as_float(w << 16);
        v[1] = __uint_as_float(w & 0xFFFF0000u);
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack_word(const float* v) {
    if constexpr (sizeof(T) == 4) {
        return __float_as_uint(v[0]);
    } else if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(v[0], v[1]);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// N = 4 consecutive elements as fp32; VEC: p is aligned to 4 elements
template <int N, bool VEC, typename T>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
    static_assert(N == 4, "one vector access");
    if constexpr (VEC && sizeof(T) == 4) {
        const float4 w = *reinterpret_cast<const float4*>(p);
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else if constexpr (VEC) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        unpack_word<T>(w.x, v);
        unpack_word<T>(w.y, v + 2);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_f32(p[i]);
    }
}

template <int N, bool VEC, typename T>
__device__ __forceinline__ void store_n(T* p, const float (&v)[N]) {
    static_assert(N == 4, "one vector access");
    if constexpr (VEC && sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else if constexpr (VEC) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_word<T>(v), pack_word<T>(v + 2));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_f32<T>(v[i]);
    }
}

// max|.| of non-negative floats by their bit patterns: infinity and NaN win
constexpr uint32_t kInfBits = 0x7F800000u;
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// the low bytes of four words
__device__ __forceinline__ uint32_t pack8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Codes rint(x / s) of values whose scale s is max|x| / 127 or more, as the
// fp32 division gives them, four to a word.  x * (1 / s) is within 2^-15 of the
// quotient (three roundings of a value up to 127), so where it is further than
// 2^-13 from a half both round to the same integer; a word with one that is
// not (one in a thousand) is divided.  Adding 1.5 * 2^23 leaves the rounded
// integer in the low bits.  A scale below fp32's normal numbers has few bits (190 of its smallest
// steps over 127 round to one step), so those quotients are kept to 127.
struct Quant8 {
    float s, inv;
    bool bad;  // the scale is NaN: codes 0
    __device__ explicit Quant8(float scale) : s(scale), inv(1.0f / scale), bad(!(scale == scale)) {
        if (!(s > 1e-30f) || !(s < 1e30f)) inv = 0.0f;  // no finite inverse worth using: divide
    }
    __device__ __forceinline__ uint32_t operator()(float x0, float x1, float x2, float x3) const {
        const float x[4] = {x0, x1, x2, x3};
        uint32_t o[4];
        float near = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float t = x[e] * inv, m = t + 12582912.0f;
            near = fmaxf(near, fabsf(t - (m - 12582912.0f)));
            o[e] = __float_as_uint(m);
        }
        if (near > 0.5f - 1.220703125e-4f || inv == 0.0f) {
            if (bad) return 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (uint32_t)max(-127, min(127, __float2int_rn(x[e] / s)));
        }
        return pack8(o[0], o[1], o[2], o[3]);
    }
};

__device__ __forceinline__ int code_of(uint32_t byte) { return (int)(int8_t)byte; }

}  // namespace lq
