// Rows of floating-point values in 8 bits with one float32 scale a row, and typed 16-byte loads and stores.
//
//   scale = max(amax * rn(1 / most), 2^-126),  code = rn(value * rn(1 / scale)),  value read back = code * scale
//
// with most = 448 (e4m3) or 127 (int8) and amax the row's largest magnitude, in float32.  The reciprocal is formed once a
// row and multiplied: a division per value would cost ten times the instructions and moves a code only where the product
// is within 2^-23 of the midpoint between two codes.  The clamp keeps the reciprocal finite, so a row of zeros (or of
// values below 2^-126 / 2) reads back as zeros.  A row that holds an infinity or a NaN has no scale: it reads back as
// NaN throughout.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace ashb {

constexpr int kFormatE4M3 = ASHB_E4M3, kFormatInt8 = ASHB_INT8;
constexpr uint32_t kInfBits = 0x7F800000u;

// Of magnitudes as unsigned words the largest is the row's, an infinity above all finite ones and a NaN above that.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

struct RowScale {
    float scale, inverse;
    __device__ __forceinline__ RowScale(uint32_t amax_bits, int format) {
        const float amax = __uint_as_float(amax_bits);
        scale = fmaxf(amax * (format == kFormatE4M3 ? 1.0f / 448.0f : 1.0f / 127.0f), 0x1p-126f);
        inverse = __frcp_rn(scale);
        if (amax_bits >= kInfBits) {
            scale = __uint_as_float(0x7FC00000u);
            inverse = 0.0f;
        }
    }
};

__device__ __forceinline__ uint32_t encode4(const float (&v)[4], float inverse, int format) {
    if (format == kFormatE4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0] * inverse, v[1] * inverse), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2] * inverse, v[3] * inverse), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) w |= ((uint32_t)__float2int_rn(v[k] * inverse) & 0xFFu) << (8 * k);
    return w;
}

__device__ __forceinline__ void decode4(uint32_t w, float scale, int format, float (&v)[4]) {
    if (format == kFormatE4M3) {
        const __half2 lo(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3));
        const __half2 hi(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
        const float2 a = __half22float2(lo), b = __half22float2(hi);
        v[0] = a.x * scale;
        v[1] = a.y * scale;
        v[2] = b.x * scale;
        v[3] = b.y * scale;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (float)(int8_t)(w >> (8 * k)) * scale;
    }
}

// ---- scalars and vectors of the three value types ------------------------------------------------------------
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive values as one access of N * sizeof(T) bytes (4, 8 or 16, aligned), or one value.
template <int BYTES>
struct Word;
template <>
struct Word<2> { using type = uint16_t; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<16> { using type = uint4; };

template <class T, int N>
__device__ __forceinline__ void load_n(const T* __restrict__ p, float (&v)[N]) {
    typename Word<N * sizeof(T)>::type w = *reinterpret_cast<const typename Word<N * sizeof(T)>::type*>(p);
    const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = to_float(t[k]);
}
template <class T, int N>
__device__ __forceinline__ void store_n(T* __restrict__ p, const float (&v)[N]) {
    typename Word<N * sizeof(T)>::type w;
    T* t = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = from_float<T>(v[k]);
    *reinterpret_cast<typename Word<N * sizeof(T)>::type*>(p) = w;
}

// The same store, first to leave L2: for what no kernel of the call reads again.
template <class T, int N>
__device__ __forceinline__ void store_n_passing(T* __restrict__ p, const float (&v)[N]) {
    typename Word<N * sizeof(T)>::type w;
    T* t = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = from_float<T>(v[k]);
    __stcs(reinterpret_cast<typename Word<N * sizeof(T)>::type*>(p), w);
}

inline int value_bytes(int dtype) { return dtype == ASHB_F32 ? 4 : 2; }
inline bool is_value_type(int dtype) { return dtype == ASHB_F32 || dtype == ASHB_F16 || dtype == ASHB_BF16; }

}  // namespace ashb
