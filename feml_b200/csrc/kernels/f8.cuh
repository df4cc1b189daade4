// Device helpers of the e4m3 kernels: element types of activations, 16-byte
// vectors of them, block scales and the packing of four e4m3 values.
//
// The 8-bit form: e4m3 values q with one f32 scale s per 128 consecutive
// values of a row (or per 128 x 128 values of a weight matrix), value = q * s.
// For a block with largest magnitude a: a' = max(a, 2^-100), s = a' / 448,
// q = e4m3(y * (448 / a')) rounded to nearest even, so the largest value of a
// block is +-448. A block that holds an infinity or a NaN has no finite
// scale: s and every q of it are NaN.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "common.cuh"

namespace fbk {

constexpr int F8B = 128;              // values per scale
constexpr float kF8Max = 448.0f;      // largest e4m3 value
constexpr float kF8Floor = 7.888609052210118e-31f;  // 2^-100: least block maximum a scale is made of

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}

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

// Two neighbouring values in one 32-bit word (low half first).
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}

// A 16-byte vector of T as f32 values, and back (rounded to nearest even).
template <typename T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    static __device__ __forceinline__ void get(const uint4 &r, float (&f)[N]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) {
                f[i] = __uint_as_float(w[i]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                f[2 * i] = p.x;
                f[2 * i + 1] = p.y;
            } else {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
    static __device__ __forceinline__ uint4 put(const float (&f)[N]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4)
                w[i] = __float_as_uint(f[i]);
            else
                w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// Streamed 16-byte load (read once: not kept in L1). Coherent, so a caller
// may store to the same address afterwards.
__device__ __forceinline__ uint4 ld_stream16(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

struct alignas(32) Wide32 {
    uint4 lo, hi;
};
// The same for 32 bytes in one instruction.
__device__ __forceinline__ Wide32 ld_stream32(const void *p) {
    Wide32 v;
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.lo.x), "=r"(v.lo.y), "=r"(v.lo.z), "=r"(v.lo.w), "=r"(v.hi.x), "=r"(v.hi.y), "=r"(v.hi.z), "=r"(v.hi.w)
                 : "l"(p));
    return v;
}

// Magnitudes compare as integers: every NaN is above infinity, infinity above
// every finite value, so an integer maximum carries a NaN along.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Scale a' / 448 and factor 448 / a' of a block from the bits of its largest
// magnitude, both as IEEE division gives them, in a dozen instructions: a' =
// m * 2^e with m in [1, 2), the quotients m / 448 and 448 / m by Newton's and
// Markstein's corrections of an approximate reciprocal (q' = q + (n - q d) y
// with fused multiply-adds; tested for all 2^23 m), then e added to or taken
// from their exponents, which stay normal for 2^-100 <= a' < 2^128. Two plain
// divisions per block and lane took more issue slots than the rest of the row
// kernels (bf16 8192 x 4096: 26.3 us).
__device__ __forceinline__ void f8_scale(uint32_t amax_bits, float &s, float &r) {
    const uint32_t a = max(amax_bits, __float_as_uint(kF8Floor));
    const float m = __uint_as_float((a & 0x007fffffu) | 0x3f800000u);
    const uint32_t e = (a & 0x7f800000u) - 0x3f800000u;  // exponent, in place
    constexpr float inv = 1.0f / kF8Max;
    float q = m * inv;
    q = fmaf(fmaf(-q, kF8Max, m), inv, q);
    float y;
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(m));
    y = fmaf(fmaf(-m, y, 1.0f), y, y);
    float p = kF8Max * y;
    p = fmaf(fmaf(-p, m, kF8Max), y, p);
    const bool broken = amax_bits >= 0x7f800000u;
    s = __uint_as_float(broken ? 0x7fffffffu : __float_as_uint(q) + e);
    r = __uint_as_float(broken ? 0x7fffffffu : __float_as_uint(p) - e);
}

__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
__device__ __forceinline__ uint8_t f8_one(float a) { return (uint8_t)__nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E4M3); }

}  // namespace fbk
