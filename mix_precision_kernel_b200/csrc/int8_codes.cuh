// Numerics of the 8-bit integer codes: one FP32 scale per row or column.
//
//   a = max(max |x|, 2^-100) over the row or column
//   scale = a / 127,   code = rint(x * (127 / a))     (FP32, each operation rounded
//                                                      to nearest, ties to even)
//
// The floor 2^-100 keeps 127 / a finite and makes the codes of an all-zero row zero
// without a case of its own.  |x| <= a gives |x * (127 / a)| <= 127 (1 + 2^-23), which
// rounds to at most 127: codes lie in [-127, 127] and -128 does not occur.
// 8-bit integers have no code for NaN or infinity: a row or column that holds one gets
// scale NaN (and codes 0), so every product with it is NaN instead of silently finite.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace mpk {
namespace int8 {

constexpr float kMinAmax = 0x1p-100f;

struct RowScale {
    float scale, inv;
};

// From the largest magnitude's FP32 bits.  Magnitudes compare as integers, and every
// NaN compares above infinity.
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits)
{
    if (amax_bits >= 0x7F800000u) return {__uint_as_float(0x7FC00000u), 0.0f};
    const float a = fmaxf(__uint_as_float(amax_bits), kMinAmax);
    return {__fdiv_rn(a, 127.0f), __fdiv_rn(127.0f, a)};
}

// rint(x * inv) as a byte.  Adding 1.5 * 2^23 rounds to an integer (ties to even) whose
// low byte is the two's complement code; 0 for inv == 0, where x may be NaN or infinite.
__device__ __forceinline__ uint32_t code_bits(float x, float inv)
{
    return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f));
}

__device__ __forceinline__ uint32_t pack4(const float* v, float inv)
{
    const uint32_t lo = __byte_perm(code_bits(v[0], inv), code_bits(v[1], inv), 0x0040);
    const uint32_t hi = __byte_perm(code_bits(v[2], inv), code_bits(v[3], inv), 0x0040);
    return inv == 0.0f ? 0u : __byte_perm(lo, hi, 0x5410);
}

// Types: a 16-byte vector of kVec elements, widened exactly to FP32.
struct F32 {
    using T = float;
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float widen(float x) { return x; }
    static __device__ __forceinline__ void widen(const uint4& q, float* v)
    {
        v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y);
        v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
    }
};
struct Bf16 {
    using T = uint16_t;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float widen(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ void widen(const uint4& q, float* v)
    {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
struct F16 {
    using T = uint16_t;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float widen(uint16_t x) { return __half2float(__ushort_as_half(x)); }
    static __device__ __forceinline__ void widen(const uint4& q, float* v)
    {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __half2float(__ushort_as_half((uint16_t)w[i]));
            v[2 * i + 1] = __half2float(__ushort_as_half((uint16_t)(w[i] >> 16)));
        }
    }
};

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// FP32 bits of the largest magnitude of a 16-byte piece.  16-bit magnitudes order as
// integers too (NaN above infinity), so two are compared at once and the larger widened.
__device__ __forceinline__ uint32_t largest(F32, const uint4& q)
{
    return max(max(q.x & 0x7FFFFFFFu, q.y & 0x7FFFFFFFu), max(q.z & 0x7FFFFFFFu, q.w & 0x7FFFFFFFu));
}
__device__ __forceinline__ uint32_t largest16(const uint4& q)
{
    const uint32_t m = __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu),
                                __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu));
    return max(m & 0xFFFFu, m >> 16);
}
__device__ __forceinline__ uint32_t largest(Bf16, const uint4& q) { return largest16(q) << 16; }
__device__ __forceinline__ uint32_t largest(F16, const uint4& q)
{
    return __float_as_uint(__half2float(__ushort_as_half((uint16_t)largest16(q)))) & 0x7FFFFFFFu;
}

}  // namespace int8
}  // namespace mpk
