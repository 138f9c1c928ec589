// Device helpers of the block-scaled FP8 operators: e4m3 rows whose 128-column
// groups have an fp32 scale each.
//
// A group of a row is quantized by 16 lanes of 8 consecutive columns each:
//   a = max(max |x|, 1e-10),  scale = a / 448,  q = e4m3(448 x / a)
// with 448 x / a correctly rounded for 16-bit x (quantize8).  448 is the largest
// e4m3 value; the floor keeps the scale of an all-zero group finite and nonzero.
// A group that holds a NaN has scale NaN and q NaN; one that holds an infinity has
// scale inf, NaN where x is infinite and 0 elsewhere, so a product with it is NaN.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "exl3_common.h"
#include "exl3_decode.h"

namespace exl3 {

constexpr int FP8_GROUP = 128;          // columns of a scale
constexpr float FP8_LEAST = 1e-10f;     // least largest magnitude of a group
constexpr float FP8_TOP = 448.0f;       // largest e4m3 value

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

constexpr int FP8_MOST = 1 << 30;       // most columns, rows of a product: indexes of a tile past the end stay in 31 bits

__host__ __device__ __forceinline__ int fp8_groups(int k) { return (int)(((uint32_t)k + FP8_GROUP - 1) / FP8_GROUP); }

// The two 16-bit numbers of a dword in fp32, and fp32 rounded to one (ties to even).
template <bool BF16>
__device__ __forceinline__ float2 f2_of(uint32_t u) {
    if constexpr (BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    const __half2 h = *reinterpret_cast<const __half2*>(&u);
    return make_float2(__low2float(h), __high2float(h));
}
template <bool BF16>
__device__ __forceinline__ uint32_t bits_of(float a, float b) {
    if constexpr (BF16)
        return (uint32_t)__bfloat16_as_ushort(__float2bfloat16(a)) |
               ((uint32_t)__bfloat16_as_ushort(__float2bfloat16(b)) << 16);
    return (uint32_t)__half_as_ushort(__float2half_rn(a)) | ((uint32_t)__half_as_ushort(__float2half_rn(b)) << 16);
}

// Largest over the 16 lanes of a DPP row, in all of them.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, false));  // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xF, 0xF, false));
    return v;
}

// Magnitudes are compared as unsigned bit patterns: finite < inf < NaN, so a NaN is the largest.
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// a / 448, correctly rounded (inf and NaN as they are).
__device__ __forceinline__ float scale_of(float a) {
    const float r = 1.0f / FP8_TOP, s = a * r;
    return a < __builtin_huge_valf() ? fmaf(fmaf(-s, FP8_TOP, a), r, s) : a;
}

__device__ __forceinline__ u32x2_t e4m3x8(const float (&t)[8]) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[4], t[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[6], t[7], hi, true);
    return u32x2_t{(uint32_t)lo, (uint32_t)hi};
}

// Eight 16-bit numbers of one lane, with the other 15 lanes of their group: the
// e4m3 bytes, and the group's scale.  448 x / a is computed as c / d with
// c = 0.875 x and d = a / 512, both exact (448 x would overflow, a / 448 is not
// exact), by a reciprocal and one correction step, which is exact wherever the
// quotient is: a 16-bit x often lies half way between two e4m3 values of its
// group, and x / scale with the rounded scale would decide those ties at random
// (one value in a thousand).
template <bool BF16>
__device__ __forceinline__ u32x2_t quantize8(u32x4_t v, float& scale) {
    typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t m = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t u = v[j] & 0x7fff7fffu;
        m = __builtin_elementwise_max(m, *reinterpret_cast<const u16x2_t*>(&u));
    }
    const uint32_t top = max16(max((uint32_t)m[0], (uint32_t)m[1]));
    float a = f2_of<BF16>(top).x;
    a = a < FP8_LEAST ? FP8_LEAST : a;
    scale = scale_of(a);
    float d = a * (1.0f / 512.0f);
    const float r = __builtin_amdgcn_rcpf(d);
    d = a < __builtin_huge_valf() ? d : 0.0f;  // finite / inf is 0
    float t[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = f2_of<BF16>(v[j]);
        const float c0 = 0.875f * f.x, c1 = 0.875f * f.y;
        const float t0 = c0 * r, t1 = c1 * r;
        t[2 * j] = fmaf(fmaf(-t0, d, c0), r, t0);
        t[2 * j + 1] = fmaf(fmaf(-t1, d, c1), r, t1);
    }
    return e4m3x8(t);
}

// The same for fp32 numbers, where ties are no more likely than any value: y * (448 / a).
__device__ __forceinline__ u32x2_t quantize8_f32(const float (&y)[8], float& scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, mag(y[j]));
    float a = __uint_as_float(max16(m));
    a = a < FP8_LEAST ? FP8_LEAST : a;
    scale = scale_of(a);
    const float r = FP8_TOP / a;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = y[j] * r;
    return e4m3x8(t);
}

// Rows of 16-bit numbers to e4m3 (exl3_fp8_rows.hip); arguments are checked by the caller.
int fp8_quant_rows(const void* x, bool bf16, long long stride, uint8_t* q, float* scale, int rows, int cols,
                   hipStream_t st);

}  // namespace exl3
