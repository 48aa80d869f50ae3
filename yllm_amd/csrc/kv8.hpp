// kv8.hpp -- the 8-bit KV pool's format: codes, scales, and their conversions.
//
// Per layer, pages of `block` positions (a multiple of 64):
//   K codes   [n_blocks][n_kv][block][D]          e4m3
//   V codes   [n_blocks][n_kv][block / 64][D][64] e4m3, d-major tiles of 64 positions
//   scales    [n_blocks][n_kv][block], of K and of V: powers of two in e5m2
// A value is code * scale.  A row (one position of one kv head) has a scale of
// its own, 2^k with
//   k = ceil(log2(amax / 448)) within -14 .. 7
// (448: e4m3's largest; amax over the row's finite elements), and codes
// x * 2^-k to nearest even.  So a row appended later changes nothing that is
// stored, and rows of any order or chunking give the same bytes; the scales are
// 1 / D of the codes.  A power of two costs e4m3 no precision but at its
// subnormals, and code * 2^k is a f16 number exactly for k in that range (2^-9 *
// 2^-14 = 2^-23 up to 448 * 2^7 = 57344), so that the products run on f16 MFMA
// without a second rounding.  e5m2 is the upper byte of f16: a scale becomes a
// f16 factor by a byte permutation.  Values past 57344 are held as that; inf and
// NaN as e4m3's NaN (0x7f, it has no inf).
#pragma once

#include "common.hpp"

#include <math.h>

namespace yhip {

constexpr uint32_t kV8Tile = 64;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// the magnitude's bits where x is finite, else 0 (they order as the values do)
__device__ inline uint32_t finite_mag(float x)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// k of a row whose largest finite magnitude has these bits: 448 = 1.75 * 2^8
__device__ inline int kv8_exponent(uint32_t mag)
{
    const int k = (int)(mag >> 23) - (127 + 8) + ((mag & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(k, -14), 7);
}
__device__ inline uint8_t kv8_scale_byte(int k) { return (uint8_t)((k + 15) << 2); }
__device__ inline float kv8_inverse(int k) { return __builtin_bit_cast(float, (uint32_t)(127 - k) << 23); }

// codes of four values, with the 2^-k of each one's row
__device__ inline uint32_t kv8_codes(const f32x4& x, const f32x4& inv)
{
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float t = __builtin_amdgcn_fmed3f(x[e] * inv[e], -448.0f, 448.0f);
        y[e] = fabsf(x[e]) < INFINITY ? t : NAN;
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    return (uint32_t)w;
}
__device__ inline uint32_t kv8_codes(const f32x4& x, float inv) { return kv8_codes(x, f32x4{inv, inv, inv, inv}); }

// the f16 factors of bytes 2 h and 2 h + 1 of four scales
__device__ inline f16x2 kv8_factors(uint32_t scales, int h)
{
    return __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0u, scales, h ? 0x030c020cu : 0x010c000cu));
}
// one scale as fp32
__device__ inline float kv8_scale(uint32_t byte)
{
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(byte << 8));
}

// eight codes of one row, with its scale
__device__ inline f16x8 kv8_values(uint32_t lo, uint32_t hi, float scale)
{
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false),
                b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true),
                c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false),
                d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// eight codes of eight rows, with their factors in pairs
__device__ inline f16x8 kv8_values(uint32_t lo, uint32_t hi, const f16x2 (&f)[4])
{
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false) * f[0],
                b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true) * f[1],
                c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false) * f[2],
                d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true) * f[3];
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// the top bit of each byte that is a NaN code
__device__ inline uint32_t kv8_nans(uint32_t codes) { return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

}  // namespace yhip
