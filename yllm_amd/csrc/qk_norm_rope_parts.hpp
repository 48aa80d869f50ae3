// qk_norm_rope_parts.hpp -- shared by the appends to the f16 and the 8-bit KV
// pool (qk_norm_rope.hip, qk_norm_rope8.hip): loads and stores of four elements,
// sines and cosines, sums over the lanes of a head, slots.
#pragma once

#include "common.hpp"
#include "internal.hpp"

namespace yhip {
namespace {

typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

template <uint32_t DT>
__device__ inline f32x4 load4(const void* p, size_t i)
{
    if constexpr (DT == kF32) {
        return __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i));
    } else {
        const u16x4 w = __builtin_nontemporal_load(reinterpret_cast<const u16x4*>(reinterpret_cast<const uint16_t*>(p) + i));
        f32x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = DT == kBF16 ? bf16_bits_to_f32(w[e]) : f16_bits_to_f32(w[e]);
        return r;
    }
}

// (the conversions to bf16 and f16 are gfx950's own, to nearest even)
__device__ inline void store4(void* p, size_t i, uint32_t dt, const f32x4& x)
{
    if (dt == kF32) {
        *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + i) = x;
    } else if (dt == kF16) {
        f16x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (_Float16)x[e];
        *reinterpret_cast<f16x4*>(reinterpret_cast<uint16_t*>(p) + i) = w;
    } else {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        bf16x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (__bf16)x[e];
        *reinterpret_cast<bf16x4*>(reinterpret_cast<uint16_t*>(p) + i) = w;
    }
}

// sine and cosine of u turns: whole turns and then quarters are taken off in
// 64 bits, and the Taylor series over an eighth of a turn to either side follow
// (what they leave out is below 2.5e-8)
__device__ inline void sincos_turns(double u, float* sn, float* cs)
{
    const double q4 = 4.0 * (u - __builtin_rint(u)), whole = __builtin_rint(q4);
    const float x = 1.5707963267948966f * (float)(q4 - whole), z = x * x;
    const int q = (int)whole;
    const float s = x + x * z * (-1.6666667e-1f + z * (8.3333333e-3f + z * (-1.9841270e-4f + z * 2.7557319e-6f)));
    const float c = 1.0f + z * (-0.5f + z * (4.1666667e-2f + z * (-1.3888889e-3f + z * 2.4801587e-5f)));
    const float a = q & 1 ? c : s, b = q & 1 ? s : c;
    *sn = q & 2 ? -a : a;
    *cs = (q + 1) & 2 ? -b : b;
}

// the sum over each aligned group of N lanes, by DPP moves: within quads, the
// other quad of eight (mirrored), the other eight of a row, the other row
template <int N>
__device__ inline float group_sum(float x)
{
    static_assert(N == 8 || N == 16 || N == 32, "a head is 8, 16 or 32 lanes");
    x += dpp_mov<0xb1>(x);   // quad_perm [1, 0, 3, 2]
    x += dpp_mov<0x4e>(x);   // quad_perm [2, 3, 0, 1]
    x += dpp_mov<0x141>(x);  // row_half_mirror
    if constexpr (N >= 16) x += dpp_mov<0x140>(x);  // row_mirror
    if constexpr (N == 32) x = sum_xor16(x);
    return x;
}

// a row's slot (negative: none)
__device__ inline int slot_of(const QkNormRopeArgs& a, uint32_t b)
{
    const uint32_t s = a.slots ? (uint32_t)a.slots[b] : a.pos_start + b;
    return s < a.n_slots ? (int)s : -1;
}

}  // namespace
}  // namespace yhip
