// qk_norm_rope8.hip -- RMSNorm of every query and key head, the position
// rotation, and the store of K and V into the 8-bit KV pool (kv8.hpp), in one
// pass over the projected rows.  Norm, angles and rotation are those of
// qk_norm_rope.hip; K and V rows become a scale and e4m3 codes.
//
// Each row is read once and written once.  A lane holds eight elements of a
// head as two runs of four, so that a head is D / 8 lanes and its sum of squares
// and largest magnitude are a few DPP moves.  A wave takes heads in rounds of
// three passes (two of fp32: 96 registers, five waves a SIMD), the next round's
// loads in flight behind one's arithmetic, and
// forms the row's sines and cosines once for all of them.  V is d-major in the
// pool: workgroups of their own turn 64 rows of a kv head over in LDS, sixteen
// aligned positions a store; a row outside such a group (a decode token, the ends
// of a sequence's new tokens) has its V stored a byte at a time by the waves of
// its other heads.
//
// Measured: 8166 tokens of three prompts, 16 / 2 heads of 256 (M-RoPE over 64),
// bf16: 36 us, 4.4 TB/s, where a large copy reaches 5.1 (31 us); of 32 / 8 heads of
// 128 40 us, 4.6 TB/s; 2070 fp32 rows, four chunks and 28 decode tokens, of 28 / 4 of
// 128 15.4 us, 3.6 TB/s; one decode token 3.5 us, 64 of 32 / 8 of 128 4.4.  What they
// wait for is asked for in the order of its use: the slots and the angles' factors
// before the row, a lone row's V before the arithmetic (39, 42.5, 17.5 and 4.0 us with
// the row first).
#include "common.hpp"
#include "internal.hpp"
#include "kv8.hpp"
#include "qk_norm_rope_parts.hpp"

#include <algorithm>

namespace yhip {
namespace {

// Up to this many rows every row's V goes with its other heads (32 / 8 heads of 128,
// decode tokens: 300 rows 8.8 us so, 400 the other way 10.8, 28 / 4: 5.9 and 9.0; of a
// prompt 6.1 and 5.6, 28 / 4: 4.8 and 5.4).
constexpr uint32_t kFewRows8 = 384;

// four elements as loaded, and widened
template <uint32_t DT>
struct Raw4;
template <>
struct Raw4<kF32> {
    typedef f32x4 type;
};
template <>
struct Raw4<kF16> {
    typedef u16x4 type;
};
template <>
struct Raw4<kBF16> {
    typedef u16x4 type;
};
template <uint32_t DT>
__device__ inline typename Raw4<DT>::type raw4(const void* p, size_t i)
{
    typedef typename Raw4<DT>::type T;
    return __builtin_nontemporal_load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + i * sizeof(T) / 4));
}
template <uint32_t DT>
__device__ inline f32x4 widen4(const typename Raw4<DT>::type& w)
{
    if constexpr (DT == kF32) {
        return w;
    } else {
        f32x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = DT == kBF16 ? bf16_bits_to_f32(w[e]) : f16_bits_to_f32(w[e]);
        return r;
    }
}

// the largest of each aligned group of N lanes, by the moves of group_sum
template <int N>
__device__ inline uint32_t group_max(uint32_t x)
{
    auto with = [&](float o) { x = max(x, __builtin_bit_cast(uint32_t, o)); };
    auto f = [&] { return __builtin_bit_cast(float, x); };
    with(dpp_mov<0xb1>(f()));
    with(dpp_mov<0x4e>(f()));
    with(dpp_mov<0x141>(f()));
    if constexpr (N >= 16) with(dpp_mov<0x140>(f()));
    if constexpr (N == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = max((uint32_t)r[0], (uint32_t)r[1]);
    }
    return x;
}
// k of a row that a group of N lanes holds, eight elements each
template <int N>
__device__ inline int group_exponent(const f32x4& y0, const f32x4& y1)
{
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, max(finite_mag(y0[e]), finite_mag(y1[e])));
    return kv8_exponent(group_max<N>(top));
}

// Of values that a head's lanes of one place formed between them, heads % 4 (head_dim 256: % 2, two each), all four
template <int D>
__device__ inline void share4(const float (&own)[D == 256 ? 2 : 1], float (&all)[4])
{
    auto bits = [](float x) { return __builtin_bit_cast(uint32_t, x); };
    auto val = [](uint32_t x) { return __builtin_bit_cast(float, x); };
    if constexpr (D == 256) {  // the halves of the wave
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const auto r = __builtin_amdgcn_permlane32_swap(bits(own[n]), bits(own[n]), false, false);
            all[2 * n] = val(r[0]);
            all[2 * n + 1] = val(r[1]);
        }
    } else if constexpr (D == 128) {  // rows of 16
        const auto r = __builtin_amdgcn_permlane32_swap(bits(own[0]), bits(own[0]), false, false);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const auto q = __builtin_amdgcn_permlane16_swap(r[n], r[n], false, false);
            all[2 * n] = val(q[0]);
            all[2 * n + 1] = val(q[1]);
        }
    } else {  // the halves of rows, and the rows of a half wave
        const bool upper = threadIdx.x & 8u;
        const auto r = __builtin_amdgcn_permlane16_swap(bits(own[0]), bits(own[0]), false, false);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const float x = val(r[n]), y = dpp_mov<0x128>(x);  // row_ror 8
            all[2 * n] = upper ? y : x;
            all[2 * n + 1] = upper ? x : y;
        }
    }
}

// A slot's place: of its scale in head 0 (K codes: D times that), and of V codes
// (dimension 0) from head 0's on
struct Place8 {
    size_t scale, v;
};
template <int D>
__device__ inline Place8 place_of(const QkNormRopeArgs& a, uint32_t slot)
{
    const uint32_t page = slot / a.block, off = slot - page * a.block;
    const size_t row = (size_t)page * a.n_kv * a.block;
    return Place8{row + off, (row + (off & ~(kV8Tile - 1))) * D + (off & (kV8Tile - 1))};
}

// V workgroup: 64 rows of one kv head.  A row's lanes form its scale and codes
// and leave them in LDS, four codes a word; sixteen rows whose slots are
// consecutive from a multiple of 16 on leave as one 16-byte store per dimension,
// by the workgroup of their first row (which therefore reads up to 15 rows more),
// four dimensions a thread, turned over by byte permutations.
template <int D, uint32_t DT>
__device__ void v8_block(const QkNormRope8Args& a, uint32_t vb)
{
    constexpr uint32_t LPH = D / 8, RPP = 256 / LPH, W = D / 4 + 1;  // lanes a row, rows a pass, words a row in LDS
    constexpr uint32_t R = (79 + RPP) / RPP * RPP;                    // rows read: 79 are needed
    __shared__ uint32_t tile[R * W];
    __shared__ int slots[64 + 15];  // of rows r0 .. r0 + 78
    __shared__ uint8_t scale[R];
    __shared__ uint32_t lead[2];
    const uint32_t h = vb % a.n_kv, r0 = vb / a.n_kv * 64u;
    const uint32_t t = threadIdx.x, i = t % LPH, rr = t / LPH;
    if (t < 79u) slots[t] = r0 + t < a.n_tok ? slot_of(a, r0 + t) : -1;
    __syncthreads();
    if (t < 64u) {  // whether rows t .. t + 15 are one group
        const int s = slots[t];
        bool ok = s >= 0 && (s & 15) == 0;
#pragma unroll
        for (int e = 1; e < 16; ++e) ok = ok && slots[t + e] == s + e;
        const uint64_t m = __ballot(ok);
        if (t == 0) {
            lead[0] = (uint32_t)m;
            lead[1] = (uint32_t)(m >> 32);
        }
    }
    __syncthreads();
    if ((lead[0] | lead[1]) == 0) return;  // workgroup-uniform
    constexpr uint32_t U = R / RPP > 5 ? 5 : R / RPP;  // passes whose loads go out together
    static_assert(R / RPP % U == 0, "whole rounds");
#pragma unroll 1
    for (uint32_t p0 = 0; p0 < R / RPP; p0 += U) {
        typename Raw4<DT>::type x[U][2];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t b = min(r0 + (p0 + u) * RPP + rr, a.n_tok - 1u);
            const size_t at = (size_t)b * a.v_stride + h * D + 4u * i;
            x[u][0] = raw4<DT>(a.v, at);
            x[u][1] = raw4<DT>(a.v, at + D / 2);
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t r = (p0 + u) * RPP + rr;
            const f32x4 y0 = widen4<DT>(x[u][0]), y1 = widen4<DT>(x[u][1]);
            const int k = group_exponent<LPH>(y0, y1);
            const float inv = kv8_inverse(k);
            tile[r * W + i] = kv8_codes(y0, inv);
            tile[r * W + LPH + i] = kv8_codes(y1, inv);
            if (i == 0) scale[r] = kv8_scale_byte(k);
        }
    }
    __syncthreads();
    // first rows of groups are at least 16 apart: at most one in each 16 rows
    if (t < D) {
        const uint32_t g = t & 3u, c = t >> 2;  // a group, four dimensions
        const uint32_t m = lead[g >> 1] >> (16u * (g & 1u)) & 0xffffu;
        if (!m) return;
        const uint32_t r = 16u * g + (uint32_t)__builtin_ctz(m);
        const Place8 p = place_of<D>(a, (uint32_t)slots[r]);
        u32x4 w[4];  // [dimension][four rows a word]
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
            const uint32_t* s = &tile[(r + 4u * q) * W + c];
            const uint32_t a0 = s[0], a1 = s[W], a2 = s[2 * W], a3 = s[3 * W];
            const uint32_t lo01 = __builtin_amdgcn_perm(a1, a0, 0x05010400u), hi01 = __builtin_amdgcn_perm(a1, a0, 0x07030602u),
                           lo23 = __builtin_amdgcn_perm(a3, a2, 0x05010400u), hi23 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
            w[0][q] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
            w[1][q] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
            w[2][q] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
            w[3][q] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
        }
        uint8_t* const dst = reinterpret_cast<uint8_t*>(a.vc) + p.v + (size_t)h * a.block * D + 4u * c * kV8Tile;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) *reinterpret_cast<u32x4*>(dst + e * kV8Tile) = w[e];
        if (c == 0) {  // the rows' scales
            u32x4 b;
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q)
                b[q] = scale[r + 4 * q] | scale[r + 4 * q + 1] << 8 | scale[r + 4 * q + 2] << 16 | (uint32_t)scale[r + 4 * q + 3] << 24;
            *reinterpret_cast<u32x4*>(a.vs + p.scale + (size_t)h * a.block) = b;  // (slots and pools are multiples of 16)
        }
    }
}

// FEW: a row a wave group, every row's V among its passes.
template <uint32_t KIND, int D, uint32_t DT, bool FEW>
__global__ __launch_bounds__(256, FEW ? 1 : 5) void qk_norm_rope8_kernel(QkNormRope8Args a)
{
    // the two roles alternate over the first 2 * min(rotation, V) workgroups (rope.hip)
    uint32_t blk = blockIdx.x;
    if constexpr (!FEW) {
        const uint32_t m = min(a.rope_blocks, a.v_blocks);
        bool v_role;
        if (blk < 2 * m) {
            v_role = blk & 1u;
            blk >>= 1;
        } else {
            v_role = a.v_blocks > a.rope_blocks;
            blk -= m;
        }
        if (v_role) {  // workgroup-uniform
            v8_block<D, DT>(a, blk);
            return;
        }
    }
    constexpr uint32_t LPH = D / 8, HPP = 64 / LPH;  // lanes per head, heads per pass
    constexpr uint32_t U = FEW ? 1 : DT == kF32 ? 2 : 3;  // passes of a round: their loads are issued together
    const uint32_t lane = threadIdx.x & 63u, i = lane % LPH, sub = lane / LPH;
    const uint32_t w = blk * 4u + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t b = w / a.groups, g = w - b * a.groups;
    if (b >= a.n_tok) return;  // wave-uniform; no barrier follows in this role
    // (the row's slot and position are waited for behind its first loads)
    const int slot = slot_of(a, b);
    const int pos = a.positions ? a.positions[b] : (int)(a.pos_start + b);

    // The lane's two runs of four elements: one of the lower and one of the upper half of the dimensions, or (MROPE)
    // of the rotated ones or the rest.  Neighbouring lanes' runs are neighbours, and the pairs of every kind lie
    // within a lane: two in each run, or one element in each.
    const uint32_t span = KIND == kRopeMrope ? a.n_rot : (uint32_t)D;
    const bool head = 8u * i < span;  // whether they are among the first `span` dimensions, which turn
    const uint32_t e0 = head ? 4u * i : span / 2 + 4u * i, e1 = e0 + (head ? span : (uint32_t)D - span) / 2;
    const bool turn = KIND != kRopeNone && head;

    // This wave's passes: HPP heads each, those of q (none without q_out), those of k, FEW: those of v.  A pass is of
    // one kind, so that everything but the lane's offsets is wave-uniform.
    const uint32_t pq = a.q_out ? (a.n_heads + HPP - 1) / HPP : 0u, pk = (a.n_kv + HPP - 1) / HPP, passes = pq + (FEW ? 2 : 1) * pk;
    const uint32_t p_lo = g * a.passes, p_hi = min(passes, p_lo + a.passes);
    auto row_at = [&](const void* base, uint32_t stride) {
        return reinterpret_cast<const char*>(base) + (size_t)b * stride * (DT == kF32 ? 4 : 2);
    };
    struct Round {  // what is loaded ahead
        typename Raw4<DT>::type x[U][2];
    };
    auto load = [&](Round& r, uint32_t p0) __attribute__((always_inline)) {  // heads past the last load it again
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t p = min(p0 + u, p_hi - 1u);
            const bool is_q = p < pq, is_v = FEW && p >= pq + pk;
            const uint32_t h = min((is_q ? p : is_v ? p - pq - pk : p - pq) * HPP + sub, (is_q ? a.n_heads : a.n_kv) - 1u);
            const char* src = is_q ? row_at(a.q, a.q_stride) : is_v ? row_at(a.v, a.v_stride) : row_at(a.k, a.k_stride);
            r.x[u][0] = raw4<DT>(src, h * D + e0);
            r.x[u][1] = raw4<DT>(src, h * D + e1);
        }
    };
    // The sines and cosines of the lane's four pairs: each of the wave's lanes of the same place in their heads forms one
    // (two at head_dim 256), e = sub % (4 / N) + 4 / N * n, and they pass them round.  What they are formed from is asked
    // for first: only this is waited for while the row is on its way.
    constexpr uint32_t N = D == 256 ? 2 : 1;
    double turns[N] = {};
    if (KIND != kRopeNone && turn) {
#pragma unroll
        for (uint32_t n = 0; n < N; ++n) {
            const uint32_t e = sub % (4 / N) + 4 / N * n;
            turns[n] = a.turns[KIND == kRopePairs ? (e < 2 ? 2u * i + e : D / 4 + 2u * i + (e - 2)) : 4u * i + e];
        }
    }
    // !FEW: the slots of the rows about this one, row b - 15 + lane's (31 lanes), say whether it is one of sixteen that a
    // V workgroup stores
    int near = -1;
    if constexpr (!FEW) {
        const int at = (int)(b + lane) - 15;
        if (lane < 31u && at >= 0 && (uint32_t)at < a.n_tok) near = slot_of(a, (uint32_t)at);
    }
    __builtin_amdgcn_sched_barrier(0);
    Round ra, rb;
    load(ra, p_lo);
    __builtin_amdgcn_sched_barrier(0);  // nothing below waits before these are issued
    if (slot < 0) return;  // wave-uniform
    const Place8 place = place_of<D>(a, (uint32_t)slot);
    // !FEW: a lone row, and its V heads of pass g, asked for before the arithmetic
    bool lone = false;
    auto load_v = [&](uint32_t v, typename Raw4<DT>::type (&x)[2]) __attribute__((always_inline)) {
        const uint32_t h = min(v * HPP + sub, a.n_kv - 1u);
        x[0] = raw4<DT>(row_at(a.v, a.v_stride), h * D + e0);
        x[1] = raw4<DT>(row_at(a.v, a.v_stride), h * D + e1);
    };
    typename Raw4<DT>::type vx[2] = {};
    if constexpr (!FEW) {
        const int l0 = 15 - (slot & 15);  // the lanes of the group's rows are l0 .. l0 + 15
        const uint64_t same = __ballot(near == (slot & ~15) + ((int)lane - l0));
        lone = (same >> l0 & 0xffffu) != 0xffffu;
        if (lone && g < pk) load_v(g, vx);
    }
    float c[4] = {1.0f, 1.0f, 1.0f, 1.0f}, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (KIND != kRopeNone) {
        float oc[N], os[N];
#pragma unroll
        for (uint32_t n = 0; n < N; ++n) {
            sincos_turns(turns[n] * (double)pos, &os[n], &oc[n]);  // (no turn: 1 and 0)
        }
        share4<D>(oc, c);
        share4<D>(os, s);
    }
    f32x4 qw[2], kw[2];
    const bool norm = a.q_norm != nullptr;
    if (norm) {
        if (a.norm_f16) {
            qw[0] = load4<kF16>(a.q_norm, e0);
            qw[1] = load4<kF16>(a.q_norm, e1);
            kw[0] = load4<kF16>(a.k_norm, e0);
            kw[1] = load4<kF16>(a.k_norm, e1);
        } else {
            qw[0] = load4<kF32>(a.q_norm, e0);
            qw[1] = load4<kF32>(a.q_norm, e1);
            kw[0] = load4<kF32>(a.k_norm, e0);
            kw[1] = load4<kF32>(a.k_norm, e1);
        }
    }

    auto store_v = [&](uint32_t h, const f32x4& y0, const f32x4& y1) __attribute__((always_inline)) {
        const int k = group_exponent<LPH>(y0, y1);
        const float inv = kv8_inverse(k);
        const uint32_t w0 = kv8_codes(y0, inv), w1 = kv8_codes(y1, inv);
        if (h < a.n_kv) {
            uint8_t* const dst = reinterpret_cast<uint8_t*>(a.vc) + place.v + (size_t)h * a.block * D;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                dst[(e0 + e) * kV8Tile] = (uint8_t)(w0 >> 8 * e);
                dst[(e1 + e) * kV8Tile] = (uint8_t)(w1 >> 8 * e);
            }
            if (i == 0) a.vs[place.scale + (size_t)h * a.block] = kv8_scale_byte(k);
        }
    };
    auto round = [&](const Round& r, uint32_t p0) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t p = p0 + u;
            if (p >= p_hi) break;  // wave-uniform
            const bool is_q = p < pq, is_v = FEW && p >= pq + pk;
            const uint32_t h = (is_q ? p : is_v ? p - pq - pk : p - pq) * HPP + sub;
            f32x4 y0 = widen4<DT>(r.x[u][0]), y1 = widen4<DT>(r.x[u][1]);
            if (is_v) {
                store_v(h, y0, y1);
                continue;
            }
            if (norm) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = fmaf(y0[e], y0[e], fmaf(y1[e], y1[e], ss));
                ss = group_sum<LPH>(ss);
                const float inv = __builtin_amdgcn_rsqf(fmaf(ss, 1.0f / D, a.eps));
                y0 *= inv;
                y1 *= inv;
                y0 *= is_q ? qw[0] : kw[0];
                y1 *= is_q ? qw[1] : kw[1];
            }
            if (KIND == kRopePairs) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f32x4& y = e < 2 ? y0 : y1;
                    const float v = y[2 * (e & 1)], t = y[2 * (e & 1) + 1];
                    y[2 * (e & 1)] = v * c[e] - t * s[e];
                    y[2 * (e & 1) + 1] = v * s[e] + t * c[e];
                }
            } else if (KIND != kRopeNone) {  // (lanes that do not turn have cosine 1 and sine 0)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = y0[e], t = y1[e];
                    y0[e] = KIND == kRopeHalf || turn ? v * c[e] - t * s[e] : v;
                    y1[e] = KIND == kRopeHalf || turn ? v * s[e] + t * c[e] : t;
                }
            }
            if (is_q) {
                if (h < a.n_heads) {
                    const size_t at = (size_t)b * a.q_out_stride + h * D;
                    store4(a.q_out, at + e0, a.q_out_dtype, y0);
                    store4(a.q_out, at + e1, a.q_out_dtype, y1);
                }
            } else {
                const int k = group_exponent<LPH>(y0, y1);
                const float inv = kv8_inverse(k);
                const uint32_t w0 = kv8_codes(y0, inv), w1 = kv8_codes(y1, inv);
                if (h < a.n_kv) {
                    const size_t at = place.scale + (size_t)h * a.block;
                    uint8_t* const row = reinterpret_cast<uint8_t*>(a.kc) + at * D;
                    *reinterpret_cast<uint32_t*>(row + e0) = w0;
                    *reinterpret_cast<uint32_t*>(row + e1) = w1;
                    if (i == 0) a.ks[at] = kv8_scale_byte(k);
                }
            }
        }
    };
    // (q_out may be q: a row's elements are read by the lane that writes them, before it does)
    if constexpr (FEW) {  // (one pass a wave)
        round(ra, p_lo);
    } else {
        for (uint32_t p0 = p_lo;;) {
            if (p0 + U < p_hi) load(rb, p0 + U);
            round(ra, p0);
            if ((p0 += U) >= p_hi) break;
            if (p0 + U < p_hi) load(ra, p0 + U);
            round(rb, p0);
            if ((p0 += U) >= p_hi) break;
        }
        if (!lone) return;
        for (uint32_t v = g; v < pk; v += a.groups) {
            if (v != g) load_v(v, vx);
            store_v(v * HPP + sub, widen4<DT>(vx[0]), widen4<DT>(vx[1]));
        }
    }
}

template <uint32_t KIND, int D, bool FEW>
hipError_t launch8_dt(const QkNormRope8Args& a, dim3 grid, hipStream_t st)
{
    switch (a.dtype) {
    case kF32: hipLaunchKernelGGL((qk_norm_rope8_kernel<KIND, D, kF32, FEW>), grid, dim3(256), 0, st, a); break;
    case kF16: hipLaunchKernelGGL((qk_norm_rope8_kernel<KIND, D, kF16, FEW>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((qk_norm_rope8_kernel<KIND, D, kBF16, FEW>), grid, dim3(256), 0, st, a); break;
    }
    return hipGetLastError();
}

template <uint32_t KIND>
hipError_t launch8_kind(const QkNormRope8Args& a, bool few, dim3 grid, hipStream_t st)
{
    switch (a.D) {
    case 64: return few ? launch8_dt<KIND, 64, true>(a, grid, st) : launch8_dt<KIND, 64, false>(a, grid, st);
    case 128: return few ? launch8_dt<KIND, 128, true>(a, grid, st) : launch8_dt<KIND, 128, false>(a, grid, st);
    case 256: return few ? launch8_dt<KIND, 256, true>(a, grid, st) : launch8_dt<KIND, 256, false>(a, grid, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_qk_norm_rope8(QkNormRope8Args a, hipStream_t st)
{
    const uint32_t hpp = 64u / (a.D / 8u), pk = (a.n_kv + hpp - 1) / hpp;
    const bool few = a.n_tok <= kFewRows8;
    const uint32_t passes = (a.q_out ? (a.n_heads + hpp - 1) / hpp : 0u) + (few ? 2 : 1) * pk;
    if (few) {
        a.passes = 1;
        a.groups = passes;
        a.v_blocks = 0;
    } else {
        // A row's passes to one wave, which forms its sines and cosines once, but at most kMostPasses, and to more of
        // them where the rows alone are less than about kWaves (8166 rows of 16 / 2 heads of 256, nine passes: 36 us
        // with one wave, 39 with two, 40 with three; of 32 / 8 of 128, ten: 40 with two, 44 with three, 49 with one;
        // 2048 fp32 rows of 28 / 4 of 128, eight: 13.8 with two, 15.2 with three, 14.1 with four; 1000 of 16 / 2 of
        // 256: 9.5 with three, 8.7 with five).  More than a row a wave was slower for all.
        constexpr uint32_t kMostPasses = 9, kWaves = 3500;
        const uint32_t want = std::min(passes, std::max((kWaves + a.n_tok - 1) / a.n_tok, (passes + kMostPasses - 1) / kMostPasses));
        a.passes = (passes + want - 1) / want;
        a.groups = (passes + a.passes - 1) / a.passes;
        a.v_blocks = a.n_kv * ((a.n_tok + 63u) / 64u);
    }
    a.rope_blocks = (uint32_t)(((uint64_t)a.n_tok * a.groups + 3u) / 4u);
    const dim3 grid(a.rope_blocks + a.v_blocks);
    switch (a.kind) {
    case kRopeNone: return launch8_kind<kRopeNone>(a, few, grid, st);
    case kRopePairs: return launch8_kind<kRopePairs>(a, few, grid, st);
    case kRopeHalf: return launch8_kind<kRopeHalf>(a, few, grid, st);
    case kRopeMrope: return launch8_kind<kRopeMrope>(a, few, grid, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace yhip
