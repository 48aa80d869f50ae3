// qk_norm_rope.hip -- RMSNorm of every query and key head, the position
// rotation, and the store of K and V into cache pages, in one pass over the
// projected rows (the step ahead of attention for models with a QK norm:
// engine.c:886-934 norms the heads, rotates them and stores K and V).
//
// Per head x of D dimensions at position pos:
//   y = x / sqrt(mean(x^2) + eps) * w             (w: one weight per dimension)
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = pos * theta^(-2j / span)
// over the pairs of the rope kind (rope.hip).  Mean and norm are fp32.  The
// angle is formed in 64 bits as a fraction of a turn, reduced there to half a
// turn and only then rounded to fp32: an fp32 product pos * freq is off by up
// to pos * 6e-8 rad, 8e-3 at position 131071.
//
// The row's slot says where K and V go: page slot / block, row slot % block.
// Rows without a slot (negative, or past the pool) are skipped.
//
// Bound by HBM: each row is read once and written once.  A lane holds eight
// elements of a head as two runs of four (for pairs half a span apart one run
// of the first and one of the second elements, so a pair never leaves the
// lane; otherwise eight consecutive ones), so a head is D / 8 lanes, a wave
// takes 64 / (D / 8) heads a pass, and the sum of squares is a few DPP steps.
// The lane's four sines and cosines serve all its passes.  V is stored
// d-major, in 16-byte groups of eight positions, by workgroups of their own
// (a few rows: by the same waves, 2 bytes at a time).
#include "common.hpp"
#include "internal.hpp"

namespace yhip {
namespace {

// Up to this many rows the rotation waves write V too, as in rope.hip.
constexpr uint32_t kScatterRows = 128;

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

__device__ inline uint16_t bf16_bits(float x)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);  // NaN stays NaN
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

__device__ inline void store4(void* p, size_t i, uint32_t dt, const f32x4& x)
{
    if (dt == kF32) {
        *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + i) = x;
    } else {
        u16x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float f = x[e];
            w[e] = dt == kF16 ? __builtin_bit_cast(uint16_t, (_Float16)f) : bf16_bits(f);
        }
        *reinterpret_cast<u16x4*>(reinterpret_cast<uint16_t*>(p) + i) = w;
    }
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

// K row and V column of a slot, as element offsets into the pools
template <int D>
__device__ inline size_t k_page_row(const QkNormRopeArgs& a, uint32_t h, uint32_t slot)
{
    const uint32_t page = slot / a.block, off = slot - page * a.block;
    return (((size_t)page * a.n_kv + h) * a.block + off) * D;
}
template <int D>
__device__ inline size_t v_page_at(const QkNormRopeArgs& a, uint32_t h, uint32_t slot, uint32_t d)
{
    const uint32_t page = slot / a.block, off = slot - page * a.block;
    return (((size_t)page * a.n_kv + h) * a.block + (off & ~31u)) * D + d * kVTile + (off & 31u);
}

// V workgroup: 64 rows x 64 channels of one kv head, transposed through LDS.
// Eight rows whose slots are consecutive from a multiple of 8 on leave as one
// 16-byte store per channel, by the workgroup of their first row (which
// therefore reads up to 7 rows more); rows outside such a group, at the ends
// of a sequence's new tokens, go 2 bytes at a time.
template <int D, uint32_t DT>
__device__ void v_block(const QkNormRopeArgs& a, uint32_t vb)
{
    constexpr uint32_t R = 80, TP = 90;  // rows read (5 passes of 16); halfs per channel (45 words: odd, spreads the banks)
    __shared__ __attribute__((aligned(16))) uint16_t tile[64 * TP];
    __shared__ int slots[7 + 64 + 7];    // of rows r0 - 7 .. r0 + 70
    __shared__ uint32_t lead[2], lone[2];
    const uint32_t ntx = a.n_kv * D / 64u;
    const uint32_t j0 = vb % ntx * 64u, r0 = vb / ntx * 64u;
    const uint32_t h = j0 / D, d0 = j0 - h * D;
    const uint32_t t = threadIdx.x, c4 = (t & 15u) * 4u, rr = t >> 4;
    f32x4 x[R / 16];
#pragma unroll
    for (uint32_t u = 0; u < R / 16; ++u) {
        const uint32_t b = min(r0 + rr + 16u * u, a.n_tok - 1u);
        x[u] = load4<DT>(a.v, (size_t)b * a.v_stride + j0 + c4);
    }
    if (t < 78u) {
        const int b = (int)(r0 + t) - 7;
        slots[t] = b >= 0 && (uint32_t)b < a.n_tok ? slot_of(a, (uint32_t)b) : -1;
    }
#pragma unroll
    for (uint32_t u = 0; u < R / 16; ++u)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const float f = x[u][e];
            // f16 rows keep their bits (the widened value rounds back to them; a NaN's payload apart)
            tile[(c4 + e) * TP + rr + 16u * u] =
                DT == kF16 ? __builtin_bit_cast(uint16_t, (_Float16)f) : f32_to_f16_ref(f);
        }
    __syncthreads();
    if (t < 64u) {
        // leads(i): rows i .. i + 7 of slots[] are one group
        auto leads = [&](int i) {
            if (i < 0) return false;
            const int s = slots[i];
            bool ok = s >= 0 && (s & 7) == 0;
#pragma unroll
            for (int e = 1; e < 8; ++e) ok = ok && slots[i + e] == s + e;
            return ok;
        };
        const int i = 7 + (int)t, s = slots[i];
        const uint64_t ml = __ballot(leads(i));
        const uint64_t mn = __ballot(s >= 0 && !leads(i - (s & 7)));
        if (t == 0) {
            lead[0] = (uint32_t)ml;
            lead[1] = (uint32_t)(ml >> 32);
            lone[0] = (uint32_t)mn;
            lone[1] = (uint32_t)(mn >> 32);
        }
    }
    __syncthreads();
    // first rows of groups are at least 8 apart: at most one in each 8 rows
    const bool wide = ((uintptr_t)a.vc & 15u) == 0;
#pragma unroll
    for (uint32_t it = 0; it < 2; ++it) {
        const uint32_t g = (t + 256u * it) & 7u, c = (t + 256u * it) >> 3;
        const uint32_t m = lead[g >> 2] >> (8u * (g & 3u)) & 255u;
        if (!m) continue;
        const uint32_t r = 8u * g + (uint32_t)__builtin_ctz(m);
        const uint16_t* src = &tile[c * TP + r];
        uint16_t* dst = a.vc + v_page_at<D>(a, h, (uint32_t)slots[7 + r], d0 + c);
        if (wide) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (uint32_t)src[2 * e] | (uint32_t)src[2 * e + 1] << 16;
            *reinterpret_cast<u32x4*>(dst) = w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = src[e];
        }
    }
    uint64_t left = (uint64_t)lone[1] << 32 | lone[0];
    for (uint32_t n = 0; left; ++n, left &= left - 1) {  // uniform: each wave takes every fourth
        if (n % 4u != t >> 6) continue;
        const uint32_t r = (uint32_t)__builtin_ctzll(left), c = t & 63u;
        a.vc[v_page_at<D>(a, h, (uint32_t)slots[7 + r], d0 + c)] = tile[c * TP + r];
    }
}

template <uint32_t KIND, int D, uint32_t DT>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkNormRopeArgs a)
{
    // the two roles alternate over the first 2 * min(rotation, V) workgroups (rope.hip)
    uint32_t blk = blockIdx.x;
    {
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
            v_block<D, DT>(a, blk);
            return;
        }
    }
    constexpr uint32_t LPH = D / 8, HPP = 64 / LPH;  // lanes per head, heads per pass
    constexpr uint32_t U = 4;                        // passes whose loads are issued together
    const uint32_t lane = threadIdx.x & 63u, i = lane % LPH, sub = lane / LPH;
    const uint32_t w = blk * 4u + (threadIdx.x >> 6);
    const uint32_t b = w / a.groups, g = w % a.groups;
    if (b >= a.n_tok) return;  // wave-uniform; no barrier follows in this role
    const int slot = slot_of(a, b);
    if (slot < 0) return;
    const int pos = a.positions ? a.positions[b] : (int)(a.pos_start + b);

    // the lane's two runs of four elements, and whether its pairs turn
    const uint32_t half = (KIND == kRopeMrope ? a.n_rot : (uint32_t)D) / 2;
    const bool far = KIND == kRopeHalf || (KIND == kRopeMrope && 4u * i < half);
    const bool turn = KIND == kRopePairs || far;
    const uint32_t e0 = far ? 4u * i : 8u * i, e1 = far ? half + 4u * i : 8u * i + 4u;
    float c[4], s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        c[e] = 1.0f;
        s[e] = 0.0f;
        if (turn) {
            const double u = a.turns[4u * i + e] * (double)pos;
            sincospif(2.0f * (float)(u - __builtin_rint(u)), &s[e], &c[e]);
        }
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

    // this wave's heads: [h_lo, h_hi) of q heads then kv heads (kv heads only without q_out)
    const uint32_t heads = a.n_heads + a.n_kv;
    const uint32_t h_lo = (a.q_out ? 0u : a.n_heads) + g * a.heads_per_wave;
    const uint32_t h_hi = min(heads, h_lo + a.heads_per_wave);
    const size_t krow = k_page_row<D>(a, 0, (uint32_t)slot), kstep = (size_t)a.block * D;  // + h * kstep
    for (uint32_t h0 = h_lo; h0 < h_hi; h0 += HPP * U) {
        // loads of U passes first, then their stores (q_out may be q: every lane reads its own elements before
        // it writes them); past the end a valid head's are loaded again
        f32x4 x[U][2];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t h = min(h0 + u * HPP + sub, h_hi - 1u);
            const bool is_q = h < a.n_heads;
            const void* src = is_q ? a.q : a.k;
            const size_t at = is_q ? (size_t)b * a.q_stride + (size_t)h * D
                                   : (size_t)b * a.k_stride + (size_t)(h - a.n_heads) * D;
            x[u][0] = load4<DT>(src, at + e0);
            x[u][1] = load4<DT>(src, at + e1);
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t h = h0 + u * HPP + sub;
            if (h0 + u * HPP >= h_hi) break;  // wave-uniform
            const bool is_q = h < a.n_heads;
            f32x4 y0 = x[u][0], y1 = x[u][1];
            if (norm) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = fmaf(y0[e], y0[e], fmaf(y1[e], y1[e], ss));
                ss = group_sum<LPH>(ss);
                const float inv = __builtin_amdgcn_rsqf(fmaf(ss, 1.0f / D, a.eps));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y0[e] *= inv * (is_q ? qw[0][e] : kw[0][e]);
                    y1[e] *= inv * (is_q ? qw[1][e] : kw[1][e]);
                }
            }
            if (turn) {
                if (KIND == kRopePairs) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f32x4& y = e < 2 ? y0 : y1;
                        const float p = y[2 * (e & 1)], r = y[2 * (e & 1) + 1];
                        y[2 * (e & 1)] = p * c[e] - r * s[e];
                        y[2 * (e & 1) + 1] = p * s[e] + r * c[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = y0[e], r = y1[e];
                        y0[e] = p * c[e] - r * s[e];
                        y1[e] = p * s[e] + r * c[e];
                    }
                }
            }
            if (h >= h_hi) continue;
            if (is_q) {
                const size_t at = (size_t)b * a.q_out_stride + (size_t)h * D;
                store4(a.q_out, at + e0, a.q_out_dtype, y0);
                store4(a.q_out, at + e1, a.q_out_dtype, y1);
            } else {
                uint16_t* row = a.kc + krow + (h - a.n_heads) * kstep;
                u16x4 k0, k1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    k0[e] = f32_to_f16_ref(y0[e]);
                    k1[e] = f32_to_f16_ref(y1[e]);
                }
                *reinterpret_cast<u16x4*>(row + e0) = k0;
                *reinterpret_cast<u16x4*>(row + e1) = k1;
            }
        }
    }
    if (a.n_tok <= kScatterRows) {
        const uint32_t kv_dim = a.n_kv * D;
        for (uint32_t j = g * 64u + lane; j < kv_dim; j += 64u * a.groups) {
            const size_t at = (size_t)b * a.v_stride + j;
            const uint16_t bits = DT == kF16 ? reinterpret_cast<const uint16_t*>(a.v)[at]
                                             : f32_to_f16_ref(load_as_f32(a.v, at, DT));
            a.vc[v_page_at<D>(a, j / D, (uint32_t)slot, j % D)] = bits;
        }
    }
}

template <uint32_t KIND, int D>
hipError_t launch_dt(const QkNormRopeArgs& a, dim3 grid, hipStream_t st)
{
    switch (a.dtype) {
    case kF32: hipLaunchKernelGGL((qk_norm_rope_kernel<KIND, D, kF32>), grid, dim3(256), 0, st, a); break;
    case kF16: hipLaunchKernelGGL((qk_norm_rope_kernel<KIND, D, kF16>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((qk_norm_rope_kernel<KIND, D, kBF16>), grid, dim3(256), 0, st, a); break;
    }
    return hipGetLastError();
}

template <uint32_t KIND>
hipError_t launch_kind(const QkNormRopeArgs& a, dim3 grid, hipStream_t st)
{
    switch (a.D) {
    case 64: return launch_dt<KIND, 64>(a, grid, st);
    case 128: return launch_dt<KIND, 128>(a, grid, st);
    case 256: return launch_dt<KIND, 256>(a, grid, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_qk_norm_rope(QkNormRopeArgs a, hipStream_t st)
{
    const uint32_t hpp = 64u / (a.D / 8u);
    const uint32_t active = a.q_out ? a.n_heads + a.n_kv : a.n_kv;
    const uint32_t passes = (active + hpp - 1) / hpp;
    const uint32_t per0 = a.n_tok <= kScatterRows ? 1u : 4u;
    const uint32_t groups = (passes + per0 - 1) / per0;
    const uint32_t per = (passes + groups - 1) / groups;  // passes per wave, evenly
    a.heads_per_wave = per * hpp;
    a.groups = (passes + per - 1) / per;
    a.rope_blocks = (uint32_t)(((uint64_t)a.n_tok * a.groups + 3u) / 4u);
    a.v_blocks = a.n_tok > kScatterRows ? a.n_kv * a.D / 64u * ((a.n_tok + 63u) / 64u) : 0u;
    const dim3 grid(a.rope_blocks + a.v_blocks);
    switch (a.kind) {
    case kRopeNone: return launch_kind<kRopeNone>(a, grid, st);
    case kRopePairs: return launch_kind<kRopePairs>(a, grid, st);
    case kRopeHalf: return launch_kind<kRopeHalf>(a, grid, st);
    case kRopeMrope: return launch_kind<kRopeMrope>(a, grid, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace yhip
