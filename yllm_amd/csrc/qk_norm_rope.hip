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
// Each row is read once and written once; few rows are bound by the launch and
// two round trips, many by the latency of their loads: a wave loads its passes,
// waits, computes, stores and ends, and nothing of another row is in flight
// meanwhile.  A lane holds eight elements of a head as two runs of four, with
// neighbouring lanes' runs next to each other (eight in one run left every load
// and store with holes), and the pairs of every rope kind within one lane; so a
// head is D / 8 lanes, a wave takes 64 / (D / 8) heads a pass, and the sum of
// squares is a few DPP steps.  The lane's four sines and cosines serve all its
// passes.  V is stored d-major, in 16-byte groups of eight positions, by
// workgroups of their own (a few rows: by the same waves, 2 bytes at a time).
//
// Measured: 8193 tokens of three prompts, 16 / 2 heads of 256 (M-RoPE over 64),
// bf16: 43.8 us, 3.8 TB/s, where a large copy reaches 5.4 (31 us); 480 VALU
// instructions a wave (some of them 64 bits wide) are 22 us, and 61 % of the wave
// cycles wait.  Three passes a wave and four waves a SIMD: one pass 54 us, two 46,
// five 45; six waves a SIMD spill, 50.  One decode token 4.7 us of GPU time, 64 of
// 32 / 8 heads of 128 6.1.
#include "common.hpp"
#include "internal.hpp"
#include "qk_norm_rope_parts.hpp"

namespace yhip {
namespace {

// Up to this many rows the rotation waves write V too, as in rope.hip.
constexpr uint32_t kScatterRows = 128;

// The value whose truncation to f16 is f32_to_f16_ref(x), without branches:
// half a step of the result is added (to the magnitude's bits where it is
// normal in f16; 2^-25 below, exactly), what rounds past the largest becomes
// inf.  (The general form is some twenty instructions and six branches for each
// element; waves that spent them were bound by them, not by HBM.)
__device__ inline float half_away(float x)
{
    const float a = fabsf(x);
    float t = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) + 0x1000u);
    const float half = 2.98023223876953125e-08f;  // below it, zero (and the sum would round up to the first step)
    t = a < 6.103515625e-05f ? x + copysignf(a < half ? 0.0f : half, x) : t;
    t = a >= 65520.0f ? copysignf(INFINITY, x) : t;
    return x == x ? t : x;
}
__device__ inline u16x4 to_cache4(const f32x4& x)
{
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 w = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(half_away(x[0]), half_away(x[1]))),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(half_away(x[2]), half_away(x[3])))};
    return __builtin_bit_cast(u16x4, w);
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
    for (uint32_t u = 0; u < R / 16; ++u) {
        u16x4 w;
        if constexpr (DT == kF16) {  // f16 rows keep their bits (the widened value is converted back; a NaN's payload apart)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __builtin_bit_cast(uint16_t, (_Float16)x[u][e]);
        } else {
            w = to_cache4(x[u]);
        }
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) tile[(c4 + e) * TP + rr + 16u * u] = w[e];
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
#pragma unroll
    for (uint32_t it = 0; it < 2; ++it) {
        const uint32_t g = (t + 256u * it) & 7u, c = (t + 256u * it) >> 3;
        const uint32_t m = lead[g >> 2] >> (8u * (g & 3u)) & 255u;
        if (!m) continue;
        const uint32_t r = 8u * g + (uint32_t)__builtin_ctz(m);
        const uint16_t* src = &tile[c * TP + r];
        uint16_t* dst = a.vc + v_page_at<D>(a, h, (uint32_t)slots[7 + r], d0 + c);
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (uint32_t)src[2 * e] | (uint32_t)src[2 * e + 1] << 16;
        *reinterpret_cast<u32x4*>(dst) = w;  // (pools are aligned to 16 bytes, checked on the host)
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
    constexpr uint32_t U = 3;                        // passes whose loads are issued together
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
    auto pair_of = [&](uint32_t e) -> uint32_t {  // the pair index of the lane's e-th pair
        return KIND == kRopePairs ? (e < 2 ? 2u * i + e : D / 4 + 2u * i + (e - 2)) : 4u * i + e;
    };

    // This wave's passes: HPP heads each, those of q (none without q_out), then those of k.  A pass is of one kind,
    // so that everything but the lane's offsets is wave-uniform.
    const uint32_t pq = a.q_out ? (a.n_heads + HPP - 1) / HPP : 0u, passes = pq + (a.n_kv + HPP - 1) / HPP;
    const uint32_t p_lo = g * a.passes, p_hi = min(passes, p_lo + a.passes);
    const size_t esz = DT == kF32 ? 4 : 2;
    const char* const qrow = reinterpret_cast<const char*>(a.q) + (size_t)b * a.q_stride * esz;
    const char* const krow = reinterpret_cast<const char*>(a.k) + (size_t)b * a.k_stride * esz;
    const size_t kstep = (size_t)a.block * D;  // between a page's heads
    size_t kpage = 0;
    float c[4], s[4];
    f32x4 qw[2], kw[2];
    const bool norm = a.q_norm != nullptr;
    for (uint32_t p0 = p_lo; p0 < p_hi; p0 += U) {
        // loads of U passes first, then their stores (q_out may be q: every lane reads its own elements before
        // it writes them); heads past the last load it again
        f32x4 x[U][2];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t p = min(p0 + u, p_hi - 1u);
            const bool is_q = p < pq;
            const uint32_t h = min((is_q ? p : p - pq) * HPP + sub, (is_q ? a.n_heads : a.n_kv) - 1u);
            const char* src = is_q ? qrow : krow;
            x[u][0] = load4<DT>(src, h * D + e0);
            x[u][1] = load4<DT>(src, h * D + e1);
        }
        if (p0 == p_lo) {  // once, behind the first loads
            __builtin_amdgcn_sched_barrier(0);
            if (slot < 0) return;  // wave-uniform
            kpage = k_page_row<D>(a, 0, (uint32_t)slot);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[e] = 1.0f;
                s[e] = 0.0f;
                if (turn) sincos_turns(a.turns[pair_of(e)] * (double)pos, &s[e], &c[e]);
            }
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
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t p = p0 + u;
            if (p >= p_hi) break;  // wave-uniform
            const bool is_q = p < pq;
            const uint32_t h = (is_q ? p : p - pq) * HPP + sub;
            f32x4 y0 = x[u][0], y1 = x[u][1];
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
                    const float v = y[2 * (e & 1)], r = y[2 * (e & 1) + 1];
                    y[2 * (e & 1)] = v * c[e] - r * s[e];
                    y[2 * (e & 1) + 1] = v * s[e] + r * c[e];
                }
            } else if (KIND != kRopeNone) {  // (lanes that do not turn have cosine 1 and sine 0)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = y0[e], r = y1[e];
                    y0[e] = KIND == kRopeHalf || turn ? v * c[e] - r * s[e] : v;
                    y1[e] = KIND == kRopeHalf || turn ? v * s[e] + r * c[e] : r;
                }
            }
            if (is_q) {
                if (h < a.n_heads) {
                    const size_t at = (size_t)b * a.q_out_stride + h * D;
                    store4(a.q_out, at + e0, a.q_out_dtype, y0);
                    store4(a.q_out, at + e1, a.q_out_dtype, y1);
                }
            } else if (h < a.n_kv) {
                uint16_t* row = a.kc + kpage + h * kstep;
                *reinterpret_cast<u16x4*>(row + e0) = to_cache4(y0);
                *reinterpret_cast<u16x4*>(row + e1) = to_cache4(y1);
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
    const uint32_t passes = (a.q_out ? (a.n_heads + hpp - 1) / hpp : 0u) + (a.n_kv + hpp - 1) / hpp;
    const uint32_t per0 = a.n_tok <= kScatterRows ? 1u : 3u;
    const uint32_t groups = (passes + per0 - 1) / per0;
    a.passes = (passes + groups - 1) / groups;  // per wave, evenly
    a.groups = (passes + a.passes - 1) / a.passes;
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
