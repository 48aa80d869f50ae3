// paged_decode.hip -- paged attention of sequences with few new tokens: those
// whose tokens of one kv head's query heads fit the 16 columns of a
// 16x16x32 MFMA (decode steps; drafted tokens being checked).
//
// Bound by HBM: every K and V byte is read once, for all of a group's heads
// and tokens together.  The formulation is the contiguous decode's
// (attn_decode.hip): S^T = K.Q^T and O^T += V^T.P^T on v_mfma_f32_16x16x32_f16,
// a wave walks 32-key blocks, K rows loaded in the order that makes its score
// registers the next product's operand, two blocks of fragments in flight per
// wave.  What differs is where the blocks are and how the work is split: the
// batch's (sequence, kv head) items lie on one line of 128-key units, cut into
// equal chunks, one per resident workgroup (paged_items.hpp), so that ragged
// lengths cost no idle time; items cut by a chunk's end are joined by the
// merge kernel.  Page numbers are read a round ahead of the loads they place.
//
// f16 queries are taken as they are, bf16 ones as f16 (exact from 2^-17 up to
// 65504, off by at most 2^-25 below), fp32 ones as f16 hi + lo parts (PREC).  The
// probabilities of all are hi + lo parts: rounded to f16 alone they double the
// variance of an f16 output's error, and the second product is in the shadow of
// the loads (64 sequences of 1024 .. 32768 keys 357 us with it or without).
//
// Measured: 64 sequences of 1024 .. 32768 keys, 32 / 8 heads of 128, 357 us, 6.67
// TB/s; one token over 131072 keys 83 us and a merge of 5, over 320 keys of 28 /
// 4 heads of 128 7.4, of 16 / 2 heads of 256 14.1.  A short call is a chain: 1.6
// us to the piece, 2 to issue two blocks' loads (64 of them at head_dim 256: 4 to
// 6), 1 to 2 for a block and 1.5 to join the waves.
#include "common.hpp"
#include "internal.hpp"
#include "paged_items.hpp"

#include <math.h>

#include <type_traits>

namespace yhip {
namespace {

constexpr uint32_t kUnit = 128;  // keys of a unit: one 32-key block a wave
// an item's fixed cost in units (kItemUnits of the prefill items; here a queue
// of loads that drains and fills again)
constexpr uint32_t kDecodeItemUnits = 1;
constexpr int kRows = 16;

__device__ inline f32x4 mfma16(const f16x8& a, const f16x8& b, const f32x4& c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// the line of units (see PagedLine, the prefill items')
struct DecodeLine {
    static __device__ uint64_t units(const PagedAttnArgs& a, const PagedSeq& s)
    {
        return s.nq ? (uint64_t)a.n_kv * item(s) : 0;
    }
    static __device__ uint32_t item(const PagedSeq& s)
    {
        return kDecodeItemUnits + (s.L > 0 ? ((uint32_t)s.L + kUnit - 1) / kUnit : 1u);
    }
};

// keys [kbeg, kend) of (sequence, kv head); part, last as in PagedItem
struct DecodePiece {
    uint32_t seq, row0, nq, kvh, kbeg, kend, part, last;
    int pos0, L;
};

// the keys that the sequence's last row sees (all, but for tokens left out past max_new)
__device__ inline int seen_keys(const PagedSeq& s) { return max(min(s.L, s.pos0 + (int)s.nq), 0); }

__device__ inline bool decode_next(const PagedAttnArgs& a, PagedCursor& C, DecodePiece& I)
{
    if (C.done >= C.len) return false;
    PagedSeq s = cursor_seq(a, C.seq);
    uint32_t units = (uint32_t)DecodeLine::units(a, s);
    while (C.off >= units) {
        C.off -= units;
        s = cursor_seq(a, ++C.seq);
        units = (uint32_t)DecodeLine::units(a, s);
    }
    const uint32_t T = DecodeLine::item(s);
    const uint32_t kvh = C.off / T;
    uint32_t t = C.off - kvh * T, n;
    if (!paged_cut(a, C, T, t, kDecodeItemUnits, kDecodeItemUnits, n, I.last)) return false;
    I.part = n == T ? 0u : t == 0 ? 1u : 2u;
    I.seq = C.seq;
    I.row0 = s.row0;
    I.nq = s.nq;
    I.kvh = kvh;
    I.pos0 = s.pos0;
    I.L = seen_keys(s);
    const uint32_t u0 = t ? t - kDecodeItemUnits : 0u, u1 = t + n - kDecodeItemUnits;
    I.kbeg = min(u0 * kUnit, (uint32_t)I.L);
    I.kend = min(u1 * kUnit, (uint32_t)I.L);
    return true;
}

// The item of this workgroup where none is cut (short contexts): one each, by
// its number, without the line; false where the sequence brings no token.
__device__ inline bool decode_whole(const PagedAttnArgs& a, DecodePiece& I)
{
    I.seq = blockIdx.x / a.n_kv;
    I.kvh = blockIdx.x - I.seq * a.n_kv;
    const PagedSeq s = cursor_seq(a, I.seq);
    I.row0 = s.row0;
    I.nq = s.nq;
    I.pos0 = s.pos0;
    I.L = seen_keys(s);
    I.kbeg = 0;
    I.kend = (uint32_t)I.L;
    I.part = I.last = 0;
    return s.nq != 0;
}

// one 32-key block of K and V as MFMA operands of one lane
template <int D>
struct Frag {
    f16x8 k[2][D / 32];
    f16x8 v[D / 16];
};

template <int D, bool PREC, int POL>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void paged_decode_kernel(PagedAttnArgs args)
{
    constexpr int kWaves = 4, D4 = D / 4, NC = D / 32, NB = D / 16, QROW = D + 8;
    // each wave's O rows; before the key loop, the queries (hi, lo) [2][16][QROW]
    __shared__ __attribute__((aligned(16))) float s_o[kWaves][kRows][D + 4];
    __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows];
    __shared__ uint32_t s_odd[kWaves];
    _Float16* const s_q = reinterpret_cast<_Float16*>(&s_o[0][0][0]);

    PagedCursor C{};
    DecodePiece I;
    if (args.n_wg == 0) {
        if (!decode_whole(fresh_args(args), I)) return;  // workgroup-uniform
    } else if (!(paged_start<256, DecodeLine>(fresh_args(args), reinterpret_cast<uint64_t*>(&s_o[0][0][0]), C) &&
          decode_next(fresh_args(args), C, I))) {
        if (threadIdx.x == 0) reinterpret_cast<PagedDesc*>(args.desc)[C.j].n = 0;
        return;
    }
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const uint32_t wave = uni(threadIdx.x >> 6);
    const int krow = 8 * (n >> 2) + (n & 3);  // + 4 t for half t
    const uint32_t k_lane = (krow * D + g * 8) * 2, v_lane = (n * kVTile + g * 8) * 2;

    for (;;) {
        const PagedAttnArgs& a = fresh_args(args);
        const uint32_t h0 = head0(a, I.kvh), G = head0(a, I.kvh + 1) - h0, rows = G * I.nq;  // row r: token r / G, head r % G
        const uint32_t nblk = (I.kend - I.kbeg + 31) / 32, nbw = nblk > wave ? (nblk - wave + kWaves - 1) / kWaves : 0;
        const ConstInts table = const_ints(a.table + (size_t)I.seq * a.table_stride);
        // this wave's i-th block: its first key, its page
        auto key_of = [&](uint32_t i) { return I.kbeg + 32u * (wave + kWaves * i); };
        auto page_of = [&](uint32_t i) -> uint32_t { return i < nbw ? (uint32_t)table[key_of(i) >> a.shift] : ~0u; };

        // the queries: loaded from valid rows everywhere (rows past the last take row 0 and are zeroed)
        f32x4 qv[D / 64];
#pragma unroll
        for (int r = 0; r < D / 64; ++r) {
            const uint32_t idx = threadIdx.x + r * 256u, hn = idx / D4, d = idx % D4 * 4u, hr = hn < rows ? hn : 0u;
            const uint32_t t = div_small(hr, G);
            const size_t at = (size_t)(I.row0 + t) * a.q_stride + (size_t)(h0 + hr - t * G) * D + d;
            if (PREC) {
                qv[r] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(a.q) + at);
            } else {
                typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
                const u16x4 w = *reinterpret_cast<const u16x4*>(reinterpret_cast<const uint16_t*>(a.q) + at);
#pragma unroll
                for (int e = 0; e < 4; ++e) qv[r][e] = a.q_dtype == kBF16 ? bf16_bits_to_f32(w[e]) : f16_bits_to_f32(w[e]);
            }
        }
        auto load = [&](Frag<D>& f, uint32_t i, uint32_t page) {
            const PagedTile p = paged_tile<D>(a, page, I.kvh);
            const uint32_t at = p.bytes ? (key_of(i) & ((1u << a.shift) - 1u)) * D * 2 : 0u;
            const __amdgpu_buffer_rsrc_t rK = __builtin_amdgcn_make_buffer_rsrc(
                reinterpret_cast<char*>(const_cast<uint16_t*>(a.kc)) + p.at, 0, p.bytes, 0x00020000);
            const __amdgpu_buffer_rsrc_t rV = __builtin_amdgcn_make_buffer_rsrc(
                reinterpret_cast<char*>(const_cast<uint16_t*>(a.vc)) + p.at, 0, p.bytes, 0x00020000);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    f.k[t][c] = __builtin_bit_cast(
                        f16x8, __builtin_amdgcn_raw_buffer_load_b128(rK, k_lane + (4 * t * D + c * 32) * 2, at, POL));
#pragma unroll
            for (int b = 0; b < NB; ++b)
                f.v[b] = __builtin_bit_cast(
                    f16x8, __builtin_amdgcn_raw_buffer_load_b128(rV, v_lane + b * 16 * (int)kVTile * 2, at, POL));
        };
        Frag<D> f0, f1;
        load(f0, 0, page_of(0));
        load(f1, 1, page_of(1));
        uint32_t page0 = page_of(2), page1 = page_of(3);
        __builtin_amdgcn_sched_barrier(0);  // nothing below waits before these are issued

#pragma unroll
        for (int r = 0; r < D / 64; ++r) {
            const uint32_t idx = threadIdx.x + r * 256u, hn = idx / D4, d = idx % D4 * 4u;
            f16x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = hn < rows ? qv[r][e] : 0.0f;
                hi[e] = (_Float16)x;
                lo[e] = (_Float16)(x - (float)hi[e]);
            }
            *reinterpret_cast<f16x4*>(s_q + hn * QROW + d) = hi;
            if (PREC) *reinterpret_cast<f16x4*>(s_q + (16 + hn) * QROW + d) = lo;
        }
        lds_barrier();
        // (at head_dim 256 the lo parts are read for each block: 32 registers too many)
        constexpr bool LO = PREC && D <= 128;
        auto read_q = [&](int part, int c) {
            return *reinterpret_cast<const f16x8*>(s_q + (16 * part + n) * QROW + c * 32 + g * 8);
        };
        f16x8 qhi[NC], qlo[LO ? NC : 1];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qhi[c] = read_q(0, c);
            if constexpr (LO) qlo[c] = read_q(1, c);
        }

        // row n sees keys below lim; keys from `cut` on are not seen by every row
        const int lim = min(I.pos0 + (int)((uint32_t)n < rows ? div_small((uint32_t)n, G) : 0u) + 1, I.L);
        const int cut = min(I.pos0 + 1, I.L);
        float m = -1e30f, l = 0.0f;
        bool odd = false;  // an inf or NaN was cleared
        f32x4 o[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] = f32x4{0.f, 0.f, 0.f, 0.f};

        // (only a wave's last block can hold keys that some row does not see: there are less than 16)
        auto compute = [&](Frag<D>& f, uint32_t i, auto last) {
            const int key0 = (int)key_of(i);
            f32x4 s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    s[t] = mfma16(f.k[t][c], qhi[c], s[t]);
                    if constexpr (LO) s[t] = mfma16(f.k[t][c], qlo[c], s[t]);
                    else if constexpr (PREC) s[t] = mfma16(f.k[t][c], read_q(1, c), s[t]);
                }
            }
            float x[8];  // row n, key key0 + 8 g + j
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = s[j >> 2][j & 3];
            if (last && key0 + 32 > cut) {  // wave-uniform
                // a value that some row does not see must be finite (0 * inf); those that a row sees are added
                // at the end.  Keys past the last were never stored.  (Two values a register: element by element
                // this took a wave 4 us at head_dim 256, with every other waiting for it.)
                const int key = key0 + 8 * g;
                uint32_t keep[4], hid[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int k0 = key + 2 * w, k1 = k0 + 1;
                    if (k0 >= lim) x[2 * w] = -INFINITY;
                    if (k1 >= lim) x[2 * w + 1] = -INFINITY;
                    keep[w] = (k0 < I.L ? 0xffffu : 0u) | (k1 < I.L ? 0xffff0000u : 0u);
                    hid[w] = (k0 >= cut ? 0x8000u : 0u) | (k1 >= cut ? 0x80000000u : 0u);
                }
                auto each = [&](auto&& fn) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        u32x4 v = __builtin_bit_cast(u32x4, f.v[b]);
#pragma unroll
                        for (int w = 0; w < 4; ++w) v[w] = fn(v[w] & keep[w], w);
                        f.v[b] = __builtin_bit_cast(f16x8, v);
                    }
                };
                if (cut < I.L) {  // wave-uniform
                    uint32_t any = 0;
                    each([&](uint32_t v, int w) {
                        // the top bit of each half where the exponent is all ones (it carries no further)
                        const uint32_t s = ((v & 0x7c007c00u) + 0x04000400u) & hid[w];
                        any |= s;
                        return v & ~(s | (s - (s >> 15)));
                    });
                    odd = odd || any != 0;
                } else {
                    each([](uint32_t v, int) { return v; });
                }
            }
            float mx = x[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mx = fmaxf(mx, x[j]);
            mx = max_xor32(max_xor16(mx)) * a.c;
            if (__ballot(mx > m + (kLift + kSlack))) {
                const float mn = mx > m + (kLift + kSlack) ? mx - kLift : m;
                const float alpha = fast_exp2(m - mn);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= alpha;
            }
            f16x8 pf, pl;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = fast_exp2(fmaf(x[j], a.c, -m));
                l += p;
                pf[j] = (_Float16)p;
                pl[j] = (_Float16)(p - (float)pf[j]);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                o[b] = mfma16(f.v[b], pf, o[b]);
                o[b] = mfma16(bounded(f.v[b]), pl, o[b]);
            }
        };
        uint32_t i = 0;
        for (; i + 2 < nbw; i += 2) {
            compute(f0, i, std::false_type{});
            load(f0, i + 2, page0);
            page0 = page_of(i + 4);
            compute(f1, i + 1, std::false_type{});
            load(f1, i + 3, page1);  // (past the wave's last block: page ~0, zeros without a read)
            page1 = page_of(i + 5);
        }
        if (i < nbw) compute(f0, i, std::true_type{});
        if (i + 1 < nbw) compute(f1, i + 1, std::true_type{});

        l = sum_xor32(sum_xor16(l));
        lds_barrier();  // every wave has read its queries
        if (g == 0) {
            s_m[wave][n] = m;
            s_l[wave][n] = l;
        }
        const bool any_odd = __ballot(odd) != 0;
        if (lane == 0) s_odd[wave] = any_odd;
        if ((uint32_t)n < rows) {
#pragma unroll
            for (int b = 0; b < NB; ++b) *reinterpret_cast<f32x4*>(&s_o[wave][n][b * 16 + 4 * g]) = o[b];
        }
        lds_barrier();
        const PagedAttnArgs& e = fresh_args(args);
        for (uint32_t idx = threadIdx.x; idx < rows * D4; idx += 256u) {
            const uint32_t hn = idx / D4, d = idx % D4 * 4u;
            float mw[kWaves], lw[kWaves];
            f32x4 ow[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                mw[w] = s_m[w][hn];
                lw[w] = s_l[w][hn];
                ow[w] = *reinterpret_cast<const f32x4*>(&s_o[w][hn][d]);
            }
            const float M = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
            f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
            float L = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float c = fast_exp2(mw[w] - M);
                O += ow[w] * c;
                L += lw[w] * c;
            }
            const uint32_t t = div_small(hn, G), h = h0 + hn - t * G;
            if (I.part == 0) O *= L == 0.0f ? 0.0f : 1.0f / L;
            if (s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3]) {
#pragma unroll 1
                for (int k = 0; k < 4; ++k) {
                    const float x = special_sum<D>(e, I.seq, I.kvh, d + k, I.pos0 + (int)t,
                                                   (uint32_t)max((int)I.kbeg, max(cut, 0)), (int)I.kend);
                    O[0] += k == 0 ? x : 0.0f;
                    O[1] += k == 1 ? x : 0.0f;
                    O[2] += k == 2 ? x : 0.0f;
                    O[3] += k == 3 ? x : 0.0f;
                }
            }
            if (I.part == 0) {
                if (e.gate) {
                    const float* gp = e.gate + (size_t)(I.row0 + t) * e.gate_stride + (size_t)h * D + d;
#pragma unroll
                    for (int k = 0; k < 4; ++k) O[k] *= sigmoid_ref(gp[k]);
                }
                store_out4(e.out, (size_t)(I.row0 + t) * e.out_stride + (size_t)h * D + d, e.out_dtype, O);
            } else {
                const size_t slot = (size_t)(2 * C.j + (I.part & 1)) * kRows + hn;
                *reinterpret_cast<f32x4*>(e.part_o + slot * D + d) = O;
                if (d == 0) {
                    e.part_ml[2 * slot] = M;
                    e.part_ml[2 * slot + 1] = L;
                }
            }
        }
        if (fresh_args(args).n_wg == 0) return;
        const uint32_t part = I.part;
        const PagedDesc desc{I.last - C.j + 1, I.row0, I.nq, I.kvh, 0, 0, 0, 0};
        if (!decode_next(fresh_args(args), C, I)) {
            if (threadIdx.x == 0) {
                PagedDesc* dp = reinterpret_cast<PagedDesc*>(fresh_args(args).desc) + C.j;
                if (part == 1) *dp = desc;
                else dp->n = 0;
            }
            return;
        }
        lds_barrier();  // the rows are read before the next piece's queries take their place
    }
}

// Workgroup (j, r): row r of the split item that chunk j begins, if any.
// Thread (s, c) joins pieces s, s + NG, ... of four dimensions, eight loads at
// a time; the NG subsets meet in LDS.
template <int D>
__global__ __launch_bounds__(256) void paged_decode_merge_kernel(PagedAttnArgs a)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t C4 = D / 4, NG = 256 / C4, kRound = 8;
    __shared__ f32x4 s_o[256];
    __shared__ float s_m[256], s_l[256];
    const uint32_t j = blockIdx.x, r = blockIdx.y, t = threadIdx.x;
    const PagedDesc d = reinterpret_cast<const PagedDesc*>(a.desc)[j];
    if (d.n == 0) return;
    const uint32_t h0 = head0(a, d.kvh), G = head0(a, d.kvh + 1) - h0;
    if (r >= G * d.nq) return;
    const uint32_t c4 = t % C4, sg = t / C4, dim = 4 * c4;
    const size_t row = (size_t)(d.row0 + r / G), col = (size_t)(h0 + r % G) * D + dim;
    // the gate is read with the pieces; without one the output row stands in as a valid address
    f32x4 gt = f32x4{0.f, 0.f, 0.f, 0.f};
    if (a.gate) {
        const float* gp = a.gate + row * a.gate_stride + col;
#pragma unroll
        for (int e = 0; e < 4; ++e) gt[e] = gp[e];
    }
    float M = -1e30f, L = 0.0f;
    f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t s0 = sg; s0 < d.n; s0 += NG * kRound) {
        f32x2 ml[kRound];
        f32x4 os[kRound];
#pragma unroll
        for (uint32_t k = 0; k < kRound; ++k) {
            const uint32_t s = s0 + k * NG < d.n ? s0 + k * NG : s0;  // (past the last one: counted as nothing)
            const size_t p = (size_t)(2 * (j + s) + (s == 0)) * kRows + r;
            ml[k] = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * p);
            os[k] = *reinterpret_cast<const f32x4*>(a.part_o + p * D + dim);
        }
        float mr = M;
#pragma unroll
        for (uint32_t k = 0; k < kRound; ++k)
            if (s0 + k * NG < d.n) mr = fmaxf(mr, ml[k][0]);
        const float co = fast_exp2(M - mr);
        L *= co;
        O *= co;
#pragma unroll
        for (uint32_t k = 0; k < kRound; ++k) {
            if (s0 + k * NG >= d.n) continue;
            const float c = fast_exp2(ml[k][0] - mr);
            L += ml[k][1] * c;
            O += os[k] * c;
        }
        M = mr;
    }
    s_o[t] = O;
    s_m[t] = M;
    s_l[t] = L;
    __syncthreads();
    if (t >= C4) return;
    float Mt = s_m[t];
#pragma unroll
    for (uint32_t k = 1; k < NG; ++k) Mt = fmaxf(Mt, s_m[k * C4 + t]);
    float Lt = 0.0f;
    f32x4 Ot = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t k = 0; k < NG; ++k) {
        const float c = fast_exp2(s_m[k * C4 + t] - Mt);
        Lt += s_l[k * C4 + t] * c;
        Ot += s_o[k * C4 + t] * c;
    }
    f32x4 v = Ot * (Lt == 0.0f ? 0.0f : 1.0f / Lt);
    if (a.gate) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= sigmoid_ref(gt[e]);
    }
    store_out4(a.out, row * a.out_stride + col, a.out_dtype, v);
}

// Cutting an item costs two partial results and the merge's launch (4 us).
// Where no item's K and V take more than this many bytes per kv head, none is
// cut: whole and cut, us for one sequence: 14 / 2 heads of 64, 768 keys 7.3 and
// 8.6, 1024 8.6 and 8.7; 28 / 4 of 128, 512 keys 9.1 and 10.3, 640 10.8 and
// 10.4; 16 / 2 of 256, 256 keys 11.7 and 15.0, 384 15.6 and 14.9.  (64 sequences:
// 512 keys at 128 12.7 and 23.8, 256 at 256 13.3 and 19.6.)
constexpr uint32_t kWholeBytes = 256 * 1024;
// On the line, beside longer ones, fewer: there the merge comes anyway and items
// that are not cut make chunks uneven (200 sequences of up to 3000 keys, 14 / 2
// heads of 64: 31.1 us, 37.6 with the bytes above; 64 of up to 2000, 28 / 4 of
// 128: 32.6 and 37.2).
constexpr uint32_t kSnapBytes = 160 * 1024;

uint32_t units_of_bytes(uint32_t bytes, uint32_t D) { return bytes / (4 * D * kUnit); }

size_t align256d(size_t x) { return (x + 255) / 256 * 256; }

// Chunks of a launch: what the GPU holds at once, or all that the bounds can
// fill; 0: none is cut.
uint32_t decode_wgs(uint32_t n_seq, uint32_t max_len, uint32_t n_kv, uint32_t D)
{
    const uint32_t units = (max_len + kUnit - 1) / kUnit;
    if (units <= units_of_bytes(kWholeBytes, D)) return 0;  // no item is cut: a workgroup each
    const uint64_t most = (uint64_t)n_seq * n_kv * (units + kDecodeItemUnits);
    const uint64_t full = (uint64_t)(D <= 128 ? 2 : 1) * (uint64_t)n_cus();
    return (uint32_t)(((most < full ? most : full) + 7) / 8 * 8);
}

size_t decode_bytes(uint32_t wgs, uint32_t D)
{
    if (wgs == 0) return 0;
    const size_t rows = (size_t)2 * wgs * kRows;
    return align256d((size_t)wgs * sizeof(PagedDesc)) + align256d(rows * 2 * sizeof(float)) + rows * D * sizeof(float);
}

template <int D, bool PREC>
void launch_decode_pieces(const PagedAttnArgs& a, bool stream, hipStream_t st)
{
    const dim3 grid(a.n_wg ? a.n_wg : a.n_seq * a.n_kv);
    if (stream)
        hipLaunchKernelGGL((paged_decode_kernel<D, PREC, 2>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((paged_decode_kernel<D, PREC, 0>), grid, dim3(256), 0, st, a);
}

}  // namespace

bool paged_decode_fits(uint32_t n_heads, uint32_t n_kv, uint32_t max_new)
{
    return (uint64_t)((n_heads + n_kv - 1) / n_kv) * max_new <= (uint64_t)kRows;
}

size_t paged_decode_workspace(uint32_t n_seq, uint32_t max_len, uint32_t n_kv, uint32_t D)
{
    return decode_bytes(decode_wgs(n_seq, max_len, n_kv, D), D);
}

hipError_t launch_paged_decode(const PagedAttnArgs& in, hipStream_t st)
{
    PagedAttnArgs a = in;
    a.gmax = (a.n_heads + a.n_kv - 1) / a.n_kv;
    a.n_wg = decode_wgs(a.n_seq, a.max_len, a.n_kv, a.D);
    a.snap_units = units_of_bytes(kSnapBytes, a.D);
    a.min_units = 1 + kDecodeItemUnits;
    char* p = reinterpret_cast<char*>(a.ws);
    a.desc = p;
    p += align256d((size_t)a.n_wg * sizeof(PagedDesc));
    a.part_ml = reinterpret_cast<float*>(p);
    a.part_o = reinterpret_cast<float*>(p + align256d((size_t)2 * a.n_wg * kRows * 2 * sizeof(float)));
    // non-temporal loads where the batch reads more than the caches keep (attn_decode.hip; an upper bound)
    const bool stream = (uint64_t)a.n_seq * a.n_kv * a.max_len * a.D * 4u >= (32ull << 20);
    const bool prec = a.q_dtype == kF32;
    switch (a.D) {
    case 64: prec ? launch_decode_pieces<64, true>(a, stream, st) : launch_decode_pieces<64, false>(a, stream, st); break;
    case 128: prec ? launch_decode_pieces<128, true>(a, stream, st) : launch_decode_pieces<128, false>(a, stream, st); break;
    case 256: prec ? launch_decode_pieces<256, true>(a, stream, st) : launch_decode_pieces<256, false>(a, stream, st); break;
    default: return hipErrorInvalidValue;
    }
    if (a.n_wg) {
        const dim3 grid(a.n_wg, a.gmax * a.max_new);
        switch (a.D) {
        case 64: hipLaunchKernelGGL(paged_decode_merge_kernel<64>, grid, dim3(256), 0, st, a); break;
        case 128: hipLaunchKernelGGL(paged_decode_merge_kernel<128>, grid, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL(paged_decode_merge_kernel<256>, grid, dim3(256), 0, st, a); break;
        }
    }
    return hipGetLastError();
}

}  // namespace yhip
