// paged_decode8.hpp -- attention over the 8-bit KV pool (kv8.hpp) for sequences
// with few new tokens, in blocks of 16 rows (the columns of a 16x16x32 MFMA): a
// kv head's query heads' tokens, token by token.
//
// Bound by HBM: K and V are read once for all heads and tokens of a row block.
//   S^T[key][row] = K . Q^T,  O^T[d][row] += V^T . P^T   (v_mfma_f32_16x16x32_f16)
// A wave walks 64-key blocks, two in flight.  Codes come as 16-byte loads: of K
// sixteen dimensions of a key, two k-slots of the product (Q is laid out to
// match); of V sixteen positions of a dimension.  The key of MFMA a's row m is
// 16 (m / 4) + 4 a + m % 4, which makes lane group g's sixteen scores of a row
// those of keys 16 g .. 16 g + 15: in registers exactly the second product's
// operand beside V's load.  Codes become f16 in registers, exactly: K's by the
// conversion that takes its row's scale (v_cvt_scalef32_pk_f16_fp8), V's by the
// same with 1 and a packed product with the positions' factors.
//
// Measured: 64 sequences of 1k to 32k keys, 32 / 8 heads of 128, bf16: 190 us, 6.3
// TB/s (f16 pages 357); fp32 queries 203; 16 / 2 of 256 108, 14 / 2 of 64 35; one
// context of 131072 keys 47 us, 5.7 TB/s, and 4.5 for its merge.  At head_dim 256
// only one V block is in flight and vmcnt's 63 loads bound K: 5.6 TB/s.
//
// The work is dealt out as in paged_decode.hip, in units of 256 keys, to the
// workgroups of a launch of their own (paged_decode8.hip) or to some of those
// that walk the same batch's tiles (attn_paged.hip).
#pragma once

#include "common.hpp"
#include "internal.hpp"
#include "kv8.hpp"
#include "paged_decode8_lds.hpp"
#include "paged_items8.hpp"

namespace yhip {
namespace {

constexpr uint32_t kUnit8 = 256;      // keys of a unit: one 64-key block a wave
constexpr uint32_t kItem8Units = 1;   // an item's fixed cost
constexpr int kRows = kDecode8Rows;

__device__ inline f32x4 mfma16(const f16x8& a, const f16x8& b, const f32x4& c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

struct Decode8Line {
    static __device__ uint32_t blocks(const PagedAttnArgs& a, const PagedSeq& s) { return (a.gmax * s.nq + kRows - 1) / kRows; }
    static __device__ uint64_t units(const PagedAttnArgs& a, const PagedSeq& s)
    {
        return few_rows(static_cast<const PagedAttn8Args&>(a), s) ? (uint64_t)a.n_kv * blocks(a, s) * item(s) : 0;
    }
    static __device__ uint32_t item(const PagedSeq& s)
    {
        return kItem8Units + (s.L > 0 ? ((uint32_t)s.L + kUnit8 - 1) / kUnit8 : 1u);
    }
};

// keys [kbeg, kend) of row block rb of (sequence, kv head); part, last as in PagedItem
struct Decode8Piece {
    uint32_t seq, row0, nq, kvh, rb, kbeg, kend, part, last;
    int pos0, L;
};

// The rows of a piece: `rows` of them, row r being row r0 + r of the kv head's G * nq, token (r0 + r) / G
struct Decode8Rows {
    uint32_t h0, G, r0, rows;
    __device__ uint32_t token(uint32_t r) const { return div_small(r0 + r, G); }
};
__device__ inline Decode8Rows rows_of(const PagedAttnArgs& a, uint32_t kvh, uint32_t rb, uint32_t nq)
{
    Decode8Rows w;
    w.h0 = head0(a, kvh);
    w.G = head0(a, kvh + 1) - w.h0;
    w.r0 = rb * kRows;
    w.rows = (uint32_t)max(min((int)(w.G * nq - w.r0), kRows), 0);
    return w;
}

// the keys that the block's last row sees
__device__ inline int seen_keys(const PagedAttnArgs& a, const Decode8Piece& I, const PagedSeq& s)
{
    const Decode8Rows w = rows_of(a, I.kvh, I.rb, s.nq);
    return w.rows ? max(min(s.L, s.pos0 + (int)w.token(w.rows - 1) + 1), 0) : 0;
}

__device__ inline bool decode8_next(const PagedAttnArgs& a, PagedCursor& C, Decode8Piece& I)
{
    for (;;) {
        if (C.done >= C.len) return false;
        PagedSeq s = cursor_seq(a, C.seq);
        uint32_t units = (uint32_t)Decode8Line::units(a, s);  // (below 2^31, checked on the host)
        while (C.off >= units) {
            C.off -= units;
            s = cursor_seq(a, ++C.seq);
            units = (uint32_t)Decode8Line::units(a, s);
        }
        const uint32_t T = Decode8Line::item(s), nb = Decode8Line::blocks(a, s);
        const uint32_t it = C.off / T;
        uint32_t t = C.off - it * T, n;
        I.kvh = it / nb;
        I.rb = it - I.kvh * nb;
        if (!paged_cut(a, C, T, t, kItem8Units, kItem8Units, n, I.last)) return false;
        I.L = seen_keys(a, I, s);
        if (rows_of(a, I.kvh, I.rb, s.nq).rows == 0) continue;  // a block of the fullest group that this one does not have
        I.part = n == T ? 0u : t == 0 ? 1u : 2u;
        I.seq = C.seq;
        I.row0 = s.row0;
        I.nq = s.nq;
        I.pos0 = s.pos0;
        const uint32_t u0 = t ? t - kItem8Units : 0u, u1 = t + n - kItem8Units;
        I.kbeg = min(u0 * kUnit8, (uint32_t)I.L);
        I.kend = min(u1 * kUnit8, (uint32_t)I.L);
        return true;
    }
}

// The item of this workgroup where none is cut (short contexts): one each, by
// its number, without the line; false where there is none.
__device__ inline bool decode8_whole(const PagedAttn8Args& a, uint32_t wg, Decode8Piece& I)
{
    const uint32_t nb = (min(a.gmax * a.max_new, a.few) + kRows - 1) / kRows, w = wg / nb;
    I.rb = wg - w * nb;
    I.seq = w / a.n_kv;
    I.kvh = w - I.seq * a.n_kv;
    const PagedSeq s = cursor_seq(a, I.seq);
    if (!few_rows(a, s) || rows_of(a, I.kvh, I.rb, s.nq).rows == 0) return false;
    I.row0 = s.row0;
    I.nq = s.nq;
    I.pos0 = s.pos0;
    I.L = seen_keys(a, I, s);
    I.kbeg = 0;
    I.kend = (uint32_t)I.L;
    I.part = I.last = 0;
    return true;
}

// Of a launch for both kinds of sequences, the workgroups of each line; those of the few are the first
struct Mixed8Share {
    uint32_t few, tiles;
};
// Shares go by what the lines cost.  Beside tiles a unit of the few (256 keys, HBM) takes as long as two of the tiles' (64
// keys of 128 rows, MFMA); the more of them there are, the longer the tiles wait for memory as well, down to 1.25 of
// theirs for three few of four units (at 0.75, 1, 1.5, 2, 3 throughout, us: 28 / 4 heads of 128, a tenth of the units few
// 102, 97, 90, 86, 88; 64 in a hundred 187, 173, 167, 169, 197; 32 / 8, three of four 281, 255, 257, 286, 346).  In eights:
// a chunk's XCD goes by its number.  `scratch`: 8 words of LDS, free again after the last barrier.
template <int NT>
__device__ inline Mixed8Share mixed8_share(const PagedMixed8Args& a, uint64_t* scratch)
{
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const bool small = a.n_seq <= 64u;  // every wave adds for itself
    uint64_t few = 0, tiles = 0;
    for (uint32_t i = small ? lane : t; i < a.n_seq; i += small ? 64u : NT) {
        const PagedSeq s = paged_seq(a, a.cu_new[i], a.cu_new[i + 1], a.kv_lens[i]);
        few += Decode8Line::units(a, s);
        tiles += Paged8Line::units(a, s);
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        few += __shfl_xor((unsigned long long)few, d);
        tiles += __shfl_xor((unsigned long long)tiles, d);
    }
    if (!small) {
        if (lane == 0) {
            scratch[2 * wave] = few;
            scratch[2 * wave + 1] = tiles;
        }
        __syncthreads();
        few = tiles = 0;
#pragma unroll
        for (uint32_t w = 0; w < NT / 64; ++w) {
            few += scratch[2 * w];
            tiles += scratch[2 * w + 1];
        }
        __syncthreads();
    }
    few = uni64(few);
    tiles = uni64(tiles);
    if (few == 0) return {0, min(gridDim.x, a.n_wg)};
    if (tiles == 0) return {min(gridDim.x, a.part.n_wg), 0};
    const float part = (float)few / ((float)few + (float)tiles), f = (2.0f - part) * part;
    const uint32_t eights = gridDim.x / 8u, want = (uint32_t)((float)eights * (f / (f + 1.0f - part)) + 0.5f);
    const uint32_t n = min(8u * max(min(want, eights - 1u), 1u), a.part.n_wg);
    return {n, min(gridDim.x - n, a.n_wg)};
}

// one 64-key block of K and V as loaded by a lane: of MFMA a's key the dimensions 64 c + 16 g .. + 15; of dimension
// 16 b + n the positions 16 g .. + 15; and sixteen scales of each
template <int D>
struct FragK8 {
    u32x4 k[4][D / 64], s;
};
template <int D>
struct FragV8 {
    u32x4 v[D / 16], s;
};

// The pieces of workgroup `wg` of `n_wg` (0: its whole item).  lds(w): wave w's share, kDecode8Lds floats, 16-byte aligned
// (the shares may lie anywhere); lds(0) takes the line's scratch and then the queries as well, (hi, lo) [2][16][D + 8], or
// their hi part alone for 16-bit ones.
template <int D, bool PREC, int POL, class A, class Lds>
__device__ __forceinline__ void decode8_pieces(const A& args, uint32_t wg, uint32_t n_wg, Lds lds)
{
    constexpr int kWaves = 4, D4 = D / 4, NC = D / 64, NB = D / 16, QROW = D + 8;
    static_assert((PREC ? 2 : 1) * kRows * QROW * sizeof(_Float16) <= kDecode8Lds<D, PREC> * sizeof(float) &&
                  24 * sizeof(uint64_t) <= kDecode8Lds<D, PREC> * sizeof(float), "the first share holds the queries and the scratch");
    // (head_dim 256: one block of V at a time, the next one's loads go out behind its products; two are too many registers)
    constexpr bool ONE = D > 128;
    auto s_o = [&](int w, uint32_t r, uint32_t d) { return lds(w) + r * (D + 4) + d; };
    auto s_m = [&](int w) { return lds(w) + kRows * (D + 4); };
    auto s_l = [&](int w) { return lds(w) + kRows * (D + 5); };
    auto s_odd = [&](int w) { return reinterpret_cast<uint32_t*>(lds(w) + kRows * (D + 6)); };
    _Float16* const s_q = reinterpret_cast<_Float16*>(lds(0));

    PagedCursor C{};
    Decode8Piece I;
    if (n_wg == 0) {
        if (!decode8_whole(fresh_args(args), wg, I)) return;  // workgroup-uniform
    } else if (!(paged_start<256, Decode8Line>(fresh_args(args), reinterpret_cast<uint64_t*>(s_q), C, wg, n_wg) &&
          decode8_next(fresh_args(args), C, I))) {
        if (threadIdx.x == 0) reinterpret_cast<PagedDesc*>(args.desc)[C.j].n = 0;
        return;
    }
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const uint32_t wave = uni(threadIdx.x >> 6);
    const int krow = 16 * (n >> 2) + (n & 3);  // + 4 a for MFMA a
    const uint32_t k_lane = krow * D + g * 16, v_lane = n * kV8Tile + g * 16;

    for (;;) {
        const PagedAttn8Args& a = fresh_args(args);
        const Decode8Rows W = rows_of(a, I.kvh, I.rb, I.nq);
        const uint32_t nblk = (I.kend - I.kbeg + 63) / 64, nbw = nblk > wave ? (nblk - wave + kWaves - 1) / kWaves : 0;
        const ConstInts table = const_ints(a.table + (size_t)I.seq * a.table_stride);
        // this wave's i-th block: its first key, its page
        auto key_of = [&](uint32_t i) { return I.kbeg + 64u * (wave + kWaves * i); };
        auto page_of = [&](uint32_t i) -> uint32_t { return i < nbw ? (uint32_t)table[key_of(i) >> a.shift] : ~0u; };

        // the queries: loaded from valid rows everywhere (rows past the last take row 0 and are zeroed)
        f32x4 qv[D / 64];
#pragma unroll
        for (int r = 0; r < D / 64; ++r) {
            const uint32_t idx = threadIdx.x + r * 256u, hn = idx / D4, d = idx % D4 * 4u, hr = hn < W.rows ? hn : 0u;
            const uint32_t t = W.token(hr);
            const size_t at = (size_t)(I.row0 + t) * a.q_stride + (size_t)(W.h0 + W.r0 + hr - t * W.G) * D + d;
            if (PREC) {
                qv[r] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(a.q) + at);
            } else {
                typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
                const u16x4 w = *reinterpret_cast<const u16x4*>(reinterpret_cast<const uint16_t*>(a.q) + at);
#pragma unroll
                for (int e = 0; e < 4; ++e) qv[r][e] = a.q_dtype == kBF16 ? bf16_bits_to_f32(w[e]) : f16_bits_to_f32(w[e]);
            }
        }
        auto rsrc = [&](const void* base, uint64_t at, uint32_t bytes) {
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(reinterpret_cast<const char*>(base)) + at, 0, bytes, 0x00020000);
        };
        // block i, in page `page` (outside the pool: no bytes, zeros are read); all but 4 KB of what a load adds to its
        // lane's place is scalar, or every load keeps a register of its own for its address
        auto load_k = [&](FragK8<D>& f, uint32_t i, uint32_t page) {
            const Paged8Tile p = paged8_tile(a, page, I.kvh);
            const uint32_t at = p.bytes ? key_of(i) & ((1u << a.shift) - 1u) : 0u;
            const __amdgpu_buffer_rsrc_t r = rsrc(a.kc, p.at * D, p.bytes * D);
            f.s = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc(a.ks, p.at, p.bytes), (n >> 2) * 16, at, POL));
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    f.k[q][c] = __builtin_bit_cast(
                        u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, k_lane + c * 64, at * D + 4 * q * D, POL));
        };
        auto load_v = [&](FragV8<D>& f, uint32_t i, uint32_t page) {
            const Paged8Tile p = paged8_tile(a, page, I.kvh);
            const uint32_t at = p.bytes ? key_of(i) & ((1u << a.shift) - 1u) : 0u;
            const __amdgpu_buffer_rsrc_t r = rsrc(a.vc, p.at * D, p.bytes * D);
            f.s = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc(a.vs, p.at, p.bytes), g * 16, at, POL));
#pragma unroll
            for (int b = 0; b < NB; ++b)
                f.v[b] = __builtin_bit_cast(
                    u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, v_lane + (b & 3) * 16 * kV8Tile,
                                                                 at * D + (b >> 2) * 64 * kV8Tile, POL));
        };
        FragK8<D> k0, k1;
        FragV8<D> v0, v1;
        load_k(k0, 0, page_of(0));
        load_v(v0, 0, page_of(0));
        load_k(k1, 1, page_of(1));
        if constexpr (!ONE) load_v(v1, 1, page_of(1));
        uint32_t page0 = page_of(2), page1 = page_of(3);
        __builtin_amdgcn_sched_barrier(0);  // nothing below waits before these are issued

#pragma unroll
        for (int r = 0; r < D / 64; ++r) {
            const uint32_t idx = threadIdx.x + r * 256u, hn = idx / D4, d = idx % D4 * 4u;
            f16x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = hn < W.rows ? qv[r][e] : 0.0f;
                hi[e] = (_Float16)x;
                lo[e] = (_Float16)(x - (float)hi[e]);
            }
            *reinterpret_cast<f16x4*>(s_q + hn * QROW + d) = hi;
            if (PREC) *reinterpret_cast<f16x4*>(s_q + (16 + hn) * QROW + d) = lo;
        }
        lds_barrier();
        // k-slot c / 2 of a load's halves c % 2
        constexpr bool LO = PREC && D <= 128;
        auto read_q = [&](int part, int c) {
            return *reinterpret_cast<const f16x8*>(s_q + (16 * part + n) * QROW + (c >> 1) * 64 + g * 16 + (c & 1) * 8);
        };
        f16x8 qhi[2 * NC], qlo[LO ? 2 * NC : 1];
#pragma unroll
        for (int c = 0; c < 2 * NC; ++c) {
            qhi[c] = read_q(0, c);
            if constexpr (LO) qlo[c] = read_q(1, c);
        }

        // row n sees keys below lim; keys from `cut` on are not seen by every row
        const int lim = min(I.pos0 + (int)((uint32_t)n < W.rows ? W.token((uint32_t)n) : W.token(0)) + 1, I.L);
        const int cut = min(I.pos0 + (int)W.token(0) + 1, I.L);
        float m = -1e30f, l = 0.0f;
        bool odd = false;  // a NaN was cleared
        f32x4 o[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] = f32x4{0.f, 0.f, 0.f, 0.f};

        // (only a wave's last block can hold keys that some row does not see: they are among the last 16)
        auto compute = [&](FragK8<D>& fk, FragV8<D>& fv, uint32_t i, auto last, auto&& refill) {
            const int key0 = (int)key_of(i);
            f32x4 s[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float scale = kv8_scale(fk.s[q] >> 8 * (n & 3) & 0xffu);
                s[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2 * NC; ++c) {
                    const u32x4& w = fk.k[q][c >> 1];
                    const f16x8 k = kv8_values(w[2 * (c & 1)], w[2 * (c & 1) + 1], scale);
                    s[q] = mfma16(k, qhi[c], s[q]);
                    if constexpr (LO) s[q] = mfma16(k, qlo[c], s[q]);
                    else if constexpr (PREC) s[q] = mfma16(k, read_q(1, c), s[q]);
                }
            }
            if constexpr (ONE) refill();
            float x[16];  // row n, key key0 + 16 g + j
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = s[j >> 2][j & 3];
            if (last && key0 + 64 > cut) {  // wave-uniform
                // what a row does not see must not make its sums NaN: codes and scales past the last key were never
                // stored, and a NaN that some row does not see is cleared here and added at the end to those that do
                const int key = key0 + 16 * g;
                u32x4 keep, hid;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t kp = 0, hd = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int k = key + 4 * w + e;
                        if (k >= lim) x[4 * w + e] = -INFINITY;
                        kp |= k < I.L ? 0xffu << 8 * e : 0u;
                        hd |= k >= cut ? 0x80u << 8 * e : 0u;
                    }
                    keep[w] = kp;
                    hid[w] = hd;
                }
                fv.s &= keep;
                uint32_t any = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t v = fv.v[b][w] & keep[w], t = kv8_nans(v) & hid[w];
                        any |= t;
                        fv.v[b][w] = v & ~(t | (t - (t >> 7)));
                    }
                odd = odd || any != 0;
            }
            float mx = x[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) mx = fmaxf(mx, x[j]);
            mx = max_xor32(max_xor16(mx)) * a.c;
            if (__ballot(mx > m + (kLift + kSlack))) {
                const float mn = mx > m + (kLift + kSlack) ? mx - kLift : m;
                const float alpha = fast_exp2(m - mn);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= alpha;
            }
            f16x8 pf[2], pl[2];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float p = fast_exp2(fmaf(x[j], a.c, -m));
                l += p;
                pf[j >> 3][j & 7] = (_Float16)p;
                pl[j >> 3][j & 7] = (_Float16)(p - (float)pf[j >> 3][j & 7]);
            }
            f16x2 fac[2][4];
#pragma unroll
            for (int w = 0; w < 8; ++w) fac[w >> 2][w & 3] = kv8_factors(fv.s[w >> 1], w & 1);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f16x8 v = kv8_values(fv.v[b][2 * h], fv.v[b][2 * h + 1], fac[h]);
                    o[b] = mfma16(v, pf[h], o[b]);
                    o[b] = mfma16(v, pl[h], o[b]);
                }
        };
        auto none = [] {};
        uint32_t i = 0;
        // (past the wave's last block: page ~0, zeros without a read)
        if constexpr (ONE) {
            uint32_t page2 = page0, page_v = page_of(1);  // of K(i + 2), K(i + 3) and V(i + 1)
            for (; i + 2 < nbw; i += 2) {
                compute(k0, v0, i, std::false_type{}, [&] { load_k(k0, i + 2, page2); });
                load_v(v0, i + 1, page_v);
                page_v = page2;
                page2 = page_of(i + 4);
                compute(k1, v0, i + 1, std::false_type{}, [&] { load_k(k1, i + 3, page1); });
                load_v(v0, i + 2, page_v);
                page_v = page1;
                page1 = page_of(i + 5);
            }
            if (i < nbw) {
                compute(k0, v0, i, std::true_type{}, none);
                if (i + 1 < nbw) {
                    load_v(v0, i + 1, page_v);
                    compute(k1, v0, i + 1, std::true_type{}, none);
                }
            }
        } else {
            for (; i + 2 < nbw; i += 2) {
                compute(k0, v0, i, std::false_type{}, none);
                load_k(k0, i + 2, page0);
                load_v(v0, i + 2, page0);
                page0 = page_of(i + 4);
                compute(k1, v1, i + 1, std::false_type{}, none);
                load_k(k1, i + 3, page1);
                load_v(v1, i + 3, page1);
                page1 = page_of(i + 5);
            }
            if (i < nbw) compute(k0, v0, i, std::true_type{}, none);
            if (i + 1 < nbw) compute(k1, v1, i + 1, std::true_type{}, none);
        }

        l = sum_xor32(sum_xor16(l));
        lds_barrier();  // every wave has read its queries
        if (g == 0) {
            s_m(wave)[n] = m;
            s_l(wave)[n] = l;
        }
        const bool any_odd = __ballot(odd) != 0;
        if (lane == 0) *s_odd(wave) = any_odd;
        if ((uint32_t)n < W.rows) {
#pragma unroll
            for (int b = 0; b < NB; ++b) *reinterpret_cast<f32x4*>(s_o(wave, n, b * 16 + 4 * g)) = o[b];
        }
        lds_barrier();
        const PagedAttn8Args& e = fresh_args(args);
        for (uint32_t idx = threadIdx.x; idx < W.rows * D4; idx += 256u) {
            const uint32_t hn = idx / D4, d = idx % D4 * 4u;
            float mw[kWaves], lw[kWaves];
            f32x4 ow[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                mw[w] = s_m(w)[hn];
                lw[w] = s_l(w)[hn];
                ow[w] = *reinterpret_cast<const f32x4*>(s_o(w, hn, d));
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
            const uint32_t t = W.token(hn), h = W.h0 + W.r0 + hn - t * W.G;
            if (I.part == 0) O *= L == 0.0f ? 0.0f : 1.0f / L;
            if (*s_odd(0) | *s_odd(1) | *s_odd(2) | *s_odd(3)) {
                const uint32_t nan = nan_dims<D>(e, I.seq, I.kvh, d, I.pos0 + (int)t, (uint32_t)max((int)I.kbeg, max(cut, 0)),
                                                 (int)I.kend);
#pragma unroll
                for (int k = 0; k < 4; ++k) O[k] = nan >> k & 1u ? NAN : O[k];
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
        if (n_wg == 0) return;
        const uint32_t part = I.part;
        const PagedDesc desc{I.last - C.j + 1, I.row0, I.nq, I.kvh, 0, I.rb, 0, 0};
        if (!decode8_next(fresh_args(args), C, I)) {
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

// Row r of the split item that chunk j begins, if any, by a workgroup whose
// thread (s, c) joins pieces s, s + NG, ... of four dimensions, eight loads at
// a time; the NG subsets meet in LDS.
template <int D>
__device__ __forceinline__ void decode8_merge(const PagedAttn8Args& a, uint32_t j, uint32_t r)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t C4 = D / 4, NG = 256 / C4, kRound = 8;
    __shared__ f32x4 s_o[256];
    __shared__ float s_m[256], s_l[256];
    const uint32_t t = threadIdx.x;
    const PagedDesc d = reinterpret_cast<const PagedDesc*>(a.desc)[j];
    if (d.n == 0) return;
    const Decode8Rows W = rows_of(a, d.kvh, d.qb, d.nq);
    if (r >= W.rows) return;
    const uint32_t c4 = t % C4, sg = t / C4, dim = 4 * c4, tok = W.token(r);
    const size_t row = (size_t)(d.row0 + tok), col = (size_t)(W.h0 + W.r0 + r - tok * W.G) * D + dim;
    f32x4 gt = f32x4{0.f, 0.f, 0.f, 0.f};  // the gate is read with the pieces
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

}  // namespace
}  // namespace yhip
