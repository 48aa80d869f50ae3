// prefill_kernel.hpp -- the kernels of causal grouped-query attention for a
// batch of prompt tokens on gfx950 MFMA (launchers: attn_prefill.hip).
//
// Semantics: engine.c:532-563 (token b at position pos_start+b attends to
// keys 0..pos_start+b; scores scaled by 1/sqrt(d); softmax; weighted V),
// with the optional qwen35 sigmoid gate (engine.c:959-960).
//
// Tiling.  A work item is 128 consecutive queries of one query head; each
// of the workgroup's 4-wave key groups (one or two, see prefill_groups)
// gives wave w 32 of them.  Keys stream through LDS in tiles of 64 (K rows
// [64][D] and V^T [D][64], straight from the cache layout), loaded from HBM
// directly into LDS -- K two tiles ahead, V one -- as unpadded rows with
// XOR-swizzled 16-byte chunks.  With two groups, group g takes tiles g,
// g+2, ... and the partial (max, sum, O) of the groups merge through LDS at
// the end.  Items are taken heaviest (latest queries) first so the causal
// triangle drains evenly; with one 8-wave workgroup per CU the grid is the
// resident workgroups, each walking its items in snake order with the next
// item's first loads issued during the current item's last key step.
//
// MFMA formulation (v_mfma_f32_32x32x16_f16), everything transposed so that a
// lane owns one query for the whole kernel:
//   S^T[key][q] = K[key][:] . Q^T[:][q]        A = K tile (LDS), B = Q (regs)
//   O^T[d][q]  += V^T[d][key] . P^T[key][q]    A = V^T tile (LDS), B = P (regs)
// Softmax statistics of a query are in one lane pair (l, l+32): row max over
// a tile is 31 in-lane maxes and one exchange, the running sum is per lane
// until the end.  K rows are written to LDS with rows 4..7 and 8..11 of every
// 16 swapped, which turns the 32x32 accumulator layout (rows 8(i/4)+4(l/32)+
// i%4) into contiguous key runs 8(l/32)+i: the score registers are then
// exactly the k-slots of the P^T operand and P stays in registers.
// Scores use exp2 with log2(e)/sqrt(d) folded into one multiply.
#pragma once

#include "common.hpp"
#include "internal.hpp"
#include "paged_items.hpp"
#include "paged_decode8.hpp"
#include "paged_items8.hpp"

#include <math.h>

#include <type_traits>

namespace yhip {
namespace {

constexpr int BM = 128;  // queries per workgroup
// Keys per tile: 64 up to head_dim 128; 32 at 256, so that a workgroup's
// double-buffered K and V tiles take 64 KB of LDS and two workgroups (two
// waves per SIMD) fit on a CU.
__host__ __device__ constexpr int bn_of(int D) { return D > 128 ? 32 : 64; }

__device__ inline f32x16 mfma32(const f16x8& a, const f16x8& b, const f32x16& c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// key row r of a tile lives in LDS row perm(r): rows 4..7 <-> 8..11 of each 16
__device__ inline int lds_row_of_key(int r)
{
    return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1);
}

// key (within a 32-key half) of accumulator element i for lane half hh
__device__ inline int key_of_acc(int i, int hh) { return i < 8 ? 8 * hh + i : 16 + 8 * hh + (i - 8); }

// 8 bf16 queries, as loaded, to f16
__device__ inline void bf16_to_f16(f16x8& q)
{
    const u32x4 w = __builtin_bit_cast(u32x4, q);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q[2 * j] = (_Float16)__builtin_bit_cast(float, w[j] << 16);
        q[2 * j + 1] = (_Float16)__builtin_bit_cast(float, w[j] & 0xffff0000u);
    }
}

// 8 fp32 query elements as f16 hi + lo parts: hi = f16(x), lo = f16(x - hi),
// so hi + lo carries ~22 bits of x and K.hi + K.lo (two MFMAs into one fp32
// accumulator) keeps the score at fp32-level error
__device__ inline void split_q8(f16x8& hi, f16x8& lo, const f32x4& a, const f32x4& b)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        hi[j] = (_Float16)a[j];
        lo[j] = (_Float16)(a[j] - (float)hi[j]);
        hi[j + 4] = (_Float16)b[j];
        lo[j + 4] = (_Float16)(b[j] - (float)hi[j + 4]);
    }
}

// One 16-byte HBM -> LDS load per lane: lane i writes at lds + 16 i.  A
// __device__ function, not a lambda: lambdas in a kernel are host-device, and
// the host compilation pass silently drops a kernel whose lambdas call this
// gfx950-only builtin.
__device__ inline void lds_load16(__amdgpu_buffer_rsrc_t r, _Float16* lds, int voff, uint32_t soff)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voff, soff, 0, 0);
}

// 16-byte chunk swizzle of an LDS tile row (XOR into the chunk index).  For
// rows of 8 chunks (128 B) the swizzle is (r & 7) ^ bit 3 of r: 8 consecutive
// rows then hit 8 distinct chunk columns (32-bank LDS, b128 reads in groups
// of 8 lanes) and 16 consecutive rows give each half of a 256-byte bank
// window 8 distinct columns (64 banks, groups of 16 lanes).  Rows of 4
// chunks (64 B, the V^T rows of 32-key tiles) take (bit 1 ^ bit 3, bit 2):
// a bijection of bits 1, 2 for the four rows of one parity among 8 (32
// banks) and of bits 2, 3 for the four rows r, r+4, r+8, r+12 that share a
// 256-byte window (64 banks).  Rows of 16 or more chunks (256 B and up) use
// r & 15.  All depend on bits 0..3 of the row only, so rows 32 apart share
// the swizzle.
template <int NCH>
__device__ inline int chunk_swz(int r)
{
    if constexpr (NCH >= 16) return r & 15;
    else if constexpr (NCH == 8) return (r & 7) ^ ((r >> 3) & 1);
    else return (((r >> 1) ^ (r >> 3)) & 1) | ((r >> 1) & 2);
}

// A tile of BN keys of the 8-bit pool (kv8.hpp) on its way into LDS, where it
// lies as an f16 one does: a thread loads CB times sixteen codes of K and of V,
// with their scales, into registers, and later writes their f16 values (exactly
// what is held) as two swizzled chunks each.  The conversion is done once a
// workgroup, not by every wave that reads the tile: 8 to 13 % of a prompt's time
// beside f16 pages, whose tiles go into LDS without passing registers (8192 tokens
// of 32 / 8 heads of 128 653 us and 604, of 14 / 2 of 64 207 and 175; 2048 at 2048 of
// 16 / 2 of 256 158 and 140).
template <int D, int BN, int LT>
struct Stage8 {
    static constexpr int CB = BN * D / (16 * LT), KC = D / 16, VC = BN / 16;  // 16-code chunks a thread, a K row, a V row
    static constexpr int KR = LT / KC, VR = LT / VC;                          // rows between a thread's chunks
    static_assert(LT % VC == 0 && KR % 16 == 0 && VR % 16 == 0, "a thread's chunks differ by a constant");
    u32x4 k[CB], v[CB], vs;
    uint32_t ks[CB];

    static __device__ __amdgpu_buffer_rsrc_t rsrc(const void* base, uint64_t at, uint32_t bytes)
    {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(reinterpret_cast<const char*>(base)) + at, 0, bytes, 0x00020000);
    }
    // (the thread's number passes through an opaque move in each of these: what is derived from it is a few instructions,
    // and kept from step to step it spilled, whose reloads then waited for the loads in flight)
    static __device__ uint32_t fresh(int t)
    {
        uint32_t u = (uint32_t)t;
        asm volatile("" : "+v"(u));
        return u;
    }
    // the tile from key `key` on, in the page at p; t0: the thread's number
    __device__ void load_k(const PagedAttn8Args& a, const Paged8Tile& p, uint32_t key, int t0)
    {
        const uint32_t t = fresh(t0), at = p.bytes ? key & ((1u << a.shift) - 1u) : 0u;
        const __amdgpu_buffer_rsrc_t r = rsrc(a.kc, p.at * D, p.bytes * D), rs = rsrc(a.ks, p.at, p.bytes);
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            k[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, t * 16, at * D + i * (LT * 16), 0));
            ks[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, t / KC, at + i * KR, 0);
        }
    }
    __device__ void load_v(const PagedAttn8Args& a, const Paged8Tile& p, uint32_t key, int t0)
    {
        const uint32_t t = fresh(t0), at = p.bytes ? key & ((1u << a.shift) - 1u) : 0u;
        const __amdgpu_buffer_rsrc_t r = rsrc(a.vc, p.at * D, p.bytes * D), rs = rsrc(a.vs, p.at, p.bytes);
        const uint32_t tile = (at & ~(kV8Tile - 1)) * D + (at & (kV8Tile - 1));  // (a tile may be half of one of 64 positions)
#pragma unroll
        for (int i = 0; i < CB; ++i)
            v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, t / VC * kV8Tile + t % VC * 16,
                                                                                   tile + i * (VR * kV8Tile), 0));
        vs = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, t % VC * 16, at, 0));
    }
    // Where the thread's chunks go, and chunk n of 2 CB (constant after unrolling): so that they can be written between
    // other work.
    struct Place {
        _Float16 *p0, *p1;
    };
    static __device__ Place place_k(_Float16* lds, int t0)
    {
        const uint32_t t = fresh(t0), c = 2 * (t % KC);
        const int r = lds_row_of_key(t / KC), swz = chunk_swz<D / 8>(r);  // (both of the row's low four bits only)
        return Place{lds + r * D + ((c ^ swz) << 3), lds + r * D + (((c + 1) ^ swz) << 3)};
    }
    static __device__ Place place_v(_Float16* lds, int t0)
    {
        const uint32_t t = fresh(t0), c = 2 * (t % VC);
        const int d = t / VC, swz = chunk_swz<BN / 8>(d);
        return Place{lds + d * BN + ((c ^ swz) << 3), lds + d * BN + (((c + 1) ^ swz) << 3)};
    }
    __device__ void put_k(const Place& p, int n) const
    {
        const int i = n >> 1, h = n & 1;
        *reinterpret_cast<f16x8*>((h ? p.p1 : p.p0) + i * (KR * D)) = kv8_values(k[i][2 * h], k[i][2 * h + 1], kv8_scale(ks[i]));
    }
    __device__ void put_v(const Place& p, int n) const
    {
        const int i = n / CB ? n - CB : n, h = n / CB;  // (the halves one after the other: their factors differ)
        const f16x2 f[4] = {kv8_factors(vs[2 * h], 0), kv8_factors(vs[2 * h], 1), kv8_factors(vs[2 * h + 1], 0),
                            kv8_factors(vs[2 * h + 1], 1)};
        *reinterpret_cast<f16x8*>((h ? p.p1 : p.p0) + i * (VR * BN)) = kv8_values(v[i][2 * h], v[i][2 * h + 1], f);
    }
    __device__ void store_k(_Float16* lds, int t0) const
    {
        const Place p = place_k(lds, t0);
#pragma unroll
        for (int n = 0; n < 2 * CB; ++n) put_k(p, n);
    }
    __device__ void store_v(_Float16* lds, int t0) const
    {
        const Place p = place_v(lds, t0);
#pragma unroll
        for (int n = 0; n < 2 * CB; ++n) put_v(p, n);
    }
};

// Values that a query does not see must not reach its output, whatever their
// bits: a masked key's probability is 0, but 0 * inf and 0 * NaN are NaN.
// Paged items look over the V tiles that their mask cuts (in LDS, before the
// product) and clear inf and NaN there; an item in which some were found adds
// them at its end, from the cache, to the rows that do see them.
// clean_v: LDS chunk `ch`, keys 8 c .. of a tile with `valid` stored keys;
// true if it held an inf or NaN and `cut`.
__device__ inline bool clean_v(f16x8* ch, int c, uint32_t valid, bool cut)
{
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    u16x8 v = *reinterpret_cast<u16x8*>(ch);
    const u16x8 b = v & (uint16_t)0x7fff;
    uint16_t top = 0;  // nearly always, the chunk is finite and wanted
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, b[e]);
    if (top < 0x7c00 && (uint32_t)(8 * c + 8) <= valid) return false;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool special = b[e] >= 0x7c00, past = (uint32_t)(8 * c + e) >= valid;
        odd = odd || (special && !past);
        v[e] = (special && cut) || past ? 0 : v[e];
    }
    *reinterpret_cast<u16x8*>(ch) = v;
    return odd && cut;
}
// the first tile of BN keys that an item's mask cuts; ~0 if its piece has none
template <int BN>
__device__ inline uint32_t cut_from(const PagedItem& I)
{
    const int first = I.pos0 + (I.pack ? 0 : (int)(I.qb * BM));  // its first query's position
    const uint32_t t = max(I.t0, (uint32_t)max(first + 1, 0) / BN);
    return I.idle || (int)I.kmax <= first || t >= I.t0 + I.nt ? ~0u : t;
}

// Schedule of one key step's MFMAs: NQ score MFMAs of the next tile and NPV
// P.V MFMAs of this tile (k-slot kc = n / NDB of NKC uses the probabilities
// 8 kc .. 8 kc + 7), with the tile's 8 NKC probabilities spread over them.
// The exp2 of a probability is quarter rate (about as long as half a
// 32x32x16 MFMA with its fma, add and convert), so one to two per MFMA hide
// under the matrix pipe, where 32 under the score MFMAs alone or under the
// PV MFMAs alone would not.  Slot order: the first NQ/2 score MFMAs under
// k-slot 0's probabilities; then for kc = 0..NKC-1 k-slot kc's PV MFMAs
// interleaved with the next score MFMAs under k-slot kc+1's probabilities.
struct FSlot {
    int8_t pv;  // 0: score MFMA n, 1: PV MFMA n
    int8_t n;
    int8_t p0;  // probabilities p0 .. p0+np-1 formed after this MFMA
    int8_t np;
};
template <int NQ, int NPV, int NDB, int NKC>
struct FusedSchedule {
    static_assert(NPV == NKC * NDB && NKC >= 2, "k-slots of 16 keys");
    static constexpr int N = NQ + NPV;
    FSlot s[N];
    constexpr FusedSchedule() : s{}
    {
        const int QA = NQ / 2, QB = (NQ - QA + NKC - 2) / (NKC - 1);
        int k = 0, q = 0, v = 0;
        for (int t = 0; t < QA; ++t)
            s[k++] = FSlot{0, (int8_t)q++, (int8_t)(t * 8 / QA), (int8_t)((t + 1) * 8 / QA - t * 8 / QA)};
        for (int kc = 0; kc < NKC; ++kc) {
            const bool more = kc < NKC - 1;
            const int nq = more ? (QB < NQ - q ? QB : NQ - q) : NQ - q;
            const int tot = NDB + nq;
            for (int t = 0; t < tot; ++t) {
                const bool is_pv = (t + 1) * NDB / tot > t * NDB / tot;
                const int p0 = more ? 8 * (kc + 1) + t * 8 / tot : 0;
                const int np = more ? (t + 1) * 8 / tot - t * 8 / tot : 0;
                s[k++] = FSlot{(int8_t)is_pv, (int8_t)(is_pv ? v++ : q++), (int8_t)p0, (int8_t)np};
            }
        }
    }
};

// first query head of kv head g: heads h with h*n_kv/n_heads == g are
// [head0(g), head0(g+1)) (engine.c:537)
__device__ inline uint32_t head0(const PrefillArgs& a, uint32_t g) { return (g * a.n_heads + a.n_kv - 1) / a.n_kv; }

// (paged launches read their arguments again, paged_items.hpp)
__device__ inline const PrefillArgs& fresh_args(const PrefillArgs& a) { return a; }

// A work item: query block qb (plain rows) or row block qb (packed rows) of
// kv head kvh, key split `split`; h is the query head of plain rows.
struct PItem {
    uint32_t qb, h, kvh, split;
};

// Row r (0..127) of an item -> query index b and head; valid is false for
// rows past the item's end (their loads are clamped to the last row).
struct PRow {
    uint32_t b, h;
    bool valid;
};
template <bool SPLIT>
__device__ inline PRow row_of(const PrefillArgs& a, const PItem& I, uint32_t r)
{
    if (!(SPLIT && a.pack)) {
        const uint32_t q = I.qb * BM + r;
        return PRow{min(q, a.B - 1), I.h, q < a.B};
    }
    const uint32_t h0 = head0(a, I.kvh), nrows = (head0(a, I.kvh + 1) - h0) * a.B;
    const uint32_t rr = I.qb * BM + r, rc = min(rr, nrows - 1);
    return PRow{rc % a.B, h0 + rc / a.B, rr < nrows};
}

// The query indices a wave's 32 rows span (wave-uniform): [first, last].
template <bool SPLIT>
__device__ inline bool wave_span(const PrefillArgs& a, const PItem& I, int wave, uint32_t& first, uint32_t& last)
{
    if (!(SPLIT && a.pack)) {
        const uint32_t q0 = I.qb * BM + wave * 32;
        first = q0;
        last = min(q0 + 31, a.B - 1);
        return q0 < a.B;
    }
    const uint32_t nrows = (head0(a, I.kvh + 1) - head0(a, I.kvh)) * a.B;
    const uint32_t r0 = I.qb * BM + wave * 32, rl = min(r0 + 31, nrows - 1);
    if (r0 / a.B == rl / a.B) {
        first = r0 % a.B;
        last = rl % a.B;
    } else {  // the rows cross into the next head: its first queries, the previous head's last
        first = 0;
        last = a.B - 1;
    }
    return r0 < nrows;
}

// Key tiles of an item: [t0, t0 + nt).  The item's last key is kmax (its
// last query's position; with packed rows (B < 128) every item holds some
// head's query B-1).
template <int BN, bool SPLIT>
__device__ inline void item_keys(const PrefillArgs& a, const PItem& I, uint32_t& kmax, uint32_t& t0, uint32_t& nt)
{
    kmax = a.pos_start + ((SPLIT && a.pack) ? a.B - 1 : min(a.B, I.qb * BM + BM) - 1);
    const uint32_t all = kmax / BN + 1;
    if (SPLIT) {
        t0 = I.split * a.split_tiles;
        const uint32_t t1 = min(all, t0 + a.split_tiles);
        nt = t1 > t0 ? t1 - t0 : 0;
    } else {
        t0 = 0;
        nt = all;
    }
}

// The same of a paged item: b is the row of q and the output, t the token's
// index in its sequence.
struct PagedRow {
    uint32_t b, h, t;
    bool valid;
};
template <class I>
__device__ inline PagedRow paged_row(const PagedAttnArgs& a, const I& it, uint32_t r)
{
    const uint32_t rr = it.qb * BM + r;
    if (!it.pack) {
        const uint32_t t = min(rr, it.nq - 1);
        return PagedRow{it.row0 + t, it.h, t, rr < it.nq};
    }
    const uint32_t h0 = head0(a, it.kvh), nrows = (head0(a, it.kvh + 1) - h0) * it.nq;
    const uint32_t rc = min(rr, nrows - 1), g = div_small(rc, it.nq), t = rc - g * it.nq;
    return PagedRow{it.row0 + t, h0 + g, t, rr < nrows};
}
__device__ inline bool paged_span(const PagedAttnArgs& a, const PagedItem& I, int wave, uint32_t& first, uint32_t& last)
{
    const uint32_t r0 = I.qb * BM + wave * 32;
    const uint32_t nrows = I.pack ? (head0(a, I.kvh + 1) - head0(a, I.kvh)) * I.nq : I.nq;
    const uint32_t rl = min(r0 + 31, nrows - 1);
    if (!I.pack) {
        first = r0;
        last = rl;
    } else {
        const uint32_t g = div_small(r0, I.nq);
        if (g == div_small(rl, I.nq)) {
            first = r0 - g * I.nq;
            last = rl - g * I.nq;
        } else {  // the rows cross into the next head
            first = 0;
            last = I.nq - 1;
        }
    }
    return r0 < nrows && !I.idle;
}

// Item `it` of this workgroup in the plain mode; false past the last.
__device__ inline bool plain_item(const PrefillArgs& a, uint32_t nqb, uint32_t it, PItem& I)
{
    I.split = 0;
    if (a.xcd_map) {
        // Consecutive workgroups go to the 8 XCDs in turn.  XCD x serves
        // kv head x % n_kv, so the query heads that read one kv head
        // share an L2 and its K/V tiles are fetched from HBM once per XCD
        // group, not once per XCD; the XCD's own workgroups take its items.
        const uint32_t x = blockIdx.x % 8u, j = blockIdx.x / 8u, W = gridDim.x / 8u;
        const uint32_t slot = it * W + ((it & 1u) ? W - 1u - j : j);
        if (slot >= nqb * a.n_heads / 8u) return false;
        const uint32_t per = 8u / a.n_kv, G = a.n_heads / a.n_kv;
        const uint32_t g = x % a.n_kv, i = slot * per + x / a.n_kv;
        I.qb = nqb - 1 - i / G;
        I.h = g * G + i % G;
    } else {
        const uint32_t W = gridDim.x;
        const uint32_t slot = it * W + ((it & 1u) ? W - 1u - blockIdx.x : blockIdx.x);
        if (slot >= nqb * a.n_heads) return false;
        I.qb = nqb - 1 - slot / a.n_heads;
        I.h = slot % a.n_heads;
    }
    I.kvh = I.h * a.n_kv / a.n_heads;  // engine.c:537
    return true;
}

// The split mode's item of this workgroup; false where the grid has none.  The
// items of a (kv head, split) tile group read the same K/V tiles, so they should
// share an XCD's L2 (consecutive workgroups go to the 8 XCDs in turn): XCD x
// serves groups x, x+8, ... where no XCD gets more of them than it has CUs for
// (split_grid; 64 tokens at 512 in three splits, 28 / 4 heads of 128: 12.6 us,
// dealt evenly 13.2; 128 tokens at 1536 in seven: 16.7 and 17.4).  Otherwise
// whole groups leave XCDs idle while others queue (2 kv heads without a split:
// six of eight; 1800 tokens of 16 / 2 heads of 256 took 195 us), so each XCD
// takes an eighth of the items in group order; within a group the order deals
// the row blocks out evenly, so that every run of it holds heavy and light ones.
__device__ inline bool split_item(const PrefillArgs& a, PItem& I)
{
    const uint32_t x = blockIdx.x % 8u, j = blockIdx.x / 8u;
    const uint32_t ipg = a.n_rb * (a.pack ? 1u : a.gmax), groups = a.n_kv * a.n_split;
    // both orders share their divisions: a second set cost 0.1 us of a 15 us launch
    const bool whole = a.xcd_map;
    const uint32_t i = whole ? j : x * ((groups * ipg + 7u) / 8u) + j, gi = i / ipg;
    const uint32_t tg = whole ? gi * 8u + x : gi;
    if (tg >= groups) return false;
    uint32_t w = i - gi * ipg;
    const uint32_t den = whole ? a.n_kv : a.n_split, hi = tg / den, lo = tg - hi * den;
    I.kvh = whole ? lo : hi;
    // dealt items: a kv head's splits follow each other, first, last, second, last but one: the later ones are cut
    // by the causal edge (600 tokens at 1000 in three, 14 / 2 heads of 64: 17.5 us, 18.3 in split order)
    I.split = whole ? hi : lo % 2u ? a.n_split - 1u - lo / 2u : lo / 2u;
    if (!whole && !a.pack) {
        // position w of the group's order: the items 0 mod 8 first, then 1 mod 8, ... (packed rows walk the
        // same keys)
        const uint32_t len = ipg / 8u, rem = ipg % 8u;
        const bool lead = w < rem * (len + 1u);  // the first `rem` residues have one item more
        const uint32_t r1 = lead ? w : w - rem * (len + 1u), l1 = lead ? len + 1u : len, q = r1 / l1;
        w = (lead ? 0u : rem) + q + 8u * (r1 - q * l1);
    }
    const uint32_t h0 = head0(a, I.kvh), h1 = head0(a, I.kvh + 1);
    if (a.pack) {
        I.qb = w;
        I.h = h0;
        return w * BM < (h1 - h0) * a.B;
    }
    I.qb = a.n_rb - 1 - w / a.gmax;  // heaviest first
    I.h = h0 + w % a.gmax;
    return I.h < h1;
}

// SPLIT: the split mode (one item per workgroup, packed rows, a key range
// per split); a separate instantiation keeps the plain mode's registers.
// QS: fp32 queries as f16 hi + lo parts, two score MFMAs per k-chunk.  With
// two key groups the lo parts live in LDS (both groups read the same ones; the
// 160 KB are full at d = 128) instead of 32 registers, so that two waves share
// a SIMD.
// A = PagedAttnArgs: the items and key pages of paged attention
// (paged_items.hpp); a workgroup walks its chunk's pieces of items as the
// plain mode walks items.  fp32 queries then also take their probabilities as
// f16 hi + lo parts (PS), so that the output keeps fp32-level error.  16-bit ones
// take f16 alone, half a step (2^-11) for each: the lo parts' products cost 604
// -> 972 us for a prompt of 8192 tokens of 32 / 8 heads of 128 and 83 -> 110 for a
// mixed step, and gain 2.6e-4 -> 2.0e-4 of relative error in f16, 1.67e-3 ->
// 1.66e-3 in bf16, whose outputs' own rounding is 2.0e-4 and 1.65e-3 of it.
template <int D, int NG, bool SPLIT, bool QS = false, class A = PrefillArgs>
__global__ __launch_bounds__(256 * NG * (D > 128 ? 2 : 1), (NG == 1 && D <= 128 && !QS) ? 2 : 1) void prefill_kernel(A args)
{
    constexpr bool PAGED = std::is_base_of<PagedAttnArgs, A>::value, KV8 = std::is_base_of<PagedAttn8Args, A>::value;
    // (sequences with few rows as well, by workgroups of their own)
    constexpr bool MIXED = std::is_same<A, PagedMixed8Args>::value;
    constexpr bool PS = PAGED && QS;
    using Item = typename std::conditional<PAGED, PagedItem, PItem>::type;
    using Pos = typename std::conditional<PAGED, int, uint32_t>::type;  // positions of paged rows may be negative
    static_assert(!(PAGED && SPLIT), "paged items are split by their chunks");
    static_assert(NG == 1 || NG == 2, "one or two key groups");
    static_assert(!SPLIT || NG == 1 || QS, "the split mode of 16-bit queries runs one key group");
    // QL: the queries' lo parts in LDS (fragment order) instead of 32 registers
    constexpr bool QL = QS && NG == 2;
    // Pair mode (head_dim 256): a wave's 32 queries with all 256 dimensions
    // need 64 registers of Q and 128 of O, which leaves one wave per SIMD.
    // Instead two waves share 32 queries and each owns half the dimensions
    // of Q and O; each forms the scores over its half, the halves meet
    // through LDS at the step barrier (the sum is formed in the same order by
    // both waves, so both hold the same scores, maximum and probabilities),
    // and each accumulates its half of O.  The workgroup is 8 waves over the
    // same 128 queries, one per CU, two waves per SIMD.
    constexpr bool PAIR = D > 128;
    static_assert(!PAIR || NG == 1, "pair mode runs one key group");
    constexpr int LT = PAIR ? 512 : 256;  // threads of a key group (they share the tile loads)
    constexpr int DQ = PAIR ? D / 2 : D;  // dimensions of Q and O a wave holds
    constexpr int BN = bn_of(D);  // keys per tile
    constexpr int NS = BN / 32;   // 32-key halves of a tile (score accumulators)
    constexpr int NKC = BN / 16;  // k-slots of the output MFMA per tile
    constexpr int NKK = DQ / 16;  // k-chunks of the score MFMA
    constexpr int NDB = DQ / 32;  // d-blocks of the output MFMA
    constexpr int CH = BN * D / (8 * LT);  // 16-byte chunks per thread per tile (K and V each)
    constexpr int KCH = D / 8;    // 16-byte chunks per K row
    constexpr int VCH = BN / 8;   // 16-byte chunks per V row
    constexpr float LIFT = PAGED ? kLift : 0.0f;
    // NG key groups of 4 waves share the workgroup's 128 queries: group g
    // walks key tiles g, g+NG, g+2NG, ... with its own LDS buffers, and the
    // groups' partial results are merged at the end, so the longest chain
    // of dependent tiles a wave walks is 1/NG of the causal row.
    //
    // Tiles go from HBM straight into LDS (buffer loads with the LDS
    // destination; lane i of a load writes 16 bytes at base + 16 i), K rows
    // [64][D] and V^T rows [D][64], unpadded with swizzled 16-byte chunks.
    // Within a group K is loaded two of its tiles ahead (the score MFMAs of
    // its next tile run during the softmax of the current one) and V one
    // tile ahead, each double buffered.  Buffers of parity 0 and 1 are
    // separate variables, so the compiler can see that a step's loads in
    // flight (into one parity) never alias its LDS reads (of the other) and
    // does not wait for them; each thread waits for its own loads before the
    // barrier that ends the step.
    //
    // Pair mode keeps three buffers of each (K three tiles ahead, V two), so
    // that every tile load has two steps to land: its steps are short (16
    // MFMAs per wave) and all eight waves meet at each step's barrier.
    constexpr int NB = PAIR ? 3 : 2;  // K buffers and V buffers
    __shared__ __attribute__((aligned(16))) _Float16 Kl0[NG][BN * D];
    __shared__ __attribute__((aligned(16))) _Float16 Kl1[NG][BN * D];
    __shared__ __attribute__((aligned(16))) _Float16 Kl2[NB > 2 ? BN * D : 8];
    __shared__ __attribute__((aligned(16))) _Float16 Vl0[NG][D * BN];
    __shared__ __attribute__((aligned(16))) _Float16 Vl1[NG][D * BN];
    __shared__ __attribute__((aligned(16))) _Float16 Vl2[NB > 2 ? D * BN : 8];
    // Pair mode: each wave's partial scores of a tile, by tile parity, as
    // [parity][wave][float4 j][lane] (consecutive lanes, consecutive 16
    // bytes).  Two key groups: (max, sum) of group 1's queries for the merge.
    // (One array: pair mode fills the 160 KB of LDS exactly.)
    __shared__ f32x4 Xl[PAIR ? 2 * 8 * 4 * NS * 64 : NG > 1 && !QL ? 128 : 1];  // (paged: one flag a wave, at least)
    // [query wave][k-chunk][lane]; between items it holds (max, sum) for the merge
    __shared__ f16x8 Qlo[QL ? 4 : 1][QL ? NKK : 1][QL ? 64 : 1];
    float* const s_ml = QL ? reinterpret_cast<float*>(&Qlo[0][0][0]) : reinterpret_cast<float*>(&Xl[0]);

    // Items (query block, head) in heaviest-first order are dealt to the
    // resident workgroups in snake order (item slot it*W + j on even rounds,
    // it*W + W-1-j on odd ones), which balances the causal triangle's
    // linearly decreasing costs; the grid is one item per workgroup when
    // there are no more items than resident slots.
    // item `it` of this workgroup (paged: the next one); false past the last
    PagedCursor C;
    auto item_of = [&](uint32_t it, Item& I) -> bool {
        const A& a = fresh_args(args);
        if constexpr (PAGED) return paged_next<BN>(a, C, I);
        else if constexpr (SPLIT) return it == 0 && split_item(a, I);  // one item per workgroup
        else return plain_item(a, (a.B + BM - 1) / BM, it, I);
    };
    // An item's first loads are issued during the previous item: its
    // group's first K, V and second K tiles in the previous item's last key
    // step, into buffers that step no longer reads (the V tile only after
    // the step when that step reads V buffer 0), and, for 16-bit queries, the
    // query fragments after the key loop (registers the key loop reads
    // cannot be loaded inside it without the compiler waiting for them
    // there).  Their latency hides under that step, the merge and the output
    // stores.  With a gate the epilogue loads the gate values, which would
    // then wait behind these loads; such items issue their loads at their
    // own start.
    const bool early = args.gate == nullptr && !PAIR && !(KV8 && QS);
    // paged, 16-bit queries: an item waits for the next one's first loads before
    // its output stores instead of behind them, so the stores drain during the
    // next item's first step
    constexpr bool AHEAD = PAGED && !QS && NB == 2;
    Item cur;
    if constexpr (PAGED) {
        using Line = typename std::conditional<KV8, Paged8Line, PagedLine>::type;
        if constexpr (MIXED) {
            constexpr size_t share8 = kDecode8Lds<D, false> * sizeof(float);
            static_assert(NG == 1 && !PAIR && !QS && sizeof(Kl0) >= share8 && sizeof(Kl1) >= share8 && sizeof(Vl0) >= share8 &&
                          sizeof(Vl1) >= share8, "an LDS buffer for each of four waves");
            const A& a = fresh_args(args);
            uint64_t* const scratch = reinterpret_cast<uint64_t*>(&Kl0[0][0]);
            const Mixed8Share share = mixed8_share<256>(a, scratch);
            const uint32_t wg = blockIdx.x;
            if (threadIdx.x == 0) {  // chunks without a workgroup
                if (wg >= share.tiles && wg < a.n_wg) reinterpret_cast<PagedDesc*>(a.desc)[wg].n = 0;
                if (wg >= share.few && wg < a.part.n_wg) reinterpret_cast<PagedDesc*>(a.part.desc)[wg].n = 0;
            }
            if (wg < share.few) {
                decode8_pieces<D, false, 0>(args.part, wg, share.few, [&](int w) {
                    return reinterpret_cast<float*>(w == 0 ? &Kl0[0][0] : w == 1 ? &Kl1[0][0] : w == 2 ? &Vl0[0][0] : &Vl1[0][0]);
                });
                return;
            }
            if (wg - share.few >= share.tiles) return;
            const bool any = paged_start<256, Line>(fresh_args(args), scratch, C, wg - share.few, share.tiles);
            if (!any || !paged_next<BN>(fresh_args(args), C, cur)) {
                if (threadIdx.x == 0) reinterpret_cast<PagedDesc*>(fresh_args(args).desc)[C.j].n = 0;
                return;
            }
        } else if (!paged_first<256 * NG * (PAIR ? 2 : 1), BN, Line>(args, reinterpret_cast<uint64_t*>(&Kl0[0][0]), C, cur)) {
            return;
        }
    } else {
        if (!item_of(0, cur)) return;  // uniform over the workgroup
    }
    // (8 bits: tiles on their way from memory to LDS; an item's second K tile from the end of the one before)
    typename std::conditional<KV8, Stage8<D, BN, LT>, int>::type stage;
    for (uint32_t it = 0;; ++it) {
        const A& a = fresh_args(args);
        // Thread indices pass through an opaque move each item so that nothing
        // derived from them is hoisted out of the item loop: the key loop's
        // register budget stays that of a single item.
        int tid;
        asm volatile("v_mov_b32 %0, %1" : "=v"(tid) : "v"((int)threadIdx.x));
        const int lane = tid & 63;
        // with one key group the group is a constant, so the LDS tile bases are
        // too and fold into the reads' offset fields; with two it is read into
        // a scalar register (the LDS destination of a direct-to-LDS load must
        // be uniform, and from a per-lane group index the compiler wrapped
        // every such load in a loop over the lanes' values)
        const int grp = NG > 1 ? (int)__builtin_amdgcn_readfirstlane(tid / LT) : 0,
                  gtid = NG > 1 ? tid % LT : tid, wave = gtid >> 6;
        // the wave's 32 queries (qw) and, in pair mode, its half of the dimensions (hf)
        const int qw = PAIR ? wave >> 1 : wave, hf = PAIR ? wave & 1 : 0;
        const int r32 = lane & 31, hh = lane >> 5;
        // (paged: formed at the group's last step or after the loop)
        Item nxt{};
        bool has_next = false;
        if constexpr (!PAGED) has_next = item_of(it + 1, nxt);

        // Chunk L = LT i + gtid of a tile is the 16 bytes this thread loads
        // with its i-th instruction.  K: LDS row R = L / KCH holds key row
        // lds_row_of_key(R) (an involution), column chunk (L % KCH) ^ swz(R).
        // V: LDS row d = L / VCH holds positions 8c..8c+7 in chunk
        // (L % VCH) ^ swz(d), from 32-position tile c / 4.
        int kgo[CH], vgo[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int L = gtid + LT * i;
            const int R = L / KCH, kc = (L % KCH) ^ chunk_swz<KCH>(R);
            kgo[i] = (lds_row_of_key(R) * D + kc * 8) * 2;
            const int d = L / VCH, vc = (L % VCH) ^ chunk_swz<VCH>(d);
            vgo[i] = (vc >> 2) * (D * (int)kVTile * 2) + d * (int)kVTile * 2 + (vc & 3) * 16;
        }
        const int ksw = chunk_swz<KCH>(r32), vsw = chunk_swz<VCH>(r32);
        // buffers by parity (a constant at every call after inlining)
        auto kbuf = [&](int par) { return par == 0 ? &Kl0[grp][0] : par == 1 ? &Kl1[grp][0] : &Kl2[0]; };
        auto vbuf = [&](int par) { return par == 0 ? &Vl0[grp][0] : par == 1 ? &Vl1[grp][0] : &Vl2[0]; };
        // Buffer resources over a kv head's K rows and V tiles.  A tile adds
        // the scalar offset kt*BN*D*2 bytes (the same for K rows and two
        // 32-position V tiles); every tile lies inside the cache (kv_stride is a
        // multiple of 64 above kmax).
        // (Paged: a resource over the kv head's part of the tile's page, made for
        // each tile from the page number, which is read a step before its use;
        // a page is a multiple of 64 positions, so a tile lies in one.)
        auto rsrc_k = [&](uint32_t kv) {
            if constexpr (PAGED) return kv;
            else
                return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.kc + k_index(kv, 0, 0, D, a.kv_stride)), 0,
                                                         a.kv_stride * D * 2, 0x00020000);
        };
        auto rsrc_v = [&](uint32_t kv) {
            if constexpr (PAGED) return kv;
            else
                return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.vc + v_index(kv, 0, 0, D, a.kv_stride)), 0,
                                                         a.kv_stride * D * 2, 0x00020000);
        };
        // paged: tile kt, in page `page`, of kv head kv into K (V) buffer par
        auto page_of = [&](const Item& I, uint32_t kt) -> uint32_t {
            if constexpr (PAGED) return paged_page(a, I.seq, min(kt, I.t0 + I.nt - 1) * BN);
            else return 0;
        };
        // (8 bits: loaded into registers here, written to LDS by put_k and put_v)
        using Tile = typename std::conditional<KV8, Paged8Tile, PagedTile>::type;
        auto tile_in = [&](uint32_t page, uint32_t kv) {
            if constexpr (KV8) return paged8_tile(a, page, kv);
            else if constexpr (PAGED) return paged_tile<D>(a, page, kv);
            else return Tile{};
        };
        auto put_k = [&](int par) {
            if constexpr (KV8) stage.store_k(kbuf(par), gtid);
        };
        auto put_v = [&](int par) {
            if constexpr (KV8) stage.store_v(vbuf(par), gtid);
        };
        auto dma_page_k = [&](const Tile& p, int par, uint32_t kt) {
            if constexpr (KV8) stage.load_k(a, p, kt * BN, gtid);
            else if constexpr (PAGED) {
                const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                    reinterpret_cast<char*>(const_cast<uint16_t*>(a.kc)) + p.at, 0, p.bytes, 0x00020000);
                const uint32_t at = p.bytes ? ((kt * BN) & ((1u << a.shift) - 1u)) * D * 2 : 0u;
#pragma unroll
                for (int i = 0; i < CH; ++i) lds_load16(r, kbuf(par) + (LT * i + 64 * wave) * 8, kgo[i], at);
            }
        };
        auto dma_page_v = [&](const Tile& p, int par, uint32_t kt) {
            if constexpr (KV8) stage.load_v(a, p, kt * BN, gtid);
            else if constexpr (PAGED) {
                const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                    reinterpret_cast<char*>(const_cast<uint16_t*>(a.vc)) + p.at, 0, p.bytes, 0x00020000);
                const uint32_t at = p.bytes ? ((kt * BN) & ((1u << a.shift) - 1u)) * D * 2 : 0u;
#pragma unroll
                for (int i = 0; i < CH; ++i) lds_load16(r, vbuf(par) + (LT * i + 64 * wave) * 8, vgo[i], at);
            }
        };
        // tile kt of a K (V) resource into K (V) buffer par
        auto dma_k_of = [&](const Item& I, auto r, int par, uint32_t kt) {
            if constexpr (PAGED) dma_page_k(tile_in(page_of(I, kt), r), par, kt);
            else {
#pragma unroll
                for (int i = 0; i < CH; ++i) lds_load16(r, kbuf(par) + (LT * i + 64 * wave) * 8, kgo[i], kt * BN * D * 2);
            }
        };
        auto dma_v_of = [&](const Item& I, auto r, int par, uint32_t kt) {
            if constexpr (PAGED) dma_page_v(tile_in(page_of(I, kt), r), par, kt);
            else {
#pragma unroll
                for (int i = 0; i < CH; ++i) lds_load16(r, vbuf(par) + (LT * i + 64 * wave) * 8, vgo[i], kt * BN * D * 2);
            }
        };
        auto dma_done = [] { __builtin_amdgcn_s_waitcnt(0x0f70); };  // vmcnt(0): this thread's loads landed
        // all but this thread's last n tile loads landed (n of 0, CH or 2 CH:
        // an immediate; memory loads retire in order)
        auto dma_wait_but = [](uint32_t n) {
            if (n >= 2 * CH) __builtin_amdgcn_s_waitcnt(0x0f70 | (2 * CH));
            else if (n >= CH) __builtin_amdgcn_s_waitcnt(0x0f70 | CH);
            else __builtin_amdgcn_s_waitcnt(0x0f70);
        };
        f16x8 qf[NKK];
        f16x8 ql[QS && !QL ? NKK : 1];  // QS: the lo parts
        // the first loads of an item, see above: the K tiles, the first V
        // tile and the queries
        auto keys_of = [&](const Item& I, uint32_t& km, uint32_t& t0, uint32_t& nt) {
            if constexpr (PAGED) {
                km = I.kmax;
                t0 = I.t0;
                nt = I.nt;
            } else {
                item_keys<BN, SPLIT>(a, I, km, t0, nt);
            }
        };
        auto row_from = [&](const A& x, const Item& I, uint32_t r) {
            if constexpr (PAGED) return paged_row(x, I, r);
            else return row_of<SPLIT>(x, I, r);
        };
        auto row_in = [&](const Item& I, uint32_t r) { return row_from(a, I, r); };
        auto item_steps = [&](const Item& I, uint32_t& t0) {
            uint32_t km, nt;
            keys_of(I, km, t0, nt);
            return nt > (uint32_t)grp ? (nt - grp + NG - 1) / NG : 0u;  // this group's tiles
        };
        auto issue_item_k = [&](const Item& I) {
            uint32_t t0;
            const uint32_t igsteps = item_steps(I, t0);
            const auto rk = rsrc_k(I.kvh);
            if (igsteps > 0) dma_k_of(I, rk, 0, t0 + grp);
            if (igsteps > 1) dma_k_of(I, rk, 1, t0 + grp + NG);
        };
        auto issue_item_q = [&](const Item& I) {
            if constexpr (!QS) {  // bf16 as it is, converted when the item starts
                const auto rw = row_in(I, qw * 32 + r32);
                const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + (size_t)rw.b * a.q_stride +
                                     (size_t)rw.h * D + hf * DQ + hh * 8;
#pragma unroll
                for (int kk = 0; kk < NKK; ++kk) qf[kk] = *reinterpret_cast<const f16x8*>(qp + kk * 16);
            }
        };
        auto issue_item_v = [&](const Item& I) {
            uint32_t t0;
            if (item_steps(I, t0) > 0) dma_v_of(I, rsrc_v(I.kvh), 0, t0 + grp);
        };
        // pair mode, after the first loads: K(2) and V(1); returns their count
        auto issue_item_deep = [&](const Item& I) -> uint32_t {
            uint32_t t0;
            const uint32_t n = item_steps(I, t0);
            if (n > 2) dma_k_of(I, rsrc_k(I.kvh), 2, t0 + 2);
            if (n > 1) dma_v_of(I, rsrc_v(I.kvh), 1, t0 + 1);
            return (n > 2 ? CH : 0) + (n > 1 ? CH : 0);
        };
        // 8 bits: an item's first K and V tile into registers, from there into LDS, and its second K tile on its way
        // (written in the prologue): the same registers as in the key loop
        auto load_first = [&](const Item& I) {
            if constexpr (KV8) {
                uint32_t t0;
                if (item_steps(I, t0) == 0) return;
                dma_k_of(I, rsrc_k(I.kvh), 0, t0 + grp);
                dma_v_of(I, rsrc_v(I.kvh), 0, t0 + grp);
            }
        };
        auto put_first = [&](const Item& I) {
            if constexpr (KV8) {
                uint32_t t0;
                const uint32_t n = item_steps(I, t0);
                if (n > 0) {
                    put_k(0);
                    put_v(0);
                }
                if (n > 1) dma_k_of(I, rsrc_k(I.kvh), 1, t0 + grp + NG);
            }
        };
        uint32_t deep_loads = 0;  // loads the prologue need not wait for
        if (KV8 && (it == 0 || !early)) {
            if (it > 0) __syncthreads();
            load_first(cur);
            issue_item_q(cur);
            put_first(cur);
        } else if (it == 0 || !early) {
            if (it > 0) __syncthreads();  // the previous item's epilogue read LDS these loads overwrite
            issue_item_k(cur);
            issue_item_v(cur);
            issue_item_q(cur);
            if constexpr (NB > 2) deep_loads = issue_item_deep(cur);
            if constexpr (AHEAD) dma_done();
        }

        const uint32_t kvh = cur.kvh;
        uint32_t kmax, t0, ntiles;  // this item's keys end at kmax; its tiles are t0 .. t0+ntiles-1
        keys_of(cur, kmax, t0, ntiles);
        const uint32_t nsteps = (ntiles + NG - 1) / NG;  // loop steps (workgroup-uniform)
        // this group's tiles: kt = t0 + grp + NG*st for st < gsteps
        const uint32_t gsteps = ntiles > (uint32_t)grp ? (ntiles - grp + NG - 1) / NG : 0;

        uint32_t wfirst, wlast;
        bool wave_active;
        Pos pos_start;
        const auto myrow = row_in(cur, qw * 32 + r32);
        Pos my_pos;
        if constexpr (PAGED) {
            wave_active = paged_span(a, cur, qw, wfirst, wlast);
            pos_start = cur.pos0;
            wave_active = wave_active && pos_start + (int)wlast >= 0;
            my_pos = pos_start + (int)myrow.t;
        } else {
            wave_active = wave_span<SPLIT>(a, cur, qw, wfirst, wlast);
            pos_start = a.pos_start;
            my_pos = pos_start + myrow.b;
        }
        const Pos wpos_first = pos_start + (Pos)wfirst;
        const Pos wpos_last = pos_start + (Pos)wlast;
        // tiles this wave computes: t0 .. t0+wtiles-1, of which this group's are st < wsteps
        const uint32_t wend = wave_active ? (uint32_t)wpos_last / BN + 1 : 0;  // one past the wave's last tile
        const uint32_t wtiles = wend > t0 ? min(wend - t0, ntiles) : 0;
        const uint32_t wsteps = wtiles > (uint32_t)grp ? (wtiles - grp + NG - 1) / NG : 0;
        auto tile_of = [&](uint32_t st) { return t0 + (uint32_t)grp + NG * st; };

        const auto rK = rsrc_k(kvh), rV = rsrc_v(kvh);
        // paged: where the tiles are whose K and V the coming step loads
        Tile at_k{}, at_v{};
        if constexpr (PAGED) {
            at_k = tile_in(page_of(cur, tile_of(NB)), kvh);
            at_v = tile_in(page_of(cur, tile_of(NB - 1)), kvh);
        }
        auto dma_k = [&](int par, uint32_t st) {
            if constexpr (PAGED) dma_page_k(at_k, par, tile_of(st));
            else dma_k_of(cur, rK, par, tile_of(st));
        };
        auto dma_v = [&](int par, uint32_t st) {
            if constexpr (PAGED) dma_page_v(at_v, par, tile_of(st));
            else dma_v_of(cur, rV, par, tile_of(st));
        };

        // MFMA operands from LDS.  K fragment (j, kk): key row r32 + 32 j, dims
        // DQ hf + 16 kk + 8 hh .. +7 = chunk 2 (kk + NKK hf) + hh.  V fragment
        // (b, kc): row d = DQ hf + 32 b + r32, positions 16 kc + 8 hh .. +7 =
        // chunk 2 kc + hh.
        auto read_k = [&](int par, int j, int kk) {
            return *reinterpret_cast<const f16x8*>(kbuf(par) + (r32 + 32 * j) * D +
                                                   (((2 * (kk + NKK * hf) + hh) ^ ksw) << 3));
        };
        auto read_v = [&](int par, int b, int kc) {
            return *reinterpret_cast<const f16x8*>(vbuf(par) + (DQ * hf + 32 * b + r32) * BN +
                                                   (((2 * kc + hh) ^ vsw) << 3));
        };
        // pair mode: publish this wave's partial scores of a tile (before the
        // step barrier), add the partner's (after it)
        auto xwrite = [&](const f32x16 (&S)[NS], int par) {
            if constexpr (PAIR) {
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4)
                        Xl[((par * 8 + wave) * 4 * NS + 4 * j + q4) * 64 + lane] =
                            f32x4{S[j][4 * q4], S[j][4 * q4 + 1], S[j][4 * q4 + 2], S[j][4 * q4 + 3]};
            }
        };
        auto xadd = [&](f32x16 (&S)[NS], int par) {
            if constexpr (PAIR) {
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) {
                        const f32x4 o4 = Xl[((par * 8 + (wave ^ 1)) * 4 * NS + 4 * j + q4) * 64 + lane];
#pragma unroll
                        for (int e = 0; e < 4; ++e) S[j][4 * q4 + e] += o4[e];
                    }
            }
        };
        // Keys past kmax in the workgroup's last tile were never stored and may
        // hold any bits: their P is 0, but their V must be finite.  The group
        // that owns that tile zeroes them in LDS once, in the step that reads it.
        auto zero_v_tail = [&](int par, uint32_t st) {
            const uint32_t k0 = tile_of(st) * BN;
            const uint32_t valid = kmax - k0 + 1;  // keys 0..valid-1 of the tile are stored
            _Float16* vb = vbuf(par);
            for (int idx = gtid; idx < D * VCH; idx += LT) {
                const int d = idx / VCH, c = idx % VCH;  // logical chunk c: keys 8c..8c+7
                if ((uint32_t)(8 * c + 7) < valid) continue;
                f16x8* ch = reinterpret_cast<f16x8*>(vb + d * BN + ((c ^ chunk_swz<VCH>(d)) << 3));
                f16x8 v = *ch;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((uint32_t)(8 * c + e) >= valid) v[e] = (_Float16)0.0f;
                *ch = v;
            }
        };

        // running max (log2 domain): finite so that a tile whose keys are all in
        // the lane's future (possible as a group's first tile) leaves l and O at
        // zero instead of forming -inf - -inf
        float m = -1e30f, l = 0.0f;
        f32x16 o[NDB];
#pragma unroll
        for (int b = 0; b < NDB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;

        auto read_lo = [&](int kk) {
            if constexpr (QL) return Qlo[qw][kk][lane];
            else return ql[QS ? kk : 0];
        };
        // scores of the tile in K buffer P into S (its 32-key halves)
        auto qk = [&](f32x16 (&S)[NS], int par) {
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) {
                f16x8 lf;
                if constexpr (QS) lf = read_lo(kk);
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    const f16x8 kf = read_k(par, j, kk);
                    S[j] = kk == 0 ? mfma32(kf, qf[0], f32x16{}) : mfma32(kf, qf[kk], S[j]);
                    if constexpr (QS) S[j] = mfma32(kf, lf, S[j]);
                }
            }
        };
        // running max update of the lane's query from tile scores S (raw, masked)
        auto update_max = [&](const f32x16 (&S)[NS]) {
            float mx = S[0][0];
#pragma unroll
            for (int j = 0; j < NS; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, S[j][i]);
            // the lane pair (l, l+32) holds one query: exchange the halves
            const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, mx),
                                                             __builtin_bit_cast(uint32_t, mx), false, false);
            mx = fmaxf(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1])) * a.c;
            if (__ballot(mx > m + (LIFT + kSlack))) {  // wave-uniform: some query's max moved
                const float mn = mx > m + (LIFT + kSlack) ? mx - LIFT : m;
                const float alpha = fast_exp2(m - mn);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int b = 0; b < NDB; ++b) o[b] *= alpha;
            }
        };
        auto probs = [&](const f32x16 (&S)[NS], f16x8 (&pf)[NKC], f16x8 (&pl)[PS ? NKC : 1]) {
            const float nm = -m;
#pragma unroll
            for (int i = 0; i < 16 * NS; ++i) {
                const float p = fast_exp2(fmaf(S[i >> 4][i & 15], a.c, nm));
                l += p;
                pf[i >> 3][i & 7] = (_Float16)p;
                if constexpr (PS) pl[i >> 3][i & 7] = (_Float16)(p - (float)pf[i >> 3][i & 7]);
            }
        };
        // O^T += V^T P^T over the tile in V buffer P; fragments are read two
        // MFMAs ahead (three in a ring)
        auto pv = [&](const f16x8 (&pf)[NKC], const f16x8 (&pl)[PS ? NKC : 1], int par) {
            constexpr int NM = NKC * NDB;  // MFMA n: kc = n / NDB, b = n % NDB
            f16x8 vf[3];
            vf[0] = read_v(par, 0, 0);
            vf[1] = read_v(par, 1 % NDB, 1 / NDB);
#pragma unroll
            for (int n = 0; n < NM; ++n) {
                if (n + 2 < NM) vf[(n + 2) % 3] = read_v(par, (n + 2) % NDB, (n + 2) / NDB);
                o[n % NDB] = mfma32(vf[n % 3], pf[n / NDB], o[n % NDB]);
                if constexpr (PS) o[n % NDB] = mfma32(bounded(vf[n % 3]), pl[n / NDB], o[n % NDB]);
            }
        };
        // Scores of the next tile (K buffer kpar) into Snext and P.V of this tile
        // (V buffer vpar), with this tile's probabilities (from Scur) formed
        // between them per FusedSchedule; K and V fragments are read two MFMAs
        // ahead in their own streams.
        auto qk_pv = [&](f32x16 (&Snext)[NS], int kpar, const f32x16 (&Scur)[NS], int vpar) {
            constexpr int NQ = NS * NKK, NPV = NKC * NDB;  // score MFMA n: half n % NS, k-chunk n / NS
            constexpr FusedSchedule<NQ, NPV, NDB, NKC> sch{};
            constexpr int MAXP = 8;
            const float nm = -m;
            constexpr int KR = QL ? 2 : 3;  // K ring: read two MFMAs ahead (a score slot of split queries has two)
            f16x8 pf[NKC], pl[PS ? NKC : 1], kf[KR], vf[3], lf[2];
            kf[0] = read_k(kpar, 0, 0);
            if constexpr (!QL) kf[1] = read_k(kpar, 1 % NS, 1 / NS);
            if constexpr (QL) lf[0] = read_lo(0);
            vf[0] = read_v(vpar, 0, 0);
            vf[1] = read_v(vpar, 1 % NDB, 1 / NDB);
#pragma unroll
            for (int t = 0; t < sch.N; ++t) {
                const int n = sch.s[t].n;
                if (sch.s[t].pv) {
                    if (n + 2 < NPV) vf[(n + 2) % 3] = read_v(vpar, (n + 2) % NDB, (n + 2) / NDB);
                    o[n % NDB] = mfma32(vf[n % 3], pf[n / NDB], o[n % NDB]);
                    if constexpr (PS) o[n % NDB] = mfma32(bounded(vf[n % 3]), pl[n / NDB], o[n % NDB]);
                } else {
                    if (n + KR - 1 < NQ) kf[(n + KR - 1) % KR] = read_k(kpar, (n + KR - 1) % NS, (n + KR - 1) / NS);
                    if constexpr (QL)
                        if (n % NS == 0 && n / NS + 1 < NKK) lf[(n / NS + 1) & 1] = read_lo(n / NS + 1);
                    Snext[n % NS] = n < NS ? mfma32(kf[n % KR], qf[0], f32x16{})
                                           : mfma32(kf[n % KR], qf[n / NS], Snext[n % NS]);
                    if constexpr (QL) Snext[n % NS] = mfma32(kf[n % KR], lf[(n / NS) & 1], Snext[n % NS]);
                    else if constexpr (QS) Snext[n % NS] = mfma32(kf[n % KR], ql[n / NS], Snext[n % NS]);
                }
#pragma unroll
                for (int u = 0; u < MAXP; ++u) {
                    if (u < sch.s[t].np) {
                        const int i = sch.s[t].p0 + u;
                        const float p = fast_exp2(fmaf(Scur[i >> 4][i & 15], a.c, nm));
                        l += p;
                        pf[i >> 3][i & 7] = (_Float16)p;
                        if constexpr (PS) pl[i >> 3][i & 7] = (_Float16)(p - (float)pf[i >> 3][i & 7]);
                    }
                }
            }
        };
        // a tile that reaches past the wave's first query: keys beyond the
        // lane's position get -inf
        auto mask = [&](f32x16 (&S)[NS], uint32_t st) {
            const uint32_t k0 = tile_of(st) * BN;
            if ((Pos)(k0 + BN - 1) > wpos_first) {
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if ((Pos)(k0 + 32 * j + key_of_acc(i, hh)) > my_pos) S[j][i] = -INFINITY;
            }
        };

        // prologue: this item's first loads are in flight (issued above or at the
        // end of the previous item); bf16 queries are converted here, f32 ones
        // loaded and split (prefetched like the others they spilled: 2048 tokens 63
        // -> 79 us).  All loads are complete before the key loop, whose waits then
        // count only tile loads (in pair mode K(2) and V(1) may still be in
        // flight; the first step waits for them).
        if constexpr (!AHEAD && !KV8) dma_wait_but(deep_loads);
        if (QL && it > 0) lds_barrier();  // the merge has read (max, sum)
        if constexpr (QS) {
            const float* qp = reinterpret_cast<const float*>(a.q) + (size_t)myrow.b * a.q_stride + (size_t)myrow.h * D +
                              hf * DQ + hh * 8;
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) {
                f16x8 lo;
                split_q8(qf[kk], lo, *reinterpret_cast<const f32x4*>(qp + kk * 16),
                         *reinterpret_cast<const f32x4*>(qp + kk * 16 + 4));
                if constexpr (!QL) ql[kk] = lo;
                else if (grp == 0) Qlo[qw][kk][lane] = lo;  // both groups hold the same queries
            }
            if (NB == 2) dma_done();
        } else if (a.q_dtype == kBF16) {
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) bf16_to_f16(qf[kk]);
        }
        if constexpr (NB > 2 || AHEAD) lds_barrier();
        else __syncthreads();
        f32x16 Sa[NS], Sb[NS];
        if (wsteps > 0) {
            qk(Sa, 0);
            xwrite(Sa, 0);
        }
        if constexpr (KV8) {
            if (gsteps > 1) put_k(1);
            if constexpr (NB > 2) {  // K(2) and V(1)
                if (gsteps > 2) {
                    dma_k_of(cur, rK, 2, tile_of(2));
                    put_k(2);
                }
                if (gsteps > 1) {
                    dma_v_of(cur, rV, 1, tile_of(1));
                    put_v(1);
                }
            }
        }
        // step 0 loads K(NB) over K(0), whose last readers are the scores above
        if constexpr (NB > 2 || AHEAD) lds_barrier();
        else __syncthreads();

        // step st (buffer phase ph = st % NB, score parity sp = st % 2): loads
        // K(st+NB) into K buffer ph (it held K(st), last read by the previous
        // step's scores) and V(st+NB-1) into V buffer (ph+NB-1) % NB (it held
        // V(st-1)); scores of st+1 (K buffer (ph+1) % NB) overlap the softmax
        // of st; P.V of st (V buffer ph); one barrier.  With pos_start not a
        // multiple of 32 a wave's queries straddle a tile boundary, so a tile
        // with a successor may still need the mask.
        // the step that reads the tile holding kmax (the item's last tile, unless
        // a later split owns it), in this group's buffers
        // paged: the first tile cut by the item's mask (~0: none), and whether this
        // thread found an inf or NaN in such tiles
        uint32_t cut_tile = ~0u;
        bool odd_v = false;
        if constexpr (PAGED) cut_tile = cut_from<BN>(cur);
        auto clean_tile = [&](int par, uint32_t st) {
            const uint32_t kt = tile_of(st), valid = kmax - kt * BN + 1;
            if (st >= gsteps || !(kt >= cut_tile || valid < BN)) return;  // uniform over the group
            for (int idx = gtid; idx < D * VCH; idx += LT) {
                const int d = idx / VCH, c = idx % VCH;
                odd_v |= clean_v(reinterpret_cast<f16x8*>(vbuf(par) + d * BN + ((c ^ chunk_swz<VCH>(d)) << 3)), c, valid,
                                 kt >= cut_tile);
            }
        };
        const bool has_tail = ntiles > 0 && t0 + ntiles == kmax / BN + 1 && (kmax + 1) % BN != 0;
        const uint32_t tail_step = (ntiles - 1) / NG;
        const int tail_grp = (int)((ntiles - 1) % NG);
        bool prefetch = has_next && early;
        // the group's last step (or, for a group without tiles, the first) issues
        // the next item's loads
        const uint32_t last_st = gsteps > 0 ? gsteps - 1 : 0;
        auto step = [&](int ph, int sp, uint32_t st, f32x16 (&Scur)[NS], f32x16 (&Snext)[NS]) {
            const bool lk = st + NB < gsteps, lv = st + NB - 1 < gsteps;
            if (lk) dma_k(ph, st + NB);
            if (lv) dma_v((ph + NB - 1) % NB, st + NB - 1);
            uint32_t page = 0;  // of the tile after those: read here, used at the step's end
            if constexpr (PAGED) page = page_of(cur, tile_of(st + NB + 1));
            if (PAGED && early && st == last_st) prefetch = has_next = item_of(it + 1, nxt);
            if (prefetch && st == last_st) {
                // K buffers are free (no scores follow), V buffer 1-p too
                if constexpr (KV8) {
                    load_first(nxt);  // (written after the key loop)
                } else {
                    issue_item_k(nxt);
                    if (ph == 1 || gsteps == 0) issue_item_v(nxt);
                }
            }
            if constexpr (PAGED) {
                // workgroup-uniform: some group's tile is cut, or the last one
                if ((has_tail && st == tail_step) || t0 + NG * st + NG - 1 >= cut_tile) {
                    clean_tile(ph, st);
                    lds_barrier();
                }
            } else if (has_tail && st == tail_step) {  // workgroup-uniform
                if (grp == tail_grp) zero_v_tail(ph, st);
                lds_barrier();
            }
            if (st + 1 < wsteps) {
                xadd(Scur, sp);
                mask(Scur, st);
                update_max(Scur);
                qk_pv(Snext, (ph + 1) % NB, Scur, ph);
                xwrite(Snext, 1 - sp);
            } else if (st < wsteps) {
                xadd(Scur, sp);
                mask(Scur, st);
                update_max(Scur);
                f16x8 pf[NKC], pl[PS ? NKC : 1];
                probs(Scur, pf, pl);
                pv(pf, pl, ph);
            }
            if constexpr (PAGED) {
                at_v = at_k;
                at_k = tile_in(page, kvh);
            }
            if constexpr (KV8) {
                if (lk) put_k(ph);
                if (lv) put_v((ph + NB - 1) % NB);
            } else if constexpr (NB > 2) {
                // the previous steps' loads (this step's have two steps to land)
                dma_wait_but((lk ? CH : 0) + (lv ? CH : 0));
            } else {
                // this step's own loads (none from the group's last step on, whose
                // next-item loads are waited for by the next item)
                if (!(prefetch && st >= last_st)) dma_done();
            }
            lds_barrier();
        };
        if constexpr (NB == 2) {
            for (uint32_t st = 0; st < nsteps; st += 2) {
                step(0, 0, st, Sa, Sb);
                if (st + 1 < nsteps) step(1, 1, st + 1, Sb, Sa);
            }
        } else {
            // buffer phase period 3, score parity period 2
            for (uint32_t st = 0; st < nsteps; st += 6) {
                step(0, 0, st, Sa, Sb);
                if (st + 1 >= nsteps) break;
                step(1, 1, st + 1, Sb, Sa);
                if (st + 2 >= nsteps) break;
                step(2, 0, st + 2, Sa, Sb);
                if (st + 3 >= nsteps) break;
                step(0, 1, st + 3, Sb, Sa);
                if (st + 4 >= nsteps) break;
                step(1, 0, st + 4, Sa, Sb);
                if (st + 5 >= nsteps) break;
                step(2, 1, st + 5, Sb, Sa);
            }
        }

        if (PAGED && !early) has_next = item_of(it + 1, nxt);
        // the next item's first V tile when the last step still read V buffer 0,
        // and its queries
        if (prefetch) {
            if constexpr (KV8) put_first(nxt);  // (the step's barrier is behind every read of these buffers)
            else if (gsteps > 0 && (last_st & 1u) == 0) issue_item_v(nxt);
            issue_item_q(nxt);
        }
        {
            // the lane pair (l, l+32) holds one query: add the halves
            const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, l),
                                                             __builtin_bit_cast(uint32_t, l), false, false);
            l = __builtin_bit_cast(float, (uint32_t)sw[0]) + __builtin_bit_cast(float, (uint32_t)sw[1]);
        }
        // Thread indices for the epilogue from a fresh opaque read, so that the
        // ones of the item's start need not stay live through the key loop.
        const A& a_e = fresh_args(args);
        int tid_e;
        asm volatile("v_mov_b32 %0, %1" : "=v"(tid_e) : "v"((int)threadIdx.x));
        const int gtid_e = NG > 1 ? tid_e % LT : tid_e, lane_e = tid_e & 63;
        const int qw_e = PAIR ? gtid_e >> 7 : gtid_e >> 6, hf_e = PAIR ? (gtid_e >> 6) & 1 : 0;
        int b_lo = 0, b_hi = NDB;  // the O blocks this thread stores
        bool add_odd = false;      // paged: add the infs and NaNs cleared above
        if constexpr (PAGED) {
            if (cut_tile != ~0u) {  // workgroup-uniform; Xl (with QL the part of Qlo behind (max, sum)) is free between key loops
                uint32_t* flags = reinterpret_cast<uint32_t*>(QL ? s_ml + 512 : s_ml + (NG > 1 ? 512 : 0));
                const bool mine = __ballot(odd_v) != 0;
                if (lane_e == 0) flags[tid_e >> 6] = mine;
                lds_barrier();
                for (int w = 0; w < LT * NG / 64; ++w) add_odd = add_odd || flags[w] != 0;
                if (NG == 1) lds_barrier();  // read before the next item's step writes there
            }
        }
        int pos_e = 0;
        if constexpr (NG > 1) {
            // The two groups' (m, l, O) meet through LDS: m, l in s_ml and O
            // through V buffer 1 of both groups (the one buffer the next item's
            // first loads leave free; 32 KB at d = 128), half the blocks at a
            // time.  Group 1 hands over blocks 0 .. HB-1, which group 0 merges
            // and stores; then group 0 hands over blocks HB .., which group 1
            // merges and stores, so both groups issue half of the output.
            constexpr int HB = NDB / 2;  // O blocks per round
            static_assert(HB * 16 * 256 * 4 <= (int)sizeof(Vl1), "merge area");
            float* oarea = reinterpret_cast<float*>(&Vl1[0][0]);
            if (grp == 1) {
                s_ml[gtid_e] = m;
                s_ml[256 + gtid_e] = l;
#pragma unroll
                for (int b = 0; b < HB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) oarea[(b * 16 + i) * 256 + gtid_e] = o[b][i];
            }
            lds_barrier();
            float mo = m, lo = l;  // the other group's (m, l)
            auto merge_half = [&](int r) {
                const float mg = fmaxf(m, mo);
                const float cs = fast_exp2(m - mg), co = fast_exp2(mo - mg);
#pragma unroll
                for (int b = 0; b < HB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[r * HB + b][i] = o[r * HB + b][i] * cs + oarea[(b * 16 + i) * 256 + gtid_e] * co;
            };
            if (grp == 0) {
                mo = s_ml[gtid_e];
                lo = s_ml[256 + gtid_e];
                merge_half(0);
            }
            lds_barrier();  // round 0 read before round 1 overwrites
            if (grp == 0) {
                s_ml[gtid_e] = m;
                s_ml[256 + gtid_e] = l;
#pragma unroll
                for (int b = 0; b < HB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) oarea[(b * 16 + i) * 256 + gtid_e] = o[HB + b][i];
            }
            lds_barrier();
            if (grp == 1) {
                mo = s_ml[gtid_e];
                lo = s_ml[256 + gtid_e];
                merge_half(1);
            }
            const float mg = fmaxf(m, mo);
            l = l * fast_exp2(m - mg) + lo * fast_exp2(mo - mg);
            m = mg;
            b_lo = grp * HB;
            b_hi = b_lo + HB;
        }
        const auto rw = row_from(a_e, cur, qw_e * 32 + (lane_e & 31));
        if constexpr (PAGED) pos_e = cur.pos0 + (int)rw.t;
        // four of the row's output values (unnormalised ones in a piece)
        auto with_odd = [&](f32x4 v, uint32_t d) {
            if constexpr (PAGED) {
                if constexpr (KV8) {
                    if (add_odd) {
                        const uint32_t nan = nan_dims<D>(a_e, cur.seq, cur.kvh, d, pos_e, cut_tile * BN,
                                                         (int)min(cur.kmax + 1, (cur.t0 + cur.nt) * BN));
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = nan >> e & 1u ? NAN : v[e];
                    }
                } else if (add_odd)
#pragma unroll 1
                    for (int e = 0; e < 4; ++e) {
                        const float x = special_sum<D>(a_e, cur.seq, cur.kvh, d + e, pos_e, cut_tile * BN,
                                                         (int)min(cur.kmax + 1, (cur.t0 + cur.nt) * BN));
                        v[0] += e == 0 ? x : 0.0f;
                        v[1] += e == 1 ? x : 0.0f;
                        v[2] += e == 2 ? x : 0.0f;
                        v[3] += e == 3 ? x : 0.0f;
                    }
            }
            return v;
        };
        bool partial;
        if constexpr (PAGED) partial = cur.part != 0;
        else partial = SPLIT && a_e.n_split > 1;
        if constexpr (AHEAD) dma_done();
        if (rw.valid) {
            if (partial) {
                // split partials: (max, sum) and the unnormalised O of this
                // row over this split's keys
                size_t pr;
                if constexpr (PAGED) pr = (size_t)(2 * C.j + (cur.part & 1)) * BM + qw_e * 32 + (lane_e & 31);
                else pr = ((size_t)cur.split * a_e.n_heads + rw.h) * a_e.B + rw.b;
                // (one key group's sum: the groups round l differently, and two
                // stores to one slot in no order would leave either)
                if ((lane_e >> 5) == 0 && hf_e == 0 && grp == 0) {
                    typedef float f32x2 __attribute__((ext_vector_type(2)));
                    *reinterpret_cast<f32x2*>(a_e.part_ml + 2 * pr) = f32x2{m, l};
                }
#pragma unroll
                for (int b = 0; b < NDB; ++b) {
                    if (b < b_lo || b >= b_hi) continue;
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        const uint32_t d = hf_e * DQ + b * 32 + 8 * i4 + 4 * (lane_e >> 5);
                        f32x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = o[b][4 * i4 + e];
                        *reinterpret_cast<f32x4*>(a_e.part_o + pr * D + d) = with_odd(v, d);
                    }
                }
            } else {
                // (paged: a row that sees no key is zero)
                const float inv = PAGED && l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int b = 0; b < NDB; ++b) {
                    if (b < b_lo || b >= b_hi) continue;
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        const uint32_t d = hf_e * DQ + b * 32 + 8 * i4 + 4 * (lane_e >> 5);
                        f32x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = o[b][4 * i4 + e] * inv;
                        v = with_odd(v, d);
                        if (a_e.gate) {
                            const float* gp = a_e.gate + (size_t)rw.b * a_e.gate_stride + (size_t)rw.h * D + d;
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] *= sigmoid_ref(gp[e]);
                        }
                        store_out4(a_e.out, (size_t)rw.b * a_e.out_stride + (size_t)rw.h * D + d, a_e.out_dtype, v);
                    }
                }
            }
        }
        if (!has_next) break;
        cur = nxt;
    }  // items
    if constexpr (PAGED) paged_leave(args, C, cur);
}

// head_dim 256, 16-bit queries.  Bound by the LDS: 128 bytes per
// cycle and CU against 4 KB of operands per 32-cycle MFMA slot of the four
// SIMDs.  A workgroup is 8 waves over 128 queries, one per CU, and two waves
// share 32 queries (a wave with all 256 dimensions of O and Q would be alone on
// its SIMD).  The pair splits the scores by keys and the output by dimensions:
// of a 64-key tile each wave forms the scores of 32 keys over all 256
// dimensions (Q in 64 registers), turns them into probabilities, hands the
// 2 KB of f16 probabilities to its partner through LDS and accumulates its
// half of the dimensions of O over all 64 keys.  Split by dimensions on both
// sides (prefill_kernel's pair mode, which keeps f32 queries), the waves
// exchange fp32 partial scores and both form every probability: 1.75 KB of LDS
// traffic per MFMA against 1.38, and twice the exp2.
// 4096 tokens, 16 / 2 heads, bf16, gated: 215 -> 170 us (808 TFLOP/s), ungated
// 188 -> 153.  (The gate is the fp32 sigmoid of the other kernels; by the
// approximate reciprocal of 1 + exp2 it took 6 us less and was up to 3.5e-6
// off at gates of -60, 2.3e-7 now.)  The probabilities are f16, as there; their
// lo parts would need 16 KB of LDS more (146 of 160 KB are taken).
//
// Step t starts with the raw scores of tile t in registers and their maxima
// in LDS.  The next tile's score MFMAs begin; the pair's common maximum is
// formed (lazily, as in prefill_kernel); the 16 probabilities of a lane go
// between the rest of the score MFMAs and then to LDS; the output MFMAs of the
// wave's own 32 keys follow; a barrier; those of the partner's keys, under
// which the next tile's maximum is formed; a barrier.  K is loaded two tiles
// ahead, V one, straight into LDS, and an item's first K and V tiles during the
// previous item's last step.
// A = PagedAttnArgs: paged items, as in prefill_kernel.
template <int D, bool SPLIT, class A = PrefillArgs>
__global__ __launch_bounds__(512) void prefill_halves_kernel(A args)
{
    static_assert(D == 256, "two waves of 128 output dimensions");
    constexpr bool PAGED = std::is_base_of<PagedAttnArgs, A>::value, KV8 = std::is_same<A, PagedAttn8Args>::value;
    using Item = typename std::conditional<PAGED, PagedItem, PItem>::type;
    static_assert(!(PAGED && SPLIT), "paged items are split by their chunks");
    constexpr int BN = 64, DH = D / 2;
    constexpr int NKK = D / 16, NDB = DH / 32;
    constexpr int KCH = D / 8, VCH = BN / 8;
    constexpr int CH = BN * D / (8 * 512);  // 16-byte chunks per thread per tile (K and V each)
    constexpr float LIFT = PAGED ? kLift : 0.0f;
    __shared__ __attribute__((aligned(16))) _Float16 Kl0[BN * D], Kl1[BN * D], Vl0[D * BN], Vl1[D * BN];
    __shared__ f16x8 Pl[8][2][64];  // each wave's probabilities: k-slot, lane
    __shared__ float Ml[8][64];     // each wave's tile maxima, then its row sums
    __shared__ uint32_t odd_flags[PAGED ? 8 : 1];

    PagedCursor C;
    auto item_of = [&](uint32_t it, Item& I) -> bool {
        const A& a = fresh_args(args);
        if constexpr (PAGED) return paged_next<BN>(a, C, I);
        else if constexpr (SPLIT) return it == 0 && split_item(a, I);
        else return plain_item(a, (a.B + BM - 1) / BM, it, I);
    };
    Item cur;
    if constexpr (PAGED) {
        using Line = typename std::conditional<KV8, Paged8Line, PagedLine>::type;
        if (!paged_first<512, BN, Line>(args, reinterpret_cast<uint64_t*>(&Kl0[0]), C, cur)) return;
    } else {
        if (!item_of(0, cur)) return;  // uniform over the workgroup
    }
    typename std::conditional<KV8, Stage8<D, BN, 512>, int>::type stage;  // (see prefill_kernel)
    for (uint32_t it = 0;; ++it) {
        const A& a = fresh_args(args);
        int tid;  // opaque per item, as in prefill_kernel
        asm volatile("v_mov_b32 %0, %1" : "=v"(tid) : "v"((int)threadIdx.x));
        const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int qw = wave >> 1, hf = wave & 1;
        const int r32 = lane & 31, hh = lane >> 5;
        Item nxt{};  // (paged: formed in the last step)
        bool has_next = false;
        if constexpr (!PAGED) has_next = !SPLIT && item_of(it + 1, nxt);

        auto kbuf = [&](int par) { return par == 0 ? &Kl0[0] : &Kl1[0]; };
        auto vbuf = [&](int par) { return par == 0 ? &Vl0[0] : &Vl1[0]; };
        // chunk 512 i + tid of a tile: K LDS row R = 16 i + tid / KCH, V LDS row d = 64 i + tid / VCH; the swizzles
        // and the row permutation are the same for every i
        const int kgo = (lds_row_of_key(tid / KCH) * D + ((tid % KCH) ^ chunk_swz<KCH>(tid / KCH)) * 8) * 2;
        const int vch = (tid % VCH) ^ chunk_swz<VCH>(tid / VCH);
        const int vgo = (vch >> 2) * (D * (int)kVTile * 2) + tid / VCH * ((int)kVTile * 2) + (vch & 3) * 16;
        // tile kt of kv head kv, counted from position p0 (a multiple of 64: 64 rows of K and two V tiles of 32
        // positions are the same number of elements)
        // (paged: in its page, see prefill_kernel)
        auto page_of = [&](const Item& I, uint32_t p0, uint32_t kt) -> uint32_t {
            if constexpr (PAGED) return paged_page(a, I.seq, p0 + min(kt, I.nt - 1) * BN);
            else return 0;
        };
        using Tile = typename std::conditional<KV8, Paged8Tile, PagedTile>::type;
        auto rsrc_at = [&](const uint16_t* pool, uint32_t kv, uint32_t p0, const PagedTile& p) {
            if constexpr (PAGED) {
                return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(const_cast<uint16_t*>(pool)) + p.at, 0,
                                                         p.bytes, 0x00020000);
            } else {  // (V tiles of 32 positions take the bytes of 32 K rows)
                return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(pool + k_index(kv, p0, 0, D, a.kv_stride)),
                                                         0, (a.kv_stride - p0) * D * 2, 0x00020000);
            }
        };
        auto tile_at = [&](uint32_t p0, uint32_t kt, const PagedTile& p) -> uint32_t {
            if constexpr (PAGED) return p.bytes ? ((p0 + kt * BN) & ((1u << a.shift) - 1u)) * D * 2 : 0u;
            else return kt * BN * D * 2;
        };
        auto place = [&](const Item& I, uint32_t p0, uint32_t kt) {  // of tile kt
            if constexpr (KV8) return paged8_tile(a, page_of(I, p0, kt), I.kvh);
            else if constexpr (PAGED) return paged_tile<D>(a, page_of(I, p0, kt), I.kvh);
            else return PagedTile{};
        };
        auto dma_k = [&](uint32_t kv, uint32_t p0, int par, uint32_t kt, const Tile& p) {
            if constexpr (KV8) stage.load_k(a, p, p0 + kt * BN, tid);
            else {
                const __amdgpu_buffer_rsrc_t r = rsrc_at(a.kc, kv, p0, p);
                const uint32_t at = tile_at(p0, kt, p);
#pragma unroll
                for (int i = 0; i < CH; ++i)
                    lds_load16(r, kbuf(par) + (512 * i + 64 * wave) * 8, kgo, at + i * (16 * D * 2));
            }
        };
        auto dma_v = [&](uint32_t kv, uint32_t p0, int par, uint32_t kt, const Tile& p) {
            if constexpr (KV8) stage.load_v(a, p, p0 + kt * BN, tid);
            else {
                const __amdgpu_buffer_rsrc_t r = rsrc_at(a.vc, kv, p0, p);
                const uint32_t at = tile_at(p0, kt, p);
#pragma unroll
                for (int i = 0; i < CH; ++i)
                    lds_load16(r, vbuf(par) + (512 * i + 64 * wave) * 8, vgo, at + i * (64 * (int)kVTile * 2));
            }
        };
        auto dma_done = [] { __builtin_amdgcn_s_waitcnt(0x0f70); };  // vmcnt(0)
        // an item's tiles: how many, from position p0 on, and its last key (split_tiles counts 32 keys, an even
        // number of them)
        auto tiles_of = [&](const Item& I, uint32_t& kmax, uint32_t& p0) -> uint32_t {
            if constexpr (PAGED) {
                kmax = I.kmax;
                p0 = I.t0 * BN;
                return I.nt;
            } else {
                kmax = a.pos_start + ((SPLIT && a.pack) ? a.B - 1 : min(a.B, I.qb * BM + BM) - 1);
                const uint32_t all = kmax / BN + 1, per = (a.split_tiles + 1) / 2;
                p0 = 0;
                if (!SPLIT) return all;
                p0 = I.split * per * BN;
                // a row block without keys in this split walks one tile, keys of later rows, with every wave idle
                return max(min(all - min(all, I.split * per), per), 1u);
            }
        };
        auto row_from = [&](const A& x, const Item& I, uint32_t r) {
            if constexpr (PAGED) return paged_row(x, I, r);
            else return row_of<SPLIT>(x, I, r);
        };
        auto row_in = [&](const Item& I, uint32_t r) { return row_from(a, I, r); };
        // the item's first K tiles; those of V follow into buffer 0
        auto issue_k = [&](const Item& I) {
            uint32_t km, p0;
            const uint32_t n = tiles_of(I, km, p0);
            dma_k(I.kvh, p0, 0, 0, place(I, p0, 0));
            if (n > 1) dma_k(I.kvh, p0, 1, 1, place(I, p0, 1));
        };
        auto issue_v = [&](const Item& I) {
            uint32_t km, p0;
            tiles_of(I, km, p0);
            dma_v(I.kvh, p0, 0, 0, place(I, p0, 0));
        };
        // (8 bits: as in prefill_kernel)
        auto load_first = [&](const Item& I) {
            if constexpr (KV8) {
                uint32_t km, p0;
                tiles_of(I, km, p0);
                const Tile p = place(I, p0, 0);
                stage.load_k(a, p, p0, tid);
                stage.load_v(a, p, p0, tid);
            }
        };
        auto put_first = [&](const Item& I) {
            if constexpr (KV8) {
                uint32_t km, p0;
                tiles_of(I, km, p0);
                stage.store_k(kbuf(0), tid);
                stage.store_v(vbuf(0), tid);
            }
        };
        const uint32_t kvh = cur.kvh;
        uint32_t kmax, p0;
        const uint32_t ntiles = tiles_of(cur, kmax, p0);
        if constexpr (KV8) {
            if (it == 0) {
                load_first(cur);
                put_first(cur);
            }
            stage.load_k(a, place(cur, p0, 1), p0 + BN, tid);  // (of a single tile's page again: not read)
        } else if (it == 0) {
            issue_k(cur);
            issue_v(cur);
        }
        f16x8 qf[NKK];  // loaded by each item itself: prefetched, they held 64 registers over the epilogue and spilled
        {
            const auto rw = row_in(cur, qw * 32 + r32);
            const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + (size_t)rw.b * a.q_stride + (size_t)rw.h * D + hh * 8;
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) qf[kk] = *reinterpret_cast<const f16x8*>(qp + kk * 16);
        }

        // positions relative to p0 from here on (negative: before this split's keys)
        uint32_t wfirst, wlast;
        bool wave_active;
        int base, my_pos;
        if constexpr (PAGED) {
            wave_active = paged_span(a, cur, qw, wfirst, wlast);
            base = cur.pos0 - (int)p0;
            my_pos = base + (int)row_in(cur, qw * 32 + r32).t;
        } else {
            wave_active = wave_span<SPLIT>(a, cur, qw, wfirst, wlast);
            base = (int)(a.pos_start - p0);
            my_pos = base + (int)row_in(cur, qw * 32 + r32).b;
        }
        const int wpos_first = __builtin_amdgcn_readfirstlane(base + (int)wfirst), wpos_last = base + (int)wlast;
        // the pair's tiles
        const uint32_t wsteps = __builtin_amdgcn_readfirstlane(
            wave_active && wpos_last >= 0 ? min((uint32_t)wpos_last / BN + 1, ntiles) : 0);

        // Fragment offsets.  K row r32 + 32 hf, chunk (2 kk + hh) ^ swz: the swizzle changes the chunk's low four bits
        // only, so k-chunks kk and kk + 8 share an offset up to a constant.  V row DH hf + 32 b + r32, chunk
        // (4 kh + 2 s + hh) ^ swz for k-slot s of key half kh.
        const int krow = (r32 + 32 * hf) * D, vrow = (DH * hf + r32) * BN;
        int ko[8], vo[2][2];
#pragma unroll
        for (int j = 0; j < 8; ++j) ko[j] = krow + (((2 * j + hh) ^ chunk_swz<KCH>(r32)) << 3);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            vo[0][s] = vrow + (((4 * hf + 2 * s + hh) ^ chunk_swz<VCH>(r32)) << 3);        // the wave's own half
            vo[1][s] = vrow + (((4 * (hf ^ 1) + 2 * s + hh) ^ chunk_swz<VCH>(r32)) << 3);  // its partner's
        }
        auto read_k = [&](int par, int kk) {
            return *reinterpret_cast<const f16x8*>(kbuf(par) + (ko[kk & 7] + (kk >> 3) * 128));
        };
        auto read_v = [&](int par, int b, int other, int s) {
            return *reinterpret_cast<const f16x8*>(vbuf(par) + (vo[other][s] + 32 * b * BN));
        };
        // keys past kmax in the item's last tile were never stored: their P is 0, their V must be finite
        auto zero_v_tail = [&](int par) {
            const uint32_t valid = kmax - p0 - (ntiles - 1) * BN + 1;
            _Float16* vb = vbuf(par);
            for (int idx = tid; idx < D * VCH; idx += 512) {
                const int d = idx / VCH, c = idx % VCH;
                if ((uint32_t)(8 * c + 7) < valid) continue;
                f16x8* ch = reinterpret_cast<f16x8*>(vb + (d * BN + ((c ^ chunk_swz<VCH>(d)) << 3)));
                f16x8 v = *ch;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((uint32_t)(8 * c + e) >= valid) v[e] = (_Float16)0.0f;
                *ch = v;
            }
        };

        float m = -1e30f, l = 0.0f, mx = 0.0f;
        f32x16 o[NDB];
#pragma unroll
        for (int b = 0; b < NDB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;

        // In a pair's last tile the upper 32 keys can lie past all its queries: their P is 0 but their V need not be
        // finite (an inf of a later key would reach these rows as NaN), so their products read the lower keys' V.
        // Leaves vo like that: nothing follows that tile.  (Paged tiles are cleaned of what is not seen instead.)
        auto upper_v = [&](uint32_t st) {
            if (PAGED || (int)(st * BN) + 32 <= wpos_last) return;  // uniform over the wave
#pragma unroll
            for (int s = 0; s < 2; ++s) vo[0][s] = vo[1][s] = hf ? vo[1][s] : vo[0][s];
        };
        // mask the wave's keys of tile st past the lanes' positions, form their maximum and publish it
        auto tile_max = [&](f32x16& S, uint32_t st) {
            const int k0 = (int)st * BN + 32 * hf;
            if (k0 + 31 > wpos_first) {
                const int rel = my_pos - k0 - 8 * hh;  // element i is key 8 hh + key_of_acc(i, 0) of the half
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key_of_acc(i, 0) > rel) S[i] = -INFINITY;
            }
            mx = S[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, S[i]);
            mx = max_xor32(mx);
            Ml[wave][lane] = mx;
        };
        auto rescale = [&](float other) {
            const float t = fmaxf(mx, other) * a.c;
            if (__ballot(t > m + (LIFT + kSlack))) {  // wave-uniform, and the same for both waves of the pair
                const float mn = t > m + (LIFT + kSlack) ? t - LIFT : m;
                const float alpha = fast_exp2(m - mn);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int b = 0; b < NDB; ++b) o[b] *= alpha;
            }
        };
        auto prob = [&](const f32x16& S, f16x8 (&pf)[2], int i) {
            const float p = fast_exp2(fmaf(S[i], a.c, -m));
            l += p;
            pf[i >> 3][i & 7] = (_Float16)p;
        };
        // O^T += V^T P^T over the wave's own or its partner's keys of the tile in V buffer par
        // (between: called after each MFMA)
        auto pv = [&](const f16x8 (&pf)[2], int par, int other, auto&& between) {
            constexpr int NM = 2 * NDB;  // MFMA n: k-slot n / NDB, block n % NDB
            f16x8 vf[3];
            vf[0] = read_v(par, 0, other, 0);
            vf[1] = read_v(par, 1, other, 0);
#pragma unroll
            for (int n = 0; n < NM; ++n) {
                if (n + 2 < NM) vf[(n + 2) % 3] = read_v(par, (n + 2) % NDB, other, (n + 2) / NDB);
                o[n % NDB] = mfma32(vf[n % 3], pf[n / NDB], o[n % NDB]);
                between(n);
            }
        };
        auto nothing = [](int) {};

        // paged: the tiles cut by the item's mask (clean_v)
        uint32_t cut_tile = ~0u;
        bool odd_v = false;
        if constexpr (PAGED) {
            const uint32_t t = cut_from<BN>(cur);
            if (t != ~0u) cut_tile = t - cur.t0;  // counted from p0
        }
        // whether tile st is cut by the mask or the last one's end (workgroup-uniform); then it is cleaned
        auto clean_tile = [&](int par, uint32_t st) {
            const uint32_t valid = kmax - p0 - st * BN + 1;
            const bool cut = st >= cut_tile;
            if (!cut && valid >= BN) return;
            for (int idx = tid; idx < D * VCH; idx += 512) {
                const int d = idx / VCH, c = idx % VCH;
                odd_v |= clean_v(reinterpret_cast<f16x8*>(vbuf(par) + (d * BN + ((c ^ chunk_swz<VCH>(d)) << 3))), c, valid, cut);
            }
            lds_barrier();
        };

        // prologue: the item's first loads are in flight
        if constexpr (!KV8) dma_done();
        if (a.q_dtype == kBF16) {
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) bf16_to_f16(qf[kk]);
        }
        lds_barrier();
        f32x16 Sa, Sb;
        if (wsteps > 0) {
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) Sa = mfma32(read_k(0, kk), qf[kk], kk == 0 ? f32x16{} : Sa);
            tile_max(Sa, 0);
        }
        if constexpr (KV8) stage.store_k(kbuf(1), tid);
        lds_barrier();

        // step st < ntiles - 1 (ph = st % 2): K(st + 2) replaces K(st), read by the previous step's scores, and
        // V(st + 1) V(st - 1)
        Tile at_k = place(cur, p0, 2), at_v = place(cur, p0, 1);  // of the coming step's loads
        auto step = [&](int ph, uint32_t st, f32x16& Scur, f32x16& Snext) {
            // (8 bits: the last K tile again where none is left; nothing reads it)
            if (KV8 || st + 2 < ntiles) dma_k(kvh, p0, ph, st + 2, at_k);
            dma_v(kvh, p0, ph ^ 1, st + 1, at_v);
            const uint32_t page = page_of(cur, p0, st + 3);  // (read here, used at the step's end)
            // opaque each step, or the compiler keeps a second set of offsets for the other buffers (and spills)
#pragma unroll
            for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(ko[j]));
#pragma unroll
            for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(vo[j >> 1][j & 1]));
            upper_v(st);
            if constexpr (PAGED) clean_tile(ph, st);
            f16x8 pf[2];
            if (st < wsteps) {
                const float other = Ml[wave ^ 1][lane];
                f16x8 kf[3];
                kf[0] = read_k(ph ^ 1, 0);
                kf[1] = read_k(ph ^ 1, 1);
                constexpr int NF = 4;  // score MFMAs ahead of the maximum
#pragma unroll
                for (int n = 0; n < NF; ++n) {
                    kf[(n + 2) % 3] = read_k(ph ^ 1, n + 2);
                    Snext = mfma32(kf[n % 3], qf[n], n == 0 ? f32x16{} : Snext);
                }
                rescale(other);
#pragma unroll
                for (int n = NF; n < NKK; ++n) {
                    if (n + 2 < NKK) kf[(n + 2) % 3] = read_k(ph ^ 1, n + 2);
                    Snext = mfma32(kf[n % 3], qf[n], Snext);
#pragma unroll
                    for (int i = 16 * (n - NF) / (NKK - NF); i < 16 * (n - NF + 1) / (NKK - NF); ++i) prob(Scur, pf, i);
                }
                Pl[wave][0][lane] = pf[0];
                Pl[wave][1][lane] = pf[1];
                if constexpr (KV8) {  // the conversions between the MFMAs (after them, all waves at once: 0.3 us a step)
                    const auto at = stage.place_k(kbuf(ph), tid);
                    pv(pf, ph, 0, [&](int n) {
                        if (n & 1) stage.put_k(at, n >> 1);
                    });
                } else {
                    pv(pf, ph, 0, nothing);
                }
            } else if constexpr (KV8) {
                stage.store_k(kbuf(ph), tid);
            }
            lds_barrier();  // the pair's probabilities are in LDS
            if (st < wsteps) {
                f16x8 po[2];
                po[0] = Pl[wave ^ 1][0][lane];
                po[1] = Pl[wave ^ 1][1][lane];
                if constexpr (KV8) {
                    const auto at = stage.place_v(vbuf(ph ^ 1), tid);
                    pv(po, ph, 1, [&](int n) {
                        if (n & 1) stage.put_v(at, n >> 1);
                    });
                } else {
                    pv(po, ph, 1, nothing);
                }
                tile_max(Snext, st + 1);
            } else if constexpr (KV8) {
                stage.store_v(vbuf(ph ^ 1), tid);
            }
            if constexpr (PAGED) {
                at_v = at_k;
                if constexpr (KV8) at_k = paged8_tile(a, page, kvh);
                else at_k = paged_tile<D>(a, page, kvh);
            }
            if constexpr (!KV8) dma_done();
            lds_barrier();
        };
        // the item's last tile: no scores follow, so both K buffers are free and the next item's first loads go out
        auto last = [&](int ph, uint32_t st, f32x16& Scur) {
            if constexpr (PAGED) has_next = item_of(it + 1, nxt);
            if (!KV8 && has_next) {
                issue_k(nxt);
                if (ph == 1) issue_v(nxt);
            }
            upper_v(st);
            if constexpr (PAGED) {
                clean_tile(ph, st);
            } else if (p0 / BN + ntiles == kmax / BN + 1 && (kmax + 1) % BN != 0) {  // uniform
                zero_v_tail(ph);
                lds_barrier();
            }
            f16x8 pf[2];
            if (st < wsteps) {
                rescale(Ml[wave ^ 1][lane]);
#pragma unroll
                for (int i = 0; i < 16; ++i) prob(Scur, pf, i);
                Pl[wave][0][lane] = pf[0];
                Pl[wave][1][lane] = pf[1];
                pv(pf, ph, 0, nothing);
            }
            lds_barrier();
            if (st < wsteps) {
                f16x8 po[2];
                po[0] = Pl[wave ^ 1][0][lane];
                po[1] = Pl[wave ^ 1][1][lane];
                pv(po, ph, 1, nothing);
            }
            l = sum_xor32(l);
            Ml[wave][lane] = l;  // read for the last time before the barrier above
            lds_barrier();       // and V is read
            if (KV8 && has_next) {load_first(nxt); put_first(nxt);}
            else if (has_next && ph == 0) issue_v(nxt);
        };
        uint32_t st = 0;
        bool odd = false;
        while (st + 1 < ntiles) {
            // (opaque: strength reduction of what st indexes took 30 vector registers and spilled)
            asm volatile("" : "+s"(st));
            step(0, st, Sa, Sb);
            if (++st + 1 >= ntiles) {
                odd = true;
                break;
            }
            step(1, st, Sb, Sa);
            ++st;
        }
        if (odd) last(1, st, Sb);
        else last(0, st, Sa);

        // Epilogue.  A lane holds four dimensions at a time of one query: stored (and the gate read) like that, an
        // instruction would touch 32 rows.  V buffer 1 is free (the next item fills it in its first step), so
        // each wave turns its 32 x 32 blocks of O over in 4 KB of it and then handles 8 rows of 32 dimensions per
        // instruction.  The gate's loads go out first.
        {
            const A& a_e = fresh_args(args);
            int le;  // the lane afresh, so that nothing of this is kept through the key loop
            asm volatile("v_mov_b32 %0, %1" : "=v"(le) : "v"((int)threadIdx.x & 63));
            const int er = le >> 3, ec = le & 7;  // row within a group of 8, four dimensions
            const uint32_t col = hf * DH + 4 * ec;
            bool partial;
            if constexpr (PAGED) partial = cur.part != 0;
            else partial = SPLIT && a_e.n_split > 1;
            // a partial result's row (of rw): its (max, sum), and D floats of O
            auto part_row = [&](const auto& rw, uint32_t r) -> size_t {
                if constexpr (PAGED) return (size_t)(2 * C.j + (cur.part & 1)) * BM + r;
                else return ((size_t)cur.split * a_e.n_heads + rw.h) * a_e.B + rw.b;
            };
            const bool gated = a_e.gate && !partial;
            // rows 8 u + er: the first element written (and of the gate), and whether the row exists
            size_t at[4], gat[4];
            bool valid[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const auto rw = row_from(a_e, cur, qw * 32 + 8 * u + er);
                valid[u] = rw.valid;
                at[u] = partial ? part_row(rw, qw * 32 + 8 * u + er) * D + col
                                : (size_t)rw.b * a_e.out_stride + (size_t)rw.h * D + col;
                gat[u] = (size_t)rw.b * a_e.gate_stride + (size_t)rw.h * D + col;
            }
            f32x4 gt[2][4];
            auto load_gate = [&](int b) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // gate rows are float-aligned
                    gt[b & 1][u] = *reinterpret_cast<const f32x4u*>(a_e.gate + gat[u] + 32 * b);
                }
            };
            if (gated) load_gate(0);
            l += Ml[wave ^ 1][lane];
            // (paged: a row that sees no key is zero)
            float inv = PAGED && l == 0.0f ? 0.0f : 1.0f / l;
            if (partial) {  // (max, sum) and the unnormalised O of the row over this split's keys
                inv = 1.0f;
                const auto rw = row_from(a_e, cur, qw * 32 + (le & 31));
                if (rw.valid && le < 32 && hf == 0) {
                    typedef float f32x2 __attribute__((ext_vector_type(2)));
                    *reinterpret_cast<f32x2*>(a_e.part_ml + 2 * part_row(rw, qw * 32 + (le & 31))) = f32x2{m, l};
                }
            }
            bool add_odd = false;  // paged: add the infs and NaNs cleared from cut tiles
            if constexpr (PAGED) {
                if (cut_tile != ~0u) {  // workgroup-uniform
                    const bool mine = __ballot(odd_v) != 0;
                    if (le == 0) odd_flags[wave] = mine;
                    lds_barrier();
                    for (int w = 0; w < 8; ++w) add_odd = add_odd || odd_flags[w] != 0;
                    lds_barrier();  // read before another item writes there
                }
            }
            f32x4* area = reinterpret_cast<f32x4*>(&Vl1[0]) + wave * 256;  // [32 rows][8 chunks], swizzled
#pragma unroll
            for (int b = 0; b < NDB; ++b) {
                if (gated && b + 1 < NDB) load_gate(b + 1);
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = o[b][4 * i4 + e] * inv;
                    area[(le & 31) * 8 + ((2 * i4 + (le >> 5)) ^ (le & 7))] = v;
                }
                __builtin_amdgcn_wave_barrier();  // one wave's LDS operations stay in order
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    f32x4 v = area[(8 * u + er) * 8 + (ec ^ er)];
                    if constexpr (PAGED) {
                        if (KV8 && add_odd) {
                            if constexpr (KV8) {
                                const uint32_t nan = nan_dims<D>(a_e, cur.seq, cur.kvh, col + 32 * b,
                                                                 cur.pos0 + (int)row_from(a_e, cur, qw * 32 + 8 * u + er).t,
                                                                 (cur.t0 + cut_tile) * BN, (int)min(cur.kmax + 1, (cur.t0 + cur.nt) * BN));
#pragma unroll
                                for (int e = 0; e < 4; ++e) v[e] = nan >> e & 1u ? NAN : v[e];
                            }
                        } else if (add_odd) {
                            const int pos = cur.pos0 + (int)row_from(a_e, cur, qw * 32 + 8 * u + er).t;
#pragma unroll 1
                            for (int e = 0; e < 4; ++e) {
                                const float x = special_sum<D>(a_e, cur.seq, cur.kvh, col + 32 * b + e, pos, (cur.t0 + cut_tile) * BN,
                                                                 (int)min(cur.kmax + 1, (cur.t0 + cur.nt) * BN));
                                v[0] += e == 0 ? x : 0.0f;
                                v[1] += e == 1 ? x : 0.0f;
                                v[2] += e == 2 ? x : 0.0f;
                                v[3] += e == 3 ? x : 0.0f;
                            }
                        }
                    }
                    if (gated) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] *= sigmoid_ref(gt[b & 1][u][e]);
                    }
                    if (!valid[u]) continue;
                    if (partial) *reinterpret_cast<f32x4*>(a_e.part_o + at[u] + 32 * b) = v;
                    else store_out4(a_e.out, at[u] + 32 * b, a_e.out_dtype, v);
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
        if (!has_next) break;
        cur = nxt;
    }
    if constexpr (PAGED) paged_leave(args, C, cur);
}

}  // namespace
}  // namespace yhip
