// paged_items.hpp -- how the work of a paged attention launch is dealt out.
//
// A sequence's new tokens form items of up to 128 rows that share a kv head:
// with 128 tokens or more, 128 consecutive tokens of one query head; with
// fewer, the group's heads' tokens one after the other.  An item walks the
// keys its last row sees, in units of 64.  All units of the launch, sequence
// by sequence, form one line, which is cut into equal chunks, one per resident
// workgroup: whatever the lengths of the batch, every workgroup walks the same
// number of units.  A cut inside an item leaves partial results (running
// maximum, sum and unnormalised output), at most one at each end of a chunk,
// which a merge kernel joins in order; cuts inside short items move to the
// item's start, which costs less than joining them.  (One sequence may go item
// by item instead, paged_whole.)  Lengths are read on the device, so a captured
// launch replays with new ones.
#pragma once

#include "common.hpp"
#include "internal.hpp"
#include "paged_chunks.hpp"

namespace yhip {
namespace {

constexpr uint32_t kItemRows = 128;
constexpr uint32_t kUnitKeys = 64;

__device__ inline uint32_t uni(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ inline uint64_t uni64(uint64_t x) { return (uint64_t)uni((uint32_t)(x >> 32)) << 32 | uni((uint32_t)x); }

// tables and lengths do not change during a launch: uniform reads may go
// through the scalar cache
typedef const int __attribute__((address_space(4))) * ConstInts;
__device__ inline ConstInts const_ints(const int* p) { return (ConstInts)(uintptr_t)p; }

// a / b for a below 2^21: the quotient with a + 1/2 is at least 1/(2 b) off
// every whole number, more than the reciprocal's error makes (five
// instructions for some thirty-five)
__device__ inline uint32_t div_small(uint32_t a, uint32_t b)
{
    return (uint32_t)(((float)a + 0.5f) * __builtin_amdgcn_rcpf((float)b));
}

// first query head of kv head g (common mapping h * n_kv / n_heads)
__device__ inline uint32_t head0(const PagedAttnArgs& a, uint32_t g)
{
    return a.gmax * a.n_kv == a.n_heads ? g * a.gmax : (g * a.n_heads + a.n_kv - 1) / a.n_kv;
}

// A sequence's rows and keys: rows row0 .. row0 + nq - 1, token t at position
// pos0 + t (negative: sees nothing), L keys.
struct PagedSeq {
    uint32_t row0, nq;
    int pos0, L;
};

__device__ inline PagedSeq paged_seq(const PagedAttnArgs& a, int c0, int c1, int len)
{
    PagedSeq s;
    s.row0 = min((uint32_t)max(c0, 0), a.n_tok);
    const uint32_t n = min((uint32_t)max(c1, 0), a.n_tok) - s.row0;
    s.nq = (int)n > 0 ? min(n, a.max_new) : 0u;
    s.L = min(max(len, 0), (int)a.max_len);
    s.pos0 = s.L - (int)((int)n > 0 ? n : 0u);
    return s;
}

__device__ inline uint32_t units_to(int keys) { return keys > 0 ? ((uint32_t)keys + kUnitKeys - 1) / kUnitKeys : 1u; }

// An item costs its tiles and kItemUnits more (queries in, first tiles, output
// out), which the line counts as units before its first tile: without them a
// chunk of many short items ran far longer than one of a few long ones (a
// prompt of 8192 tokens, 32 / 8 heads of 128: 733 us, 600 with them; 12 of
// them are too many, 5 too few).
constexpr uint32_t kItemUnits = 8;

// Units of one query head's (or one packed group's) items, in order:
// packed items all see every key; of plain ones, block b of 128 tokens sees
// c + 2 (b + 1) tiles (c: those of the keys before the new tokens), the last
// block all.  (Tokens at negative positions are counted as if at their index;
// the walk leaves out what is not there.)
__device__ inline uint32_t plain_c(const PagedSeq& s) { return ((uint32_t)max(s.pos0, 0) + kUnitKeys - 1) / kUnitKeys + kItemUnits; }
__device__ inline uint32_t plain_before(uint32_t b, uint32_t c) { return b * c + b * (b + 1); }
__device__ inline uint32_t plain_last(const PagedSeq& s) { return units_to(max(s.pos0, 0) + (int)s.nq) + kItemUnits; }

__device__ inline uint64_t seq_units(const PagedAttnArgs& a, const PagedSeq& s)
{
    if (s.nq == 0) return 0;
    if (s.nq < kItemRows) return (uint64_t)a.n_kv * ((a.gmax * s.nq + kItemRows - 1) / kItemRows) * (units_to(s.L) + kItemUnits);
    const uint32_t nb = (s.nq + kItemRows - 1) / kItemRows, c = plain_c(s);
    return (uint64_t)a.n_kv * a.gmax * (plain_before(nb - 1, c) + plain_last(s));
}

// How the line of units is made up (paged_decode.hip has another)
struct PagedLine {
    static __device__ uint64_t units(const PagedAttnArgs& a, const PagedSeq& s) { return seq_units(a, s); }
};

// A piece of an item: `n` key tiles from t0 on.  part: 0 the whole item, 1 its
// first piece, 2 a later one.  idle: no key of it is seen (its tile is loaded
// and not used).
struct PagedItem {
    uint32_t seq, row0, nq, kvh, h, qb, pack;
    int pos0;
    uint32_t kmax, t0, nt, part, idle, last;
};

// what a workgroup that begins a split item leaves for the merge
struct PagedDesc {
    uint32_t n;  // pieces; 0: none
    uint32_t row0, nq, kvh, h, qb, pack, pad;
};

// Where a workgroup is in its chunk of `len` units: `done` of them are behind
// it (negative: units taken over from the chunk before), the next is unit `off`
// of sequence seq.
struct PagedCursor {
    uint32_t seq, off, chunk, j;
    int done, len;
    bool fresh;
};

__device__ inline PagedSeq cursor_seq(const PagedAttnArgs& a, uint32_t seq)
{
    const ConstInts cu = const_ints(a.cu_new);
    return paged_seq(a, cu[seq], cu[seq + 1], const_ints(a.kv_lens)[seq]);
}

// The launch's arguments, read again: kept in scalar registers from one end of
// an item to the other they displaced what the key loop needs.
__device__ inline const PagedAttnArgs& fresh_args(const PagedAttnArgs&)
{
    auto p = (const PagedAttnArgs __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const PagedAttnArgs*)p;
}

// This workgroup's chunk, units begin .. of a line of `total`; false if it has
// none.  Active chunks are spread over the XCDs (consecutive workgroups go to
// the 8 XCDs in turn), neighbours on one XCD, whose L2 then holds the keys they
// share.
__device__ inline bool paged_chunk(const PagedAttnArgs& a, PagedCursor& C, uint64_t total, uint64_t& begin)
{
    const PagedChunks cut = paged_chunks(total, a.n_wg, a.min_units);
    C.chunk = cut.units;
    const uint32_t active = min(cut.n, a.n_wg);  // (more only if offsets that overlap pass the bounds checked on the host)
    const uint32_t x = blockIdx.x % 8u, y = blockIdx.x / 8u, share = (active + 7u) / 8u;
    C.j = y < share ? x * share + y : 8u * share + (y - share) * 8u + x;
    begin = (uint64_t)C.j * C.chunk;
    C.done = 0;
    C.len = (int)min((uint64_t)C.chunk, total - begin);
    C.fresh = true;
    return C.j < active;
}

// This workgroup's place in the line; false if it has no chunk.  `scratch`: 24
// words of LDS, free again after the call's last barrier.
template <int NT, class Line = PagedLine>
__device__ inline bool paged_start(const PagedAttnArgs& a, uint64_t* scratch, PagedCursor& C)
{
    if (a.n_seq == 1) {  // nothing to scan
        C.seq = 0;
        uint64_t begin;
        const bool any = paged_chunk(a, C, Line::units(a, cursor_seq(a, 0)), begin);
        C.off = (uint32_t)begin;
        return any;
    }
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const bool small = a.n_seq <= 64u;  // every wave scans for itself
    const uint32_t per = small ? 1u : (a.n_seq + NT - 1) / NT;
    const uint32_t lo = min((small ? lane : t) * per, a.n_seq), hi = min(lo + per, a.n_seq);
    uint64_t sum = 0;
    for (uint32_t i = lo; i < hi; ++i) sum += Line::units(a, paged_seq(a, a.cu_new[i], a.cu_new[i + 1], a.kv_lens[i]));
    uint64_t inc = sum;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up((unsigned long long)inc, d);
        if (lane >= d) inc += o;
    }
    uint64_t before = inc - sum, total = uni64(__shfl((unsigned long long)inc, 63));
    if (!small) {
        if (lane == 63) scratch[wave] = inc;
        __syncthreads();
        total = 0;
#pragma unroll
        for (uint32_t w = 0; w < NT / 64; ++w) {
            if (w < wave) before += scratch[w];
            total += scratch[w];
        }
        total = uni64(total);
    }
    uint64_t begin;
    if (!paged_chunk(a, C, total, begin)) return false;  // workgroup-uniform
    const bool mine = before <= begin && begin < before + sum;
    if (small) {
        const uint32_t at = (uint32_t)__builtin_ctzll(__ballot(mine));
        C.seq = at;
        C.off = (uint32_t)(begin - uni64(__shfl((unsigned long long)before, (int)at)));
    } else {
        if (mine) {
            uint32_t i = lo;
            for (;; ++i) {
                const uint64_t n = Line::units(a, paged_seq(a, a.cu_new[i], a.cu_new[i + 1], a.kv_lens[i]));
                if (begin < before + n) break;
                before += n;
            }
            scratch[16] = i;
            scratch[17] = begin - before;
        }
        __syncthreads();
        C.seq = uni((uint32_t)scratch[16]);
        C.off = uni((uint32_t)scratch[17]);
        __syncthreads();
    }
    return true;
}

// An item of T units, the cursor at its unit t: moves the cursor past the
// chunk's piece of it, units t .. t + n - 1; false if the chunk ends before
// it.  Cuts inside items of at most snap_units + fixed units, and at or before
// unit `start`, move to the item's start (the chunk that begins with such a
// cut takes the item whole, t becomes 0).  last: the chunk that ends the item.
__device__ inline bool paged_cut(const PagedAttnArgs& a, PagedCursor& C, uint32_t T, uint32_t& t, uint32_t fixed,
                                 uint32_t start, uint32_t& n, uint32_t& last)
{
    auto at_start = [&](uint32_t cut) { return T <= a.snap_units + fixed || cut <= start; };
    if (C.fresh && t > 0 && at_start(t)) {
        C.off -= t;
        C.done -= (int)t;
        t = 0;
    }
    C.fresh = false;
    const int to_end = C.done + (int)(T - t);  // of the chunk, at the item's end
    n = T - t;
    if (to_end > C.len) {  // the chunk ends inside the item
        n = (uint32_t)(C.len - C.done);
        if (at_start(t + n)) {
            C.done = C.len;
            return false;
        }
    }
    last = C.j + (uint32_t)(to_end - 1) / C.chunk;
    C.off += n;
    C.done += (int)n;
    return true;
}

// The chunk's next piece in tiles of BN keys; false past its end.
template <int BN>
__device__ inline bool paged_next(const PagedAttnArgs& a, PagedCursor& C, PagedItem& I)
{
    constexpr uint32_t TU = kUnitKeys / BN;  // tiles per unit
    for (;;) {
        if (C.done >= C.len) return false;
        PagedSeq s = cursor_seq(a, C.seq);
        uint32_t units = (uint32_t)seq_units(a, s);  // (below 2^31, checked on the host)
        while (C.off >= units) {
            C.off -= units;
            s = cursor_seq(a, ++C.seq);
            units = (uint32_t)seq_units(a, s);
        }
        const uint32_t per_kv = units / a.n_kv, kvh = C.off / per_kv;
        uint32_t rem = C.off - kvh * per_kv, T, t;
        const uint32_t h0 = head0(a, kvh), h1 = head0(a, kvh + 1);
        I.pack = s.nq < kItemRows;
        bool none;  // an item of the fullest group that this one does not have
        int seen;
        if (I.pack) {
            T = units_to(s.L) + kItemUnits;
            I.qb = rem / T;
            t = rem - I.qb * T;
            I.h = h0;
            none = I.qb * kItemRows >= (h1 - h0) * s.nq;
            seen = s.L;
        } else {
            const uint32_t nb = (s.nq + kItemRows - 1) / kItemRows, c = plain_c(s);
            // block b with plain_before(b) <= rem / gmax < plain_before(b + 1)
            const uint32_t want = rem / a.gmax;
            const float hc = 0.5f * (float)(c + 1u);
            uint32_t b = (uint32_t)max(sqrtf(hc * hc + (float)want) - hc, 0.0f);
            b = min(b, nb - 1);
            while (b > 0 && plain_before(b, c) > want) --b;
            while (b + 1 < nb && plain_before(b + 1, c) <= want) ++b;
            rem -= a.gmax * plain_before(b, c);
            T = b + 1 < nb ? c + 2 * (b + 1) : plain_last(s);
            const uint32_t g = rem / T;
            t = rem - g * T;
            I.qb = b;
            I.h = h0 + g;
            none = I.h >= h1;
            seen = s.pos0 + (int)min(s.nq, (b + 1) * kItemRows);
        }
        uint32_t n;
        if (!paged_cut(a, C, T, t, kItemUnits, kItemUnits + 1, n, I.last)) return false;
        if (none) continue;
        I.part = n == T ? 0u : t == 0 ? 1u : 2u;
        const uint32_t tile0 = t ? t - kItemUnits : 0u;  // the piece's tiles of 64 keys
        n -= t ? 0u : kItemUnits;
        I.seq = C.seq;
        I.row0 = s.row0;
        I.nq = s.nq;
        I.pos0 = s.pos0;
        I.kvh = kvh;
        I.kmax = (uint32_t)max(seen - 1, 0);
        const uint32_t all = I.kmax / BN + 1;
        I.t0 = tile0 * TU;
        I.idle = seen <= 0 || I.t0 >= all;
        if (I.idle) {
            I.t0 = all - 1;
            I.nt = 1;
        } else {
            I.nt = min(all - I.t0, n * TU);
        }
        return true;
    }
}

// The item of this workgroup where each takes a whole one of the only sequence
// (n_wg 0: paged_whole_wgs, attn_paged.hip), those of the last tokens, the
// longest, first; false if there is none.
template <int BN>
__device__ inline bool paged_whole(const PagedAttnArgs& a, PagedItem& I)
{
    const PagedSeq s = cursor_seq(a, 0);
    const uint32_t w = blockIdx.x;
    int seen;
    I.pack = s.nq < kItemRows;
    if (I.pack) {
        I.qb = w / a.n_kv;
        I.kvh = w - I.qb * a.n_kv;
        I.h = head0(a, I.kvh);
        if (I.qb * kItemRows >= (head0(a, I.kvh + 1) - I.h) * s.nq) return false;
        seen = s.L;
    } else {
        const uint32_t nb = (s.nq + kItemRows - 1) / kItemRows, i = w / a.n_heads;
        if (i >= nb) return false;
        I.qb = nb - 1 - i;
        I.h = w - i * a.n_heads;
        I.kvh = I.h * a.n_kv / a.n_heads;
        seen = s.pos0 + (int)min(s.nq, (I.qb + 1) * kItemRows);
    }
    I.part = I.last = I.seq = I.t0 = 0;
    I.row0 = s.row0;
    I.nq = s.nq;
    I.pos0 = s.pos0;
    I.kmax = (uint32_t)max(seen - 1, 0);
    I.idle = seen <= 0;
    I.nt = I.kmax / BN + 1;
    return true;
}

// The workgroup's first piece; false if it has none.
template <int NT, int BN>
__device__ inline bool paged_first(const PagedAttnArgs& args, uint64_t* scratch, PagedCursor& C, PagedItem& I)
{
    if (args.n_wg == 0) {
        C = PagedCursor{};  // an empty chunk: nothing comes after the item
        return paged_whole<BN>(fresh_args(args), I);
    }
    if (paged_start<NT>(fresh_args(args), scratch, C) && paged_next<BN>(fresh_args(args), C, I)) return true;
    if (threadIdx.x == 0) reinterpret_cast<PagedDesc*>(args.desc)[C.j].n = 0;
    return false;
}

// The workgroup's last piece, which may begin a split item: what the merge
// needs to know of it.
__device__ inline void paged_leave(const PagedAttnArgs& a, const PagedCursor& C, const PagedItem& I)
{
    if (threadIdx.x != 0 || a.n_wg == 0) return;
    PagedDesc* d = reinterpret_cast<PagedDesc*>(a.desc) + C.j;
    if (I.part == 1) *d = PagedDesc{I.last - C.j + 1, I.row0, I.nq, I.kvh, I.h, I.qb, I.pack, 0};
    else d->n = 0;
}

// byte address and size (0: outside the pool) of kv head kvh's part of the
// page that holds key `key`; K rows and V tiles of a page are the same bytes
struct PagedTile {
    uint64_t at;
    uint32_t bytes;
};
template <int D>
__device__ inline PagedTile paged_tile(const PagedAttnArgs& a, uint32_t page, uint32_t kvh)
{
    const bool in = page < a.n_blocks;
    const uint32_t lg = a.shift + (D == 64 ? 7 : D == 128 ? 8 : 9);  // (n_blocks * n_kv fits 32 bits, checked on the host)
    return PagedTile{(uint64_t)(in ? page * a.n_kv + kvh : 0u) << lg, in ? 1u << lg : 0u};
}
__device__ inline uint32_t paged_page(const PagedAttnArgs& a, uint32_t seq, uint32_t key)
{
    return (uint32_t)const_ints(a.table + (size_t)seq * a.table_stride)[key >> a.shift];
}

// ---- shared by the kernels ----

__device__ inline float sigmoid_ref(float g) { return 1.0f / (1.0f + expf(-g)); }

__device__ inline void store_out4(void* out, size_t off, uint32_t dt, f32x4 v)
{
    if (dt == kF32) {
        *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(out) + off) = v;
    } else if (dt == kF16) {
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        f16x4 h;
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = (_Float16)v[j];
        *reinterpret_cast<f16x4*>(reinterpret_cast<uint16_t*>(out) + off) = h;
    } else {
        // gfx950's own conversion, to nearest even (an addition to the bits would carry a NaN of all ones to zero)
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        bf16x4 h;
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = (__bf16)v[j];
        *reinterpret_cast<bf16x4*>(reinterpret_cast<uint16_t*>(out) + off) = h;
    }
}

// Probabilities enter the products scaled by 2^kLift: the running maximum that
// they are formed against stays kLift below the true one, in powers of two, as
// it is up to kSlack behind it (so that it seldom moves), and 2^(kLift + kSlack)
// is below f16's largest.  f16 has nothing below 2^-25: without the scale, keys
// below 2^-25 of the largest counted as nothing, and 100,000 of them are 2^-8 of
// a row (a key that draws nearly all the attention, over a long context).  Sums
// and partial results carry the scale; the division takes it out.
constexpr float kSlack = 8.0f, kLift = 7.0f;

// Values for the product with the probabilities' lo parts: an inf or NaN as a
// finite value.  The hi parts bring it in; with a lo part, 0 or negative
// beside a positive hi, the same inf would make NaN.
__device__ inline f16x8 bounded(const f16x8& v)
{
    const f16x8 top = {65504, 65504, 65504, 65504, 65504, 65504, 65504, 65504};
    return __builtin_elementwise_max(__builtin_elementwise_min(v, top), -top);
}
// The sum of the infs and NaNs among the values of dimension d that a query at
// position pos sees of keys lo .. end - 1.
template <int D>
__device__ float special_sum(const PagedAttnArgs& a, uint32_t seq, uint32_t kvh, uint32_t d, int pos, uint32_t lo, int end)
{
    float s = 0.0f;
#pragma unroll 1
    for (uint32_t k = lo; (int)k < end && (int)k <= pos; ++k) {
        const PagedTile t = paged_tile<D>(a, (uint32_t)a.table[(size_t)seq * a.table_stride + (k >> a.shift)], kvh);
        if (t.bytes == 0) continue;
        const uint32_t off = k & ((1u << a.shift) - 1u);
        const uint16_t* p = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(a.vc) + t.at);
        const uint16_t b = p[(size_t)(off & ~31u) * D + d * kVTile + (off & 31u)];
        if ((b & 0x7fff) >= 0x7c00) s += f16_bits_to_f32(b);
    }
    return s;
}
}  // namespace
}  // namespace yhip
