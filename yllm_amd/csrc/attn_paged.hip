// attn_paged.hip -- causal grouped-query attention of each sequence's new
// tokens over its pages of a KV pool.
//
// Token t of the n new ones of a sequence with L stored positions (its own
// included) sits at position p = L - n + t and attends to keys 0 .. p
// (engine.c:532-563 with the sequence's own start); a token at a negative
// position sees nothing and its row is zero.  Key j of a sequence is row
// j % block of page table[j / block].
//
// The products run on the prefill kernels (prefill_kernel.hpp) over pieces of
// 128-row items, dealt out as paged_items.hpp says; the merge kernel here
// joins the pieces of items that a chunk's end cut.
//
// Measured: a prompt of 8192 tokens, 32 / 8 heads of 128, 595 to 612 us by box,
// 900 to 924 TFLOP/s (a contiguous cache: 553 to 600), of them 14 for the merge
// and as much for the partial results it reads; a gated chunk of 2048 tokens at
// 2048, 16 / 2 heads of 256, 140 us, 735 TFLOP/s.  A short call is a chain: 1.7 us
// to the piece, 3.3 to its first tiles, 1.2 a tile, 2 to 3 out.
#include "common.hpp"
#include "internal.hpp"
#include "paged_items.hpp"
#include "prefill_kernel.hpp"

#include <algorithm>

namespace yhip {
namespace {

constexpr uint32_t kMergeRows = 4;  // rows of a merge thread

// Workgroup (j, y): the y-th 256 / (D / 4) rows of the split item that chunk j
// begins, if any.  Pieces are joined in their order; a thread holds four
// dimensions of a row.  Nearly all split items of a full launch have two
// pieces: there every kMergeRows-th workgroup takes the rows of as many, and
// their loads, and the gate's, go out together (one row after the other, 16
// dependent round trips: 2048 tokens of 16 / 2 heads of 256 with a gate merged
// in 22 us; so, in 19, 6 TB/s).
template <int D>
__device__ __forceinline__ void paged_merge(const PagedAttnArgs& a, uint32_t j, uint32_t y)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t C4 = D / 4, RP = 256 / C4, kRound = 8;
    const PagedDesc d = reinterpret_cast<const PagedDesc*>(a.desc)[j];
    if (d.n == 0) return;
    const uint32_t dim = threadIdx.x % C4 * 4u, r0 = y * RP + threadIdx.x / C4;
    if (d.n == 2 && y % kMergeRows != 0) return;
    auto finish = [&](const PagedRow& rw, f32x4 O, float L, const f32x4& g) {
        f32x4 v = O * (L == 0.0f ? 0.0f : 1.0f / L);
        if (a.gate) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= sigmoid_ref(g[e]);
        }
        store_out4(a.out, (size_t)rw.b * a.out_stride + (size_t)rw.h * D + dim, a.out_dtype, v);
    };
    auto gate_of = [&](const PagedRow& rw) {
        typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // gate rows are float-aligned
        return (f32x4)*reinterpret_cast<const f32x4u*>(a.gate + (size_t)rw.b * a.gate_stride + (size_t)rw.h * D + dim);
    };
    if (d.n == 2) {
        PagedRow rw[kMergeRows];
        f32x2 ml[kMergeRows][2];
        f32x4 os[kMergeRows][2], g[kMergeRows];
#pragma unroll
        for (uint32_t i = 0; i < kMergeRows; ++i) {  // rows past the item's end read its last row's
            rw[i] = paged_row(a, d, r0 + i * RP);
            const uint32_t r = min(r0 + i * RP, kItemRows - 1);
            const size_t p0 = (size_t)(2 * j + 1) * kItemRows + r, p1 = (size_t)(2 * j + 2) * kItemRows + r;
            ml[i][0] = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * p0);
            ml[i][1] = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * p1);
            os[i][0] = *reinterpret_cast<const f32x4*>(a.part_o + p0 * D + dim);
            os[i][1] = *reinterpret_cast<const f32x4*>(a.part_o + p1 * D + dim);
            g[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (a.gate) g[i] = gate_of(rw[i]);
        }
#pragma unroll
        for (uint32_t i = 0; i < kMergeRows; ++i) {
            const float M = fmaxf(ml[i][0][0], ml[i][1][0]);
            const float c0 = fast_exp2(ml[i][0][0] - M), c1 = fast_exp2(ml[i][1][0] - M);
            if (rw[i].valid) finish(rw[i], os[i][0] * c0 + os[i][1] * c1, ml[i][0][1] * c0 + ml[i][1][1] * c1, g[i]);
        }
        return;
    }
    {
        const uint32_t r = r0;
        const PagedRow rw = paged_row(a, d, r);
        if (!rw.valid) return;
        float M = -1e30f, L = 0.0f;
        f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
        for (uint32_t s0 = 0; s0 < d.n; s0 += kRound) {
            f32x2 ml[kRound];
            f32x4 os[kRound];
#pragma unroll
            for (uint32_t k = 0; k < kRound; ++k) {
                // piece s in slot 2 (j + s) + (s == 0); past the last one, the first again, counted as nothing
                const uint32_t s = s0 + k < d.n ? s0 + k : 0u;
                const size_t p = (size_t)(2 * (j + s) + (s == 0)) * kItemRows + r;
                ml[k] = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * p);
                os[k] = *reinterpret_cast<const f32x4*>(a.part_o + p * D + dim);
            }
            float mr = M;
#pragma unroll
            for (uint32_t k = 0; k < kRound; ++k)
                if (s0 + k < d.n) mr = fmaxf(mr, ml[k][0]);
            const float co = fast_exp2(M - mr);
            L *= co;
            O *= co;
#pragma unroll
            for (uint32_t k = 0; k < kRound; ++k) {
                if (s0 + k >= d.n) continue;
                const float c = fast_exp2(ml[k][0] - mr);
                L += ml[k][1] * c;
                O += os[k] * c;
            }
            M = mr;
        }
        f32x4 g = f32x4{0.f, 0.f, 0.f, 0.f};
        if (a.gate) g = gate_of(rw);
        finish(rw, O, L, g);
    }
}

template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a)
{
    paged_merge<D>(a, blockIdx.x, blockIdx.y);
}

// Both lines' (PagedMixed8Args): `tile_wgs` workgroups for the tiles', then one for each row of the other's chunks (four
// of four rows: 46.5 us for 45.0, a mixed step of 14 / 2 heads of 64)
template <int D>
__global__ __launch_bounds__(256) void paged_mixed8_merge_kernel(PagedMixed8Args a, uint32_t tile_wgs)
{
    if (blockIdx.x < tile_wgs) {
        paged_merge<D>(a, blockIdx.x % a.n_wg, blockIdx.x / a.n_wg);
        return;
    }
    const uint32_t w = blockIdx.x - tile_wgs;
    decode8_merge<D>(a.part, w % a.part.n_wg, w / a.part.n_wg);
}

}  // namespace

namespace {

// The longest item that is not cut (without its fixed units), and the shortest
// chunk, in units of 64 keys.  Where a line does not fill the GPU, a piece more
// of an item of T units costs its merge 0.4 us, and a unit more of a piece its
// walk 1.2: pieces of sqrt(T / 3) units (28 / 4 heads of 128, 16 tokens at 1000:
// 19 us, 25 with pieces of nine; 14 / 2 heads of 64, 64 tokens at 16000: 26, 34
// with pieces of four).
constexpr uint32_t kSnapUnits = 4, kMinUnits = 4;
uint32_t min_units(uint32_t max_len)
{
    const uint32_t T = (max_len - 1) / kUnitKeys + 1 + kItemUnits;
    return std::max(kMinUnits, (uint32_t)lroundf(sqrtf((float)T / 3.0f)));
}

uint32_t round8(uint64_t x) { return (uint32_t)((x + 7) / 8 * 8); }

// Workgroups of a launch: what the GPU holds at once (per_cu a CU), or all that
// the bounds on the batch can fill with chunks of `shortest` units.  (A workspace
// is sized for the shortest there are: larger bounds never need less.)
uint32_t paged_wgs(uint32_t n_tok, uint32_t n_seq, uint32_t max_len, uint32_t n_heads, uint32_t n_kv, uint32_t per_cu,
                   uint32_t shortest)
{
    const uint64_t gmax = (n_heads + n_kv - 1) / n_kv;
    const uint64_t items = (uint64_t)n_kv * gmax * ((uint64_t)n_tok / kItemRows + n_seq);
    const uint64_t units = ((uint64_t)max_len + kUnitKeys - 1) / kUnitKeys + kItemUnits;
    const uint64_t most = (items * units + shortest - 1) / shortest;
    const uint64_t full = (uint64_t)per_cu * (uint64_t)n_cus();
    return round8(most < full ? most : full);
}

// Workgroups of a launch that gives each a whole item of its one sequence,
// without the merge; 0: it does not.  Where a whole item's walk takes no longer than a piece's with what cutting
// costs, the merge's launch and its partial results (28 / 4 heads of 128, 1000
// tokens: 31 us, 39 cut; 2048: 55, 66; 16 / 2 heads of 256, 2048 at 2048: 142,
// 149; 14 / 2 heads of 64, 2048, where cutting is better: 38, 35).  In
// microseconds, a tile 1 to 2 by head_dim, more with two workgroups on a CU.
uint32_t paged_whole_wgs(const PagedAttnArgs& a, uint32_t per_cu, bool qs)
{
    if (a.n_seq != 1) return 0;
    const uint64_t cus = (uint64_t)n_cus(), tiles = ((uint64_t)a.max_len + kUnitKeys - 1) / kUnitKeys;
    const bool pack = a.max_new < kItemRows;
    const uint64_t items = pack ? (uint64_t)a.n_kv * ((a.gmax * a.max_new + kItemRows - 1) / kItemRows)
                                : (uint64_t)a.n_kv * a.gmax * ((a.max_new + kItemRows - 1) / kItemRows);
    if (items > cus * per_cu) return 0;
    const double mean = (double)tiles - (pack ? 0.0 : std::min(a.max_new, a.max_len) / (2.0 * kUnitKeys));
    const double piece = std::max(((double)items * (mean + kItemUnits)) / a.n_wg, (double)a.min_units);
    const double pieces = (double)items * (mean + kItemUnits) / piece;
    const double tile = (a.D == 64 ? 1.0 : a.D == 128 ? 1.2 : 2.0) * (qs ? 1.5 : 1.0);
    const double whole = tile * std::max((double)tiles, items > cus ? 1.5 * mean : 0.0);
    const double cut = tile * piece * (pieces > (double)cus ? 1.25 : 1.0) + 5.0 + pieces * a.D * 2e-4;
    return whole <= cut ? (uint32_t)items : 0;
}

size_t align256a(size_t x) { return (x + 255) / 256 * 256; }

size_t paged_bytes(uint32_t wgs, uint32_t D)
{
    const size_t rows = (size_t)2 * wgs * kItemRows;
    return align256a((size_t)wgs * sizeof(PagedDesc)) + align256a(rows * 2 * sizeof(float)) + rows * D * sizeof(float);
}

template <int D, int NG, bool QS, class A>
void launch_tiles(const A& a, uint32_t grid, hipStream_t st)
{
    constexpr int threads = 256 * NG * (D > 128 ? 2 : 1);
    hipLaunchKernelGGL((prefill_kernel<D, NG, false, QS, A>), dim3(grid), dim3(threads), 0, st, a);
}

// an item may be split (with more new tokens than keys its units go by its tokens, paged_items.hpp)
bool may_split(const PagedAttnArgs& a) { return std::max(a.max_len, a.max_new) > a.snap_units * kUnitKeys; }
uint32_t merge_wgs(const PagedAttnArgs& a)  // for a chunk
{
    const uint32_t rp = 1024u / a.D;  // rows of a merge workgroup
    return (std::min(a.gmax * a.max_new, kItemRows) + rp - 1) / rp;
}

// what the launcher sets
void set_line(PagedAttnArgs& a, uint32_t per_cu)
{
    a.gmax = (a.n_heads + a.n_kv - 1) / a.n_kv;
    a.min_units = min_units(a.max_len);
    a.n_wg = paged_wgs(a.n_tok, a.n_seq, a.max_len, a.n_heads, a.n_kv, per_cu, a.min_units);
    a.snap_units = kSnapUnits;
    char* p = reinterpret_cast<char*>(a.ws);
    a.desc = p;
    p += align256a((size_t)a.n_wg * sizeof(PagedDesc));
    a.part_ml = reinterpret_cast<float*>(p);
    a.part_o = reinterpret_cast<float*>(p + align256a((size_t)2 * a.n_wg * kItemRows * 2 * sizeof(float)));
}

template <class A>
hipError_t launch_items(const A& in, hipStream_t st)
{
    A a = in;
    const bool qs = a.q_dtype == kF32;
    const uint32_t per_cu = a.D <= 128 && !qs ? 2 : 1;
    set_line(a, per_cu);
    const uint32_t whole = paged_whole_wgs(a, per_cu, qs), grid = whole ? whole : a.n_wg;
    if (whole) a.n_wg = 0;
    switch (a.D) {
    case 64: qs ? launch_tiles<64, 1, true>(a, grid, st) : launch_tiles<64, 1, false>(a, grid, st); break;
    case 128: qs ? launch_tiles<128, 2, true>(a, grid, st) : launch_tiles<128, 1, false>(a, grid, st); break;
    case 256:
        if (qs) launch_tiles<256, 1, true>(a, grid, st);
        else hipLaunchKernelGGL((prefill_halves_kernel<256, false, A>), dim3(grid), dim3(512), 0, st, a);
        break;
    default: return hipErrorInvalidValue;
    }
    if (!whole && may_split(a)) {
        const dim3 merge(a.n_wg, merge_wgs(a));
        switch (a.D) {
        case 64: hipLaunchKernelGGL(paged_merge_kernel<64>, merge, dim3(256), 0, st, static_cast<const PagedAttnArgs&>(a)); break;
        case 128: hipLaunchKernelGGL(paged_merge_kernel<128>, merge, dim3(256), 0, st, static_cast<const PagedAttnArgs&>(a)); break;
        default: hipLaunchKernelGGL(paged_merge_kernel<256>, merge, dim3(256), 0, st, static_cast<const PagedAttnArgs&>(a)); break;
        }
    }
    return hipGetLastError();
}

}  // namespace

size_t paged_attn_workspace(uint32_t n_tok, uint32_t n_seq, uint32_t max_new, uint32_t max_len, uint32_t n_heads,
                            uint32_t n_kv, uint32_t D)
{
    // (the decode kernel's, where it serves every call within the bounds; else also large enough for its calls)
    const size_t decode = paged_decode_workspace(n_seq, max_len, n_kv, D);
    if (paged_decode_fits(n_heads, n_kv, max_new)) return decode;
    return std::max(decode, paged_bytes(paged_wgs(n_tok, n_seq, max_len, n_heads, n_kv, D <= 128 ? 2 : 1, kMinUnits), D));
}

hipError_t launch_paged_attn(const PagedAttnArgs& a, hipStream_t st)
{
    return paged_decode_fits(a.n_heads, a.n_kv, a.max_new) ? launch_paged_decode(a, st) : launch_items(a, st);
}

size_t paged_tiles8_workspace(uint32_t n_tok, uint32_t n_seq, uint32_t max_len, uint32_t n_heads, uint32_t n_kv, uint32_t D)
{
    return paged_bytes(paged_wgs(n_tok, n_seq, max_len, n_heads, n_kv, D <= 128 ? 2 : 1, kMinUnits), D);
}
hipError_t launch_paged_tiles8(const PagedAttn8Args& a, hipStream_t st) { return launch_items(a, st); }

// (16-bit queries, head_dim 64 or 128: both kinds' workgroups are of 256 threads, two to a CU)
hipError_t launch_paged_mixed8(const PagedAttn8Args& tiles, const PagedAttn8Args& few, hipStream_t st)
{
    PagedMixed8Args a;
    static_cast<PagedAttn8Args&>(a) = tiles;
    static_cast<PagedAttn8Args&>(a.part) = few;
    set_line(a, 2);
    const uint32_t grid = std::min(a.n_wg + a.part.n_wg, round8(2u * (uint32_t)n_cus()));
    if (a.D == 64) hipLaunchKernelGGL((prefill_kernel<64, 1, false, false, PagedMixed8Args>), dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((prefill_kernel<128, 1, false, false, PagedMixed8Args>), dim3(grid), dim3(256), 0, st, a);
    const uint32_t tile_wgs = may_split(a) ? a.n_wg * merge_wgs(a) : 0, merge = tile_wgs + kRows * a.part.n_wg;
    if (a.D == 64) hipLaunchKernelGGL(paged_mixed8_merge_kernel<64>, dim3(merge), dim3(256), 0, st, a, tile_wgs);
    else hipLaunchKernelGGL(paged_mixed8_merge_kernel<128>, dim3(merge), dim3(256), 0, st, a, tile_wgs);
    return hipGetLastError();
}

}  // namespace yhip
