// attn_prefill.hip -- launch plans of the prefill kernels (prefill_kernel.hpp)
// and the merge of the split mode's partial results.
#include "common.hpp"
#include "internal.hpp"
#include "prefill_kernel.hpp"

#include <math.h>
#include <stdlib.h>

namespace yhip {
namespace {

// One thread per (row, 4 output dimensions) of the split mode: the splits'
// (max, sum, O) partials of query b of head h are combined in the log2
// domain, then normalised, gated and stored.  Rows are b * n_heads + h, so a
// workgroup's output stores are contiguous; each round of 8 splits issues
// its loads together.
template <int D>
__global__ __launch_bounds__(256) void prefill_merge_kernel(PrefillArgs a)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t C4 = D / 4;
    constexpr uint32_t kRound = 8;
    const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
    const uint32_t row = idx / C4, c4 = idx % C4;
    if (row >= a.B * a.n_heads) return;
    const uint32_t b = row / a.n_heads, h = row % a.n_heads;
    const size_t split_stride = (size_t)a.n_heads * a.B;
    const size_t p0 = (size_t)h * a.B + b;
    const uint32_t d = 4 * c4;
    // the gate is read with the partials, not after them (a second memory
    // round trip); without a gate the output row stands in as a valid address
    const float* gp = a.gate ? a.gate + (size_t)b * a.gate_stride + (size_t)h * D + d
                             : reinterpret_cast<const float*>(a.out);
    f32x4 gt;
#pragma unroll
    for (int e = 0; e < 4; ++e) gt[e] = gp[e];
    float M = -1e30f, L = 0.0f;
    f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t s0 = 0; s0 < a.n_split; s0 += kRound) {
        f32x2 ml[kRound];
        f32x4 os[kRound];
#pragma unroll
        for (uint32_t r = 0; r < kRound; ++r) {
            if (s0 + r < a.n_split) {
                const size_t p = (s0 + r) * split_stride + p0;
                ml[r] = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * p);
                os[r] = *reinterpret_cast<const f32x4*>(a.part_o + p * D + 4 * c4);
            } else {
                ml[r] = f32x2{-1e30f, 0.0f};
                os[r] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
        float mr = M;
#pragma unroll
        for (uint32_t r = 0; r < kRound; ++r) mr = fmaxf(mr, ml[r][0]);
        const float co = fast_exp2(M - mr);
        L *= co;
        O *= co;
#pragma unroll
        for (uint32_t r = 0; r < kRound; ++r) {
            const float c = fast_exp2(ml[r][0] - mr);
            L += ml[r][1] * c;
            O += os[r] * c;
        }
        M = mr;
    }
    // every query has key 0 in split 0, so L > 0
    f32x4 v = O * (1.0f / L);
    if (a.gate) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= sigmoid_ref(gt[e]);
    }
    store_out4(a.out, (size_t)b * a.out_stride + (size_t)h * D + d, a.out_dtype, v);
}

}  // namespace

int n_cus()
{
    static const int n_cu = [] {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) != hipSuccess ||
            hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
            n = 256;
        return n;
    }();
    return n_cu;
}

namespace {

// threads of a prefill workgroup: 4 waves per key group, 8 in pair mode
constexpr int prefill_threads(int D, int NG) { return 256 * NG * (D > 128 ? 2 : 1); }

// the XCD mapping needs whole kv groups per XCD group and an equal share
// per XCD (measured 470 -> 478 TFLOP/s at 2048 tokens x 28 heads)
uint32_t xcd_mapped(const PrefillArgs& a)
{
    static const int env = [] {
        const char* e = getenv("YHIP_PREFILL_XCD");
        return e ? atoi(e) : 1;
    }();
    const uint32_t nqb = (a.B + BM - 1) / BM;
    return env != 0 && a.n_kv <= 8 && 8 % a.n_kv == 0 && a.n_heads % a.n_kv == 0 &&
           ((uint64_t)nqb * (a.n_heads / a.n_kv)) % (8 / a.n_kv) == 0;
}

// YHIP_PREFILL_PERSIST=0/1 forces resident workgroups off / on, YHIP_PREFILL_NG
// =1/2 the key groups of head_dim 64 and 128, for comparisons (-1, 0: unset).
int forced_persist()
{
    static const int env = [] {
        const char* e = getenv("YHIP_PREFILL_PERSIST");
        return e ? atoi(e) : -1;
    }();
    return env;
}
int forced_groups()
{
    static const int env = [] {
        const char* e = getenv("YHIP_PREFILL_NG");
        const int n = e ? atoi(e) : 0;
        return n == 1 || n == 2 ? n : 0;
    }();
    return env;
}

template <int D, int NG, bool QS>
hipError_t launch_prefill_d(PrefillArgs a, hipStream_t st)
{
    a.xcd_map = xcd_mapped(a);
    const uint32_t items = (a.B + BM - 1) / BM * a.n_heads;
    // resident workgroups: one round of the grid fills every slot once
    static const int per_cu = [] {
        int n = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, prefill_kernel<D, NG, false, QS>, prefill_threads(D, NG),
                                                         0) != hipSuccess ||
            n < 1)
            n = 1;
        return n;
    }();
    // Resident workgroups walking the item list pay off with one 8-wave
    // workgroup per CU (two key groups), where nothing else on the CU covers
    // a workgroup's start and end (2048 tokens x 28 heads: 57.1 -> 55.7 us);
    // with two 4-wave workgroups per CU the hardware's own dispatch of the
    // next workgroup already overlaps them and is about 1 % faster (8192
    // tokens).
    const int persist = forced_persist();
    uint32_t grid = items;
    if (persist > 0 || (persist < 0 && prefill_threads(D, NG) > 256)) {
        const uint64_t slots = (uint64_t)per_cu * (uint64_t)n_cus();
        if (slots < grid) grid = (uint32_t)slots;
        if (a.xcd_map) grid = grid / 8u * 8u;  // whole XCD groups (items are a multiple of 8)
        if (grid == 0) grid = items;
    }
    hipLaunchKernelGGL((prefill_kernel<D, NG, false, QS>), dim3(grid), dim3(prefill_threads(D, NG)), 0, st, a);
    return hipGetLastError();
}

// The split mode at head_dim 256 with 16-bit queries: walks of up to four
// 32-key tiles (seven in one range; eight where packed rows do not fill a
// workgroup, so that idle waves leave the other kernel's shorter steps
// uncovered) stay with prefill_kernel, whose first scores need half the bytes
// and MFMAs and which walks an odd tile alone (16 / 2 heads, us with it / with
// prefill_halves_kernel: 64 tokens at 0 12.0 / 14.2, 33 at 100 15.6 / 18.5, four
// tiles each at 1984 23.0 / 23.2; 24 / 4 heads in one range of five tiles, 133
// at 11 15.8 / 16.9; 8 / 8 heads, 33 tokens at 4000 in eight 18.4 / 19.8); longer
// ones are shorter in the other (64 tokens at 4000 in eight 27.6 / 26.1, at 16000
// 54 / 45, 1000 at 4000 215 / 98; 24 / 4 heads in one range of eight, 133 at 100
// 19.2 / 18.4).  n_split is set.
bool split_halves(const PrefillArgs& a)
{
    const uint32_t most = a.pack && a.gmax * a.B < (uint32_t)BM ? 8u : a.n_split == 1 ? 7u : 4u;
    return a.D > 128 && a.q_dtype != kF32 && a.split_tiles > most;
}

// one workgroup per CU walking the items in snake order
hipError_t launch_prefill_halves(PrefillArgs a, hipStream_t st)
{
    a.xcd_map = xcd_mapped(a);
    const uint32_t items = (a.B + BM - 1) / BM * a.n_heads;
    uint32_t grid = items < (uint32_t)n_cus() || forced_persist() == 0 ? items : (uint32_t)n_cus();
    if (a.xcd_map && grid >= 8u) grid = grid / 8u * 8u;  // whole XCD groups (items are a multiple of 8)
    hipLaunchKernelGGL((prefill_halves_kernel<256, false>), dim3(grid), dim3(512), 0, st, a);
    return hipGetLastError();
}

// The split mode's order (split_item) and grid: whole tile groups to XCDs
// where the fullest XCD still has a CU for each of its items.
uint32_t split_grid(PrefillArgs& a)
{
    const uint32_t ipg = a.n_rb * (a.pack ? 1u : a.gmax), groups = a.n_kv * a.n_split;
    const uint32_t most = (groups + 7u) / 8u * ipg;
    a.xcd_map = groups % 8u == 0 || most <= (uint32_t)n_cus() / 8u;
    return a.xcd_map ? most * 8u : (groups * ipg + 7u) / 8u * 8u;
}

template <int D, bool QS>
hipError_t launch_prefill_split_d(PrefillArgs a, hipStream_t st)
{
    const uint32_t grid = split_grid(a);
    bool halves = false;
    if constexpr (D > 128 && !QS) {
        halves = split_halves(a);
        if (halves) hipLaunchKernelGGL((prefill_halves_kernel<D, true>), dim3(grid), dim3(512), 0, st, a);
    }
    bool two = false;
    if constexpr (D <= 128 && QS) {
        // fp32 queries: two key groups from four tiles per split on (28 / 4 heads of 128, us with one / two: 64
        // tokens at 0 10.2 / 12.0, at 1000 20.3 / 19.6, at 16000 47 / 40), six where the workgroups go round twice
        // (32 / 32 heads, 64 tokens at 4000 in four 36.1 / 38.3); at d 64, where a CU holds two workgroups of one
        // group, only while the grid leaves it at one (400 at 2000 22.4 / 26.7)
        two = forced_groups() ? forced_groups() == 2
                              : grid <= (uint32_t)n_cus() ? a.split_tiles >= 4 : D == 128 && a.split_tiles >= 6;
        if (two) hipLaunchKernelGGL((prefill_kernel<D, 2, true, QS>), dim3(grid), dim3(prefill_threads(D, 2)), 0, st, a);
    }
    if (!halves && !two)
        hipLaunchKernelGGL((prefill_kernel<D, 1, true, QS>), dim3(grid), dim3(prefill_threads(D, 1)), 0, st, a);
    if (a.n_split > 1) {
        const uint64_t threads = (uint64_t)a.B * a.n_heads * (D / 4);
        hipLaunchKernelGGL(prefill_merge_kernel<D>, dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

// Key groups per workgroup.  Two groups halve the longest chain of tiles a
// wave walks, which is what bounds a grid that fills the machine only once
// (2048 tokens x 28 heads: 448 workgroups on 256 CUs, 420 -> 479 TFLOP/s);
// with many workgroups per CU two independent 4-wave workgroups hide latency
// better than one 8-wave workgroup under one barrier (8192 tokens: 888 vs
// 790 TFLOP/s).  Two groups need the LDS of two groups' tiles (head_dim <=
// 128).
int prefill_groups(const PrefillArgs& a)
{
    const int n_cu = n_cus();
    if (a.D > 128) return 1;
    if (forced_groups()) return forced_groups();
    const uint64_t wgs = (uint64_t)((a.B + BM - 1) / BM) * a.n_heads;
    // fp32 queries: at d 128 always two (one group alone, 352 registers, is one
    // wave per SIMD: 28 / 4 heads, 2048 tokens 80 -> 68 us, 6000 478 -> 410); at
    // d 64 one workgroup per CU or less gains nothing from it (14 / 2 heads, 1500
    // tokens 29.7 / 30.3, 3000 59 -> 44, 6000 130 either way), nor do heads of
    // few query blocks, which two workgroups per CU balance better (64 / 8 heads,
    // 635 tokens at 500 27.9 -> 30.6, 800 19.8 -> 22.5; 32 / 8, 1147 25.3 -> 21.3)
    if (a.q_dtype == kF32) {
        const bool pays = wgs > (uint64_t)n_cu && wgs <= 2 * (uint64_t)n_cu && a.B > 8u * (uint32_t)BM;
        return a.D == 128 || pays ? 2 : 1;
    }
    return wgs <= 2 * (uint64_t)n_cu ? 2 : 1;
}

}  // namespace

namespace {

size_t align256p(size_t x) { return (x + 255) / 256 * 256; }

// Split-mode tunables (YHIP_PREFILL_SPLIT=0 turns the mode off; the others
// bound the split count and the tiles per split, for sweeps).
struct SplitTune {
    int on;
    uint32_t max_split, min_tiles;
};
const SplitTune& split_tune()
{
    static const SplitTune t = [] {
        SplitTune r{1, 16, 4};
        if (const char* e = getenv("YHIP_PREFILL_SPLIT")) r.on = atoi(e) != 0;
        if (const char* e = getenv("YHIP_PREFILL_MAXSPLIT")) r.max_split = (uint32_t)(atoi(e) > 0 ? atoi(e) : 1);
        if (const char* e = getenv("YHIP_PREFILL_MINTILES")) r.min_tiles = (uint32_t)(atoi(e) > 0 ? atoi(e) : 1);
        return r;
    }();
    return t;
}

size_t split_bytes(uint32_t n_split, uint32_t B, uint32_t n_heads, uint32_t D)
{
    if (n_split <= 1) return 0;
    const size_t rows = (size_t)n_split * n_heads * B;
    return align256p(rows * 2 * sizeof(float)) + rows * D * sizeof(float);
}

// Items of a split-mode launch before splitting, and the workgroups that
// fill the GPU once.
void split_shape(uint32_t B, uint32_t n_heads, uint32_t n_kv, uint32_t D, uint32_t& pack, uint32_t& n_rb,
                 uint32_t& gmax, uint64_t& base, uint64_t& target)
{
    gmax = (n_heads + n_kv - 1) / n_kv;
    pack = B < (uint32_t)BM;
    n_rb = pack ? (gmax * B + BM - 1) / BM : (B + BM - 1) / BM;
    base = (uint64_t)n_kv * n_rb * (pack ? 1u : gmax);
    target = (uint64_t)(D <= 128 ? 2 : 1) * (uint64_t)n_cus();  // resident workgroups per CU
}

}  // namespace

size_t prefill_plan(PrefillArgs& a)
{
    a.split_mode = a.pack = 0;
    a.n_split = 1;
    a.split_tiles = 0;
    a.n_rb = 0;
    a.gmax = 0;
    const SplitTune& t = split_tune();
    // The plain mode, (query block, head) items, fills the GPU when there
    // are at least as many items as CUs (prompts of a few hundred tokens and
    // up).  Fewer items -- the engine's 64-token chunks over a long prefix
    // -- would leave most CUs idle while each walks the whole prefix: the
    // split mode packs a kv head's query heads into full 128-row items and
    // splits the keys so that the launch fills the GPU.
    if (!t.on || (uint64_t)((a.B + BM - 1) / BM) * a.n_heads >= (uint64_t)n_cus()) return 0;
    uint64_t base, target;
    split_shape(a.B, a.n_heads, a.n_kv, a.D, a.pack, a.n_rb, a.gmax, base, target);
    a.split_mode = 1;
    const uint32_t ntiles = (a.pos_start + a.B - 1) / bn_of((int)a.D) + 1;
    uint64_t most = target / base;
    if (most > t.max_split) most = t.max_split;
    const uint32_t by_tiles = (ntiles + t.min_tiles - 1) / t.min_tiles;
    if (most > by_tiles) most = by_tiles;
    // Of up to `most` splits, the number with the least cost: the walk of the
    // longest split (us per 64 keys; past one workgroup per CU half again as
    // long where a CU holds two, twice where it holds one: fp32 queries at
    // head_dim 128) and, from two on, the merge launch and the partials written
    // and read (1.4 us, 5 TB/s; 28 / 4 heads of 128, f16: 1000 tokens 25.6 us
    // unsplit, 34.4 in two; f32 38 and 55, 400 tokens at 2000 49 in four, 42 in
    // two; 64 tokens at 1984 16 us in eight; 2 tokens at 300 11.8 unsplit, 9.7
    // in two; 16 / 2 heads of 256, f32: 256 tokens at 512 30.1 in four, 28.0 in six).
    // An unsplit launch applies the gate in its few workgroups' epilogues (2.9, 5.7
    // and 5.4 us at head_dim 64, 128 and 256), a split one in the merge's many
    // (0.2 to 2): what fits the 16-bit walks beside the merge's estimate is 1.3, 2.6
    // and 3 us (f16, gated, unsplit / in two: 24 / 4 heads of 256, 33 tokens at 100
    // 22.6 / 15.5; 8 / 8, 133 at 11 22.0 / 16.3; 28 / 4 of 128, 192 at 100 18.3 /
    // 14.6), for fp32 queries the same 3 at 256 and nothing below, where the walk
    // is estimated long.
    const bool f32q = a.q_dtype == kF32;
    const float per64 = !f32q ? 0.35f + (float)a.D / 160.0f : a.D > 128 ? 3.5f : 1.6f * (0.35f + (float)a.D / 160.0f);
    const float round2 = f32q && a.D == 128 ? 2.0f : 1.5f;
    const float rows_us = (float)a.n_heads * a.B * a.D * 8.0f / 5.0e6f;
    const float gate_us = !a.gate || (f32q && a.D <= 128) ? 0.0f : fminf((float)a.D / 50.0f, 3.0f);
    uint64_t S = 1;
    float best = 0.0f;
    for (uint64_t n = 1; n <= most; ++n) {
        const float walk = (float)((ntiles + n - 1) / n * bn_of((int)a.D)) / 64.0f * per64;
        const float cost = walk * (base * n > (uint64_t)n_cus() ? round2 : 1.0f) + (n > 1 ? 1.4f + rows_us * n : gate_us);
        if (n == 1 || cost < best) {
            best = cost;
            S = n;
        }
    }
    // An unsplit launch of whole query blocks over 512 keys or more runs the
    // plain mode (two key groups for 16-bit queries up to d 128): 1000 tokens
    // 24.9 against 25.6 us, 14 / 2 heads of 64 16.6 against 17.4.
    if (S == 1 && !a.pack && ntiles * bn_of((int)a.D) >= 512) {
        a.split_mode = 0;
        return 0;
    }
    a.split_tiles = (ntiles + (uint32_t)S - 1) / (uint32_t)S;
    a.n_split = (ntiles + a.split_tiles - 1) / a.split_tiles;
    // prefill_halves_kernel walks pairs of 32-key tiles (of two ranges or more of five tiles at least, so two remain)
    if (split_halves(a)) {
        a.split_tiles += a.split_tiles & 1u;
        a.n_split = (ntiles + a.split_tiles - 1) / a.split_tiles;
    }
    return split_bytes(a.n_split, a.B, a.n_heads, a.D);
}

size_t prefill_workspace_bound(uint32_t B, uint32_t max_end, uint32_t n_heads, uint32_t n_kv, uint32_t D)
{
    // the plan for any pos_start <= max_end - B: its split count is at most
    // min(target/base, max_split, ceil(tiles/min_tiles)) with the most tiles
    const SplitTune& t = split_tune();
    if (!t.on || B == 0 || n_kv == 0 || max_end < B || (uint64_t)((B + BM - 1) / BM) * n_heads >= (uint64_t)n_cus())
        return 0;
    uint32_t pack, n_rb, gmax;
    uint64_t base, target;
    split_shape(B, n_heads, n_kv, D, pack, n_rb, gmax, base, target);
    const uint32_t ntiles = (max_end - 1) / bn_of((int)D) + 1;
    uint64_t S = target / base;
    if (S > t.max_split) S = t.max_split;
    const uint32_t by_tiles = (ntiles + t.min_tiles - 1) / t.min_tiles;
    if (S > by_tiles) S = by_tiles;
    return split_bytes((uint32_t)(S < 1 ? 1 : S), B, n_heads, D);
}

uint32_t prefill_tile_keys(uint32_t D) { return (uint32_t)bn_of((int)D); }

void prefill_bind_workspace(PrefillArgs& a, void* workspace)
{
    if (a.n_split <= 1 || !workspace) {
        a.part_ml = a.part_o = nullptr;
        return;
    }
    char* p = reinterpret_cast<char*>(workspace);
    a.part_ml = reinterpret_cast<float*>(p);
    a.part_o = reinterpret_cast<float*>(p + align256p((size_t)a.n_split * a.n_heads * a.B * 2 * sizeof(float)));
}

hipError_t launch_prefill(const PrefillArgs& a, hipStream_t st)
{
    // fp32 queries keep fp32-level scores (hi + lo parts)
    const bool qs = a.q_dtype == kF32;
    if (a.split_mode) {
        switch (a.D) {
        case 64: return qs ? launch_prefill_split_d<64, true>(a, st) : launch_prefill_split_d<64, false>(a, st);
        case 128: return qs ? launch_prefill_split_d<128, true>(a, st) : launch_prefill_split_d<128, false>(a, st);
        case 256: return qs ? launch_prefill_split_d<256, true>(a, st) : launch_prefill_split_d<256, false>(a, st);
        default: return hipErrorInvalidValue;
        }
    }
    const int ng = prefill_groups(a);
    switch (a.D) {
    case 64:
        return qs ? (ng == 2 ? launch_prefill_d<64, 2, true>(a, st) : launch_prefill_d<64, 1, true>(a, st))
                  : ng == 2 ? launch_prefill_d<64, 2, false>(a, st) : launch_prefill_d<64, 1, false>(a, st);
    case 128:
        return qs ? (ng == 2 ? launch_prefill_d<128, 2, true>(a, st) : launch_prefill_d<128, 1, true>(a, st))
                  : ng == 2 ? launch_prefill_d<128, 2, false>(a, st) : launch_prefill_d<128, 1, false>(a, st);
    case 256: return qs ? launch_prefill_d<256, 1, true>(a, st) : launch_prefill_halves(a, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace yhip
