// paged_decode8.hip -- the launches of attention over the 8-bit KV pool: of
// sequences with few new tokens (paged_decode8.hpp), of prompts and chunks (tiles,
// attn_paged.hip) and of both at once.
#include "common.hpp"
#include "internal.hpp"
#include "paged_decode8.hpp"

#include <algorithm>

namespace yhip {
namespace {

template <int D, bool PREC, int POL>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void paged_decode8_kernel(PagedAttn8Args args)
{
    __shared__ __attribute__((aligned(16))) float s_lds[4][kDecode8Lds<D, PREC>];
    decode8_pieces<D, PREC, POL>(args, blockIdx.x, args.n_wg, [&](int w) { return &s_lds[w][0]; });
}

template <int D>
__global__ __launch_bounds__(256) void paged_decode8_merge_kernel(PagedAttn8Args a)
{
    decode8_merge<D>(a, blockIdx.x, blockIdx.y);
}

// Cutting an item costs two partial results and the merge's launch.  Where no
// item's K and V take more than this many bytes per kv head, none is cut: whole
// and cut, us for one sequence: 14 / 2 heads of 64, 2048 keys 10.4 and 11.0, 2560
// 12.0 and 11.1; 28 / 4 of 128, 1024 keys 11.8 and 13.2, 1280 13.2 and 13.6, 1792
// 15.9 and 13.2; 16 / 2 of 256, 768 keys 15.9 and 16.6, 1024 18.7 and 18.1.
constexpr uint32_t whole_bytes(uint32_t D) { return (D == 64 ? 256 : D == 128 ? 320 : 384) * 1024; }
// Up to this many where there are items for half the GPU, but no more than it
// holds at once: 64 sequences of 2048 keys, 28 / 4 heads of 128, 24.8 whole, 37.6
// cut; of 4096, 14 / 2 of 64, 18.3 and 21.4; 128 of 1024, 16 / 2 of 256, 27.1 and
// 30.8.  (16 sequences of 2048 keys: 18.9 and 20.0, of 4096 of 64 18.0 and 13.1.)
constexpr uint32_t kWholeMany = 512 * 1024, kManyItems = 128;
// On the line, beside longer ones, fewer: there the merge comes anyway and items
// that are not cut make chunks uneven (64 sequences of 1k to 32k keys, 14 / 2
// heads of 64: 35.4 us, 38.3 with 160 KB; 200 of up to 3000 21.3 and 22.5).
constexpr uint32_t kSnapBytes = 64 * 1024;

uint32_t units_of_bytes(uint32_t bytes, uint32_t D) { return bytes / (2 * D * kUnit8); }

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Sequences of up to this many rows are walked here, in blocks of 16, the others
// in tiles of 128 rows: 32 sequences of 4000 keys, 28 / 4 heads of 128, 3 tokens
// (21 rows) 46.3 us, in tiles 53.8; 14 / 2 of 64, 4 tokens 19.2 and 31.7; 16 / 2 of
// 256, 4 tokens 51.5 and 63; 5 tokens of 28 / 4 (35 rows) 75 and 60.  (64 sequences
// of up to 20000 keys, 3 tokens of 28 / 4: 106 and 98: the second block reads K and
// V again.)
constexpr uint32_t kFewRows = 32;

// row blocks of a sequence at most
uint32_t row_blocks(uint32_t max_new, uint32_t n_heads, uint32_t n_kv)
{
    const uint64_t rows = (uint64_t)((n_heads + n_kv - 1) / n_kv) * max_new;
    return (uint32_t)((std::min(rows, (uint64_t)kFewRows) + kRows - 1) / kRows);
}

uint32_t decode8_slots(uint32_t D) { return (D <= 128 ? 2u : 1u) * (uint32_t)n_cus(); }

// Chunks of a line: what the GPU holds at once, or all that the bounds can fill
uint32_t line8_wgs(uint32_t n_seq, uint32_t max_new, uint32_t max_len, uint32_t n_heads, uint32_t n_kv, uint32_t D)
{
    const uint32_t units = (max_len + kUnit8 - 1) / kUnit8;
    const uint64_t most = (uint64_t)n_seq * row_blocks(max_new, n_heads, n_kv) * n_kv * (units + kItem8Units);
    const uint64_t full = decode8_slots(D);
    return (uint32_t)(((most < full ? most : full) + 7) / 8 * 8);
}

// whether no item is cut, whatever their number
bool short_items(uint32_t max_len, uint32_t D) { return (max_len + kUnit8 - 1) / kUnit8 <= units_of_bytes(whole_bytes(D), D); }

// Chunks of a launch of their own; 0: a workgroup for each item.  (The workspace
// goes by the line all the same: one that serves a call serves smaller ones.)
uint32_t decode8_wgs(uint32_t n_seq, uint32_t max_new, uint32_t max_len, uint32_t n_heads, uint32_t n_kv, uint32_t D)
{
    const uint64_t items = (uint64_t)n_seq * row_blocks(max_new, n_heads, n_kv) * n_kv;
    if (short_items(max_len, D)) return 0;
    if (items >= kManyItems && items <= decode8_slots(D) && (max_len + kUnit8 - 1) / kUnit8 <= units_of_bytes(kWholeMany, D)) return 0;
    return line8_wgs(n_seq, max_new, max_len, n_heads, n_kv, D);
}

size_t decode8_bytes(uint32_t wgs, uint32_t D)
{
    if (wgs == 0) return 0;
    const size_t rows = (size_t)2 * wgs * kRows;
    return align256((size_t)wgs * sizeof(PagedDesc)) + align256(rows * 2 * sizeof(float)) + rows * D * sizeof(float);
}

template <int D, bool PREC>
void launch_decode8_pieces(const PagedAttn8Args& a, uint32_t grid, bool stream, hipStream_t st)
{
    if (stream)
        hipLaunchKernelGGL((paged_decode8_kernel<D, PREC, 2>), dim3(grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((paged_decode8_kernel<D, PREC, 0>), dim3(grid), dim3(256), 0, st, a);
}

// what the launcher sets, for a line of n_wg chunks
void set_line8(PagedAttn8Args& a, uint32_t n_wg)
{
    a.n_wg = n_wg;
    a.snap_units = units_of_bytes(kSnapBytes, a.D);
    a.min_units = 1 + kItem8Units;
    char* p = reinterpret_cast<char*>(a.ws);
    a.desc = p;
    p += align256((size_t)a.n_wg * sizeof(PagedDesc));
    a.part_ml = reinterpret_cast<float*>(p);
    a.part_o = reinterpret_cast<float*>(p + align256((size_t)2 * a.n_wg * kRows * 2 * sizeof(float)));
}

hipError_t launch_decode8(const PagedAttn8Args& in, hipStream_t st)
{
    PagedAttn8Args a = in;
    set_line8(a, decode8_wgs(a.n_seq, a.max_new, a.max_len, a.n_heads, a.n_kv, a.D));
    const uint32_t nb = row_blocks(a.max_new, a.n_heads, a.n_kv);
    const uint32_t grid = a.n_wg ? a.n_wg : a.n_seq * a.n_kv * nb;
    // non-temporal loads where the batch reads more than the caches keep (an upper bound), and once
    const bool stream = nb == 1 && (uint64_t)a.n_seq * a.n_kv * a.max_len * a.D * 2u >= (32ull << 20);
    const bool prec = a.q_dtype == kF32;
    switch (a.D) {
    case 64: prec ? launch_decode8_pieces<64, true>(a, grid, stream, st) : launch_decode8_pieces<64, false>(a, grid, stream, st); break;
    case 128: prec ? launch_decode8_pieces<128, true>(a, grid, stream, st) : launch_decode8_pieces<128, false>(a, grid, stream, st); break;
    case 256: prec ? launch_decode8_pieces<256, true>(a, grid, stream, st) : launch_decode8_pieces<256, false>(a, grid, stream, st); break;
    default: return hipErrorInvalidValue;
    }
    if (a.n_wg) {
        const dim3 merge(a.n_wg, std::min((uint64_t)kRows, (uint64_t)a.gmax * a.max_new));
        switch (a.D) {
        case 64: hipLaunchKernelGGL(paged_decode8_merge_kernel<64>, merge, dim3(256), 0, st, a); break;
        case 128: hipLaunchKernelGGL(paged_decode8_merge_kernel<128>, merge, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL(paged_decode8_merge_kernel<256>, merge, dim3(256), 0, st, a); break;
        }
    }
    return hipGetLastError();
}

// whether every sequence within the bounds is few
bool all_few(uint32_t n_heads, uint32_t n_kv, uint32_t max_new)
{
    return (uint64_t)((n_heads + n_kv - 1) / n_kv) * max_new <= kFewRows;
}

}  // namespace

// (both parts have a place of their own)
size_t paged_attn8_workspace(uint32_t n_tok, uint32_t n_seq, uint32_t max_new, uint32_t max_len, uint32_t n_heads,
                             uint32_t n_kv, uint32_t D)
{
    const size_t few = align256(decode8_bytes(line8_wgs(n_seq, max_new, max_len, n_heads, n_kv, D), D));
    if (all_few(n_heads, n_kv, max_new)) return short_items(max_len, D) ? 0 : few;
    return few + paged_tiles8_workspace(n_tok, n_seq, max_len, n_heads, n_kv, D);
}

// Sequences with few rows go to the decode kernel, the others to the tiles; which
// are which is known on the device only.  One launch walks both lines where their
// workgroups are alike, two to a CU (28 / 4 heads of 128, 28 decode tokens and
// four chunks of 512: 86 us; one line after the other, each with its merge, 103;
// 32 / 8, 63 of up to 32768 and a chunk of 256: 257 and 280; 14 / 2 heads of 64: 45
// and 56); elsewhere the lines follow each other (28 decode tokens and four chunks
// of 512, 28 / 4 heads of 128, fp32 queries 141; 16 / 2 of 256 with a gate 131, fp32
// 178).  One sequence (a prompt's chunk) is the tiles' whatever it brings.
hipError_t launch_paged_attn8(const PagedAttn8Args& in, hipStream_t st)
{
    PagedAttn8Args a = in;
    a.gmax = (a.n_heads + a.n_kv - 1) / a.n_kv;
    a.few = kFewRows;
    if (all_few(a.n_heads, a.n_kv, a.max_new)) return launch_decode8(a, st);
    if (a.n_seq == 1) {
        a.few = 0;
        return launch_paged_tiles8(a, st);
    }
    PagedAttn8Args few = a;
    set_line8(few, line8_wgs(a.n_seq, a.max_new, a.max_len, a.n_heads, a.n_kv, a.D));
    a.ws = reinterpret_cast<char*>(a.ws) + align256(decode8_bytes(few.n_wg, a.D));
    if (a.D <= 128 && a.q_dtype != kF32) return launch_paged_mixed8(a, few, st);
    if (const hipError_t e = launch_decode8(few, st)) return e;
    return launch_paged_tiles8(a, st);
}

}  // namespace yhip
