// paged_plan.hip -- block tables, slot map, positions and row offsets of one
// serving step, from the request lengths and the list of free blocks.
//
// With B positions per block, sequence i holds ceil(ctx_i / B) blocks and
// needs need_i = ceil((ctx_i + new_i) / B) - ceil(ctx_i / B) more (0 if its
// table row cannot hold them all); taken in
// order from the end of the free list, its t-th new block is
//   free[n_free - 1 - (need_0 + ... + need_{i-1}) - t].
// Row r of the step belongs to the sequence with cu_i <= r < cu_{i+1} (cu the
// prefix sums of new), position p = ctx_i + r - cu_i, slot
// table_i[p / B] * B + p % B.
//
// One launch and no communication between workgroups: every workgroup forms
// both prefix sums itself (a step has few sequences: 64 of them are one load
// and a scan), keeps them in LDS and resolves 256 rows, one per thread, by
// bisection.  The row that opens a block (p % B == 0) also writes its table
// entry, so the new entries need no pass of their own.  What bounds it is
// latency, not bytes: two dependent memory round trips (lengths, then the
// table or the free list) and the launch (64 sequences: 3.3 us of GPU time, 256
// with 16 chunks 4.3).
#include "common.hpp"
#include "internal.hpp"

namespace yhip {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kTop = 0x7fffffffu;

__device__ inline uint32_t blocks_of(uint32_t n, uint32_t shift) { return (n >> shift) + ((n & ((1u << shift) - 1u)) != 0); }

// One sequence's lengths as the plan takes them: a negative new length is
// zero rows, and one that cannot be served whatever comes before it (a negative
// length, more blocks than its table row has entries) counts no blocks.  So the
// blocks of those served are the free list's last: behind the first that is
// refused for blocks or rows none is served that needs any.
struct SeqLen {
    uint32_t ctx, rows, held, need;
    bool ok;
};
__device__ inline SeqLen seq_len(const PagedPlanArgs& a, uint32_t i)
{
    const int c = a.ctx[i], n = a.fresh[i];
    SeqLen s;
    s.ok = c >= 0 && n >= 0;
    s.ctx = c > 0 ? (uint32_t)c : 0u;
    s.rows = n > 0 ? (uint32_t)n : 0u;
    s.held = blocks_of(s.ctx, a.shift);
    const uint32_t all = blocks_of(s.ctx + s.rows, a.shift);
    s.ok = s.ok && all <= a.width;
    s.need = s.ok ? all - s.held : 0u;
    return s;
}

// A sequence is served as a whole or not at all.
__device__ inline bool served(const PagedPlanArgs& a, const SeqLen& s, uint64_t need_before, uint64_t rows_before,
                              uint32_t n_free)
{
    return s.ok && (s.need == 0 || need_before + s.need <= n_free) && rows_before + s.rows <= a.n_tok;
}

__device__ inline uint32_t clamp31(uint64_t x) { return x < kTop ? (uint32_t)x : kTop; }

__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PagedPlanArgs a)
{
    // prefix sums before each sequence, of rows and of blocks (they end at
    // 2^31 - 1: a sequence that starts there is not served)
    __shared__ uint32_t s_row[kPlanSeqs + 1], s_need[kPlanSeqs];
    __shared__ uint64_t s_wave[2][kThreads / 64];
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint32_t per = (a.n_seq + kThreads - 1) / kThreads;
    const uint32_t lo = min(t * per, a.n_seq), hi = min(lo + per, a.n_seq);
    const int nf = *a.n_free;
    const uint32_t n_free = nf < 0 ? 0u : min((uint32_t)nf, a.free_cap);

    uint64_t rows = 0, need = 0;
    for (uint32_t i = lo; i < hi; ++i) {
        const SeqLen s = seq_len(a, i);
        rows += s.rows;
        need += s.need;
    }
    uint64_t rsum = rows, nsum = need;  // inclusive over the wave
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t r = __shfl_up((unsigned long long)rsum, d), n = __shfl_up((unsigned long long)nsum, d);
        if (lane >= d) {
            rsum += r;
            nsum += n;
        }
    }
    if (lane == 63) {
        s_wave[0][wave] = rsum;
        s_wave[1][wave] = nsum;
    }
    __syncthreads();
    uint64_t rtot = 0, ntot = 0, rb = rsum - rows, nb = nsum - need;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64; ++w) {
        if (w < wave) {
            rb += s_wave[0][w];
            nb += s_wave[1][w];
        }
        rtot += s_wave[0][w];
        ntot += s_wave[1][w];
    }
    const bool first = blockIdx.x == 0;
    uint32_t missed = 0, used = 0;
    for (uint32_t i = lo; i < hi; ++i) {
        const SeqLen s = seq_len(a, i);
        s_row[i] = clamp31(rb);
        s_need[i] = clamp31(nb);
        if (first) {
            const bool ok = served(a, s, nb, rb, n_free);
            a.cu_new[i] = (int)clamp31(rb);
            a.kv_lens[i] = ok ? (int)min(s.ctx + s.rows, kTop) : 0;
            missed += !ok;
            used += ok ? s.need : 0u;
        }
        rb += s.rows;
        nb += s.need;
    }
    if (t == 0) s_row[a.n_seq] = clamp31(rtot);
    __syncthreads();
    if (first) {  // workgroup 0: the totals
#pragma unroll
        for (uint32_t d = 32; d > 0; d >>= 1) {
            missed += __shfl_xor(missed, d);
            used += __shfl_xor(used, d);
        }
        uint32_t* s_tot = reinterpret_cast<uint32_t*>(&s_wave[0][0]);
        if (lane == 0) {
            s_tot[wave] = missed;
            s_tot[8 + wave] = used;
        }
        __syncthreads();
        if (t == 0) {
            uint32_t m = 0, u = 0;
            for (uint32_t w = 0; w < kThreads / 64; ++w) {
                m += s_tot[w];
                u += s_tot[8 + w];
            }
            a.cu_new[a.n_seq] = (int)clamp31(rtot);
            a.counts[0] = (int)(n_free - u);
            a.counts[1] = (int)clamp31(rtot);
            a.counts[2] = (int)m;
            a.counts[3] = (int)(ntot > n_free ? clamp31(ntot - n_free) : 0u);
        }
    }

    const uint32_t r = blockIdx.x * kThreads + t;
    if (r >= a.n_tok) return;
    int slot = -1, pos = 0;
    if (r < s_row[a.n_seq]) {
        uint32_t b = 0, e = a.n_seq;  // s_row[b] <= r < s_row[e]
        while (e - b > 1) {
            const uint32_t m = (b + e) >> 1;
            if (s_row[m] <= r) b = m;
            else e = m;
        }
        const SeqLen s = seq_len(a, b);
        const uint32_t p = s.ctx + (r - s_row[b]);
        pos = (int)min(p, kTop);
        if (served(a, s, s_need[b], s_row[b], n_free)) {
            const uint32_t blk = p >> a.shift, off = p & ((1u << a.shift) - 1u);
            int* entry = a.table + (size_t)b * a.table_stride + blk;
            int id;
            if (blk < s.held) {
                id = *entry;
            } else {
                id = a.free_list[n_free - 1u - (s_need[b] + (blk - s.held))];
                if (off == 0) *entry = id;
            }
            // a negative entry, or a block whose slots pass 31 bits: no slot
            if (id >= 0 && (uint32_t)id <= (kTop >> a.shift)) slot = (int)(((uint32_t)id << a.shift) + off);
        }
    }
    a.slots[r] = slot;
    a.positions[r] = pos;
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t st)
{
    const uint32_t grid = a.n_tok ? (a.n_tok + kThreads - 1) / kThreads : 1u;
    hipLaunchKernelGGL(paged_plan_kernel, dim3(grid), dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace yhip
