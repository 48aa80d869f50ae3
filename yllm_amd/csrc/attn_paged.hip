// attn_paged.hip -- causal grouped-query attention of each sequence's new
// tokens over its pages of a KV pool.
//
// Token t of the n new ones of a sequence with L stored positions (its own
// included) sits at position p = L - n + t and attends to keys 0 .. p
// (engine.c:532-563 with the sequence's own start); a token at a negative
// position sees nothing and its row is zero.  Key j of a sequence is row
// j % block of page table[j / block].
//
// One wave per (row, query head): scores of 64 keys at a time, one per lane,
// the running maximum and sum of the softmax, then P.V with the lanes over
// the dimensions.  Everything is fp32.
#include "common.hpp"
#include "internal.hpp"

namespace yhip {
namespace {

__device__ inline float sigmoid_ref(float g) { return 1.0f / (1.0f + expf(-g)); }

template <int D>
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedAttnArgs a)
{
    __shared__ float s_q[4][D];
    __shared__ float s_p[4][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t row = blockIdx.x, h = blockIdx.y * 4u + wave;
    if (h >= a.n_heads) return;  // wave-uniform, and no workgroup barrier follows
    uint32_t lo = 0, hi = a.n_seq;  // cu[lo] <= row < cu[hi]
    if (row >= (uint32_t)max(a.cu_new[a.n_seq], 0)) return;  // rows behind the last sequence
    while (hi - lo > 1) {
        const uint32_t m = (lo + hi) >> 1;
        if ((uint32_t)max(a.cu_new[m], 0) <= row) lo = m;
        else hi = m;
    }
    const int len = max(0, min(a.kv_lens[lo], (int)a.max_len));
    const int pos = len - (a.cu_new[lo + 1] - a.cu_new[lo]) + ((int)row - a.cu_new[lo]);
    const int keys = min(pos + 1, len);
    const int* table = a.table + (size_t)lo * a.table_stride;
    const uint32_t kvh = h * a.n_kv / a.n_heads, mask = (1u << a.shift) - 1u;
    for (uint32_t d = lane; d < D; d += 64)
        s_q[wave][d] = load_as_f32(a.q, (size_t)row * a.q_stride + (size_t)h * D + d, a.q_dtype);
    __builtin_amdgcn_wave_barrier();
    constexpr int NO = D / 64;
    float m = -1e30f, l = 0.0f, o[NO] = {};
    for (int k0 = 0; k0 < keys; k0 += 64) {
        const int key = k0 + (int)lane;
        const uint32_t page0 = (uint32_t)table[(uint32_t)k0 >> a.shift];
        float s = -INFINITY;
        if (key < keys) {
            const uint32_t page = (uint32_t)table[(uint32_t)key >> a.shift];
            s = 0.0f;
            if (page < a.n_blocks) {
                const uint16_t* kr = a.kc + ((((size_t)page * a.n_kv + kvh) << a.shift) + ((uint32_t)key & mask)) * D;
                for (int d = 0; d < D; ++d) s = fmaf(f16_bits_to_f32(kr[d]), s_q[wave][d], s);
            }
            s *= a.c;
        }
        float mx = s;
        for (int i = 32; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor(mx, i));
        const float mn = fmaxf(m, mx), alpha = fast_exp2(m - mn);
        const float p = key < keys ? fast_exp2(s - mn) : 0.0f;
        m = mn;
        l = l * alpha + p;
        s_p[wave][lane] = p;
        __builtin_amdgcn_wave_barrier();
        const int nk = min(64, keys - k0);
        for (int r = 0; r < NO; ++r) {
            const uint32_t d = lane + 64u * r;
            float acc = o[r] * alpha;
            if (page0 < a.n_blocks) {  // a block is 64 positions or more: one page
                const uint16_t* vr = a.vc + ((((size_t)page0 * a.n_kv + kvh) << a.shift) + ((uint32_t)k0 & mask)) * D;
                for (int j = 0; j < nk; ++j)
                    acc = fmaf(s_p[wave][j], f16_bits_to_f32(vr[(size_t)(j / 32) * 32 * D + d * 32 + j % 32]), acc);
            }
            o[r] = acc;
        }
        __builtin_amdgcn_wave_barrier();
    }
    for (int i = 32; i > 0; i >>= 1) l += __shfl_xor(l, i);
    for (int r = 0; r < NO; ++r) {
        const uint32_t d = lane + 64u * r;
        float v = l > 0.0f || l != l ? o[r] / l : 0.0f;
        if (a.gate) v *= sigmoid_ref(a.gate[(size_t)row * a.gate_stride + (size_t)h * D + d]);
        const size_t at = (size_t)row * a.out_stride + (size_t)h * D + d;
        if (a.out_dtype == kF32) {
            reinterpret_cast<float*>(a.out)[at] = v;
        } else if (a.out_dtype == kF16) {
            reinterpret_cast<_Float16*>(a.out)[at] = (_Float16)v;
        } else {
            const uint32_t x = __builtin_bit_cast(uint32_t, v);
            reinterpret_cast<uint16_t*>(a.out)[at] =
                v != v ? (uint16_t)((x >> 16) | 0x40u) : (uint16_t)((x + 0x7fffu + ((x >> 16) & 1u)) >> 16);
        }
    }
}

}  // namespace

size_t paged_attn_workspace(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 0; }

hipError_t launch_paged_attn(const PagedAttnArgs& a, hipStream_t st)
{
    const dim3 grid(a.n_tok, (a.n_heads + 3) / 4);
    switch (a.D) {
    case 64: hipLaunchKernelGGL(paged_rows_kernel<64>, grid, dim3(256), 0, st, a); break;
    case 128: hipLaunchKernelGGL(paged_rows_kernel<128>, grid, dim3(256), 0, st, a); break;
    case 256: hipLaunchKernelGGL(paged_rows_kernel<256>, grid, dim3(256), 0, st, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace yhip
