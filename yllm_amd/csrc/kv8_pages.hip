// kv8_pages.hip -- pages of the f16 KV pool into the 8-bit one (kv8.hpp) and back.
//
// A workgroup takes 64 positions of one kv head of one page: K rows of D and two
// V tiles of 32 positions on the f16 side, 64 rows and one V tile of 64 on the
// other.  A K row is D / 8 lanes, its largest magnitude a few DPP moves.  V is
// d-major on both sides: a thread holds eight positions of D / 32 dimensions, so
// a position's largest magnitude is the maximum over a thread's dimensions, over
// the lanes eight apart and over the four waves (LDS).  Bound by HBM: every byte
// is read and written once.
//
// Measured: 128 pages of 64, 8 kv heads of 128, into 8 bits: 12.2 us, 4.1 TB/s (the
// bytes alone 9.8 at a large copy's rate: one round of 1024 workgroups, whose loads
// all go out before the first conversion), back 11.1 us; 1024 pages 83 us in and 81
// back, 4.9 and 5.0 TB/s; three pages of 2 of 256 back: 3.2 us.
#include "common.hpp"
#include "internal.hpp"
#include "kv8.hpp"

namespace yhip {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct Pair {
    size_t f16, kv8;  // first element (code) of the tile's 64 positions in the pools
    size_t scale;
    bool ok;
};

// workgroup b's tile; not ok where the source or destination page is outside its pool
template <bool FROM>
__device__ inline Pair pair_of(const Kv8PagesArgs& a, uint32_t D)
{
    const uint32_t tiles = a.block / 64u, tile = blockIdx.x % tiles, w = blockIdx.x / tiles, h = w % a.n_kv, i = w / a.n_kv;
    const uint32_t s = (uint32_t)a.src[i], d = (uint32_t)a.dst[i], pf = FROM ? s : d, p8 = FROM ? d : s;
    const size_t f = ((size_t)pf * a.n_kv + h) * a.block + tile * 64u, e = ((size_t)p8 * a.n_kv + h) * a.block + tile * 64u;
    return Pair{f * D, e * D, e, pf < a.n_f16 && p8 < a.n_8};
}

// the largest magnitude bits over each aligned group of N lanes (a K row), N = 8, 16, 32
template <int N>
__device__ inline uint32_t row_max(uint32_t x)
{
#pragma unroll
    for (int m = 1; m < N; m <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, m));
    return x;
}

template <int D>
__global__ __launch_bounds__(256) void kv8_from_pages_kernel(Kv8PagesArgs a)
{
    constexpr int LPH = D / 8, RPP = 256 / LPH, NK = 64 / RPP, NV = D / 32;
    __shared__ uint32_t top[4][64];
    __shared__ float inv[64];
    const Pair p = pair_of<true>(a, D);
    if (!p.ok) return;  // workgroup-uniform
    const int t = threadIdx.x, wave = t >> 6;
    const f16x8* const kin = reinterpret_cast<const f16x8*>(a.kc + p.f16);
    const int c = t & 7;  // positions 8 c .. of dimensions t / 8 + 32 i
    const f16x8* const vin = reinterpret_cast<const f16x8*>(a.vc + p.f16 + (c >> 2) * (D * 32)) + (c & 3);
    f16x8 k[NK], v[NV];
#pragma unroll
    for (int i = 0; i < NK; ++i) k[i] = __builtin_nontemporal_load(kin + t + 256 * i);
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = __builtin_nontemporal_load(vin + (t / 8 + 32 * i) * 4);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        f32x4 x[2];
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e >> 2][e & 3] = (float)k[i][e];
            m = max(m, finite_mag(x[e >> 2][e & 3]));
        }
        const int ex = kv8_exponent(row_max<LPH>(m));
        const float s = kv8_inverse(ex);
        const u32x2 w = {kv8_codes(x[0], s), kv8_codes(x[1], s)};
        reinterpret_cast<u32x2*>(a.k8 + p.kv8)[t + 256 * i] = w;
        if (t % LPH == 0) a.ks[p.scale + t / LPH + RPP * i] = kv8_scale_byte(ex);
    }
    uint32_t m[8] = {};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) m[e] = max(m[e], finite_mag((float)v[i][e]));
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int x = 8; x < 64; x <<= 1) m[e] = max(m[e], (uint32_t)__shfl_xor((int)m[e], x));
    if ((t & 63) < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) top[wave][8 * c + e] = m[e];
    }
    __syncthreads();
    if (t < 64) {
        const int ex = kv8_exponent(max(max(top[0][t], top[1][t]), max(top[2][t], top[3][t])));
        inv[t] = kv8_inverse(ex);
        a.vs[p.scale + t] = kv8_scale_byte(ex);
    }
    __syncthreads();
    const f32x4 s0 = *reinterpret_cast<const f32x4*>(&inv[8 * c]), s1 = *reinterpret_cast<const f32x4*>(&inv[8 * c + 4]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        f32x4 x[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = (float)v[i][e];
        const u32x2 w = {kv8_codes(x[0], s0), kv8_codes(x[1], s1)};
        reinterpret_cast<u32x2*>(a.v8 + p.kv8)[(t / 8 + 32 * i) * 8 + c] = w;
    }
}

template <int D>
__global__ __launch_bounds__(256) void kv8_to_pages_kernel(Kv8PagesArgs a)
{
    constexpr int LPH = D / 8, RPP = 256 / LPH, NK = 64 / RPP, NV = D / 32;
    const Pair p = pair_of<false>(a, D);
    if (!p.ok) return;
    const int t = threadIdx.x, c = t & 7;
    u32x2 k[NK], v[NV];
    uint8_t ks[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(a.k8 + p.kv8) + t + 256 * i);
        ks[i] = a.ks[p.scale + t / LPH + RPP * i];
    }
    const u32x2 vs = *reinterpret_cast<const u32x2*>(a.vs + p.scale + 8 * c);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(a.v8 + p.kv8) + (t / 8 + 32 * i) * 8 + c);
#pragma unroll
    for (int i = 0; i < NK; ++i)
        reinterpret_cast<f16x8*>(a.kc + p.f16)[t + 256 * i] = kv8_values(k[i][0], k[i][1], kv8_scale(ks[i]));
    const f16x2 f[4] = {kv8_factors(vs[0], 0), kv8_factors(vs[0], 1), kv8_factors(vs[1], 0), kv8_factors(vs[1], 1)};
    f16x8* const vout = reinterpret_cast<f16x8*>(a.vc + p.f16 + (c >> 2) * (D * 32)) + (c & 3);
#pragma unroll
    for (int i = 0; i < NV; ++i) vout[(t / 8 + 32 * i) * 4] = kv8_values(v[i][0], v[i][1], f);
}

template <bool FROM>
hipError_t launch_pages(const Kv8PagesArgs& a, hipStream_t st)
{
    const dim3 grid(a.n * a.n_kv * (a.block / 64u));
    auto go = [&](auto from, auto to) { hipLaunchKernelGGL((FROM ? from : to), grid, dim3(256), 0, st, a); };
    switch (a.D) {
    case 64: go(kv8_from_pages_kernel<64>, kv8_to_pages_kernel<64>); break;
    case 128: go(kv8_from_pages_kernel<128>, kv8_to_pages_kernel<128>); break;
    case 256: go(kv8_from_pages_kernel<256>, kv8_to_pages_kernel<256>); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_from_pages(const Kv8PagesArgs& a, hipStream_t st) { return launch_pages<true>(a, st); }
hipError_t launch_kv8_to_pages(const Kv8PagesArgs& a, hipStream_t st) { return launch_pages<false>(a, st); }

}  // namespace yhip
