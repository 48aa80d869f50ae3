// paged_items8.hpp -- what the kernels over the 8-bit KV pool (kv8.hpp) add to
// paged_items.hpp: where a page's codes and scales are, and its NaNs.
#pragma once

#include "kv8.hpp"
#include "paged_items.hpp"

#include <math.h>

#include <type_traits>

namespace yhip {
namespace {

__device__ inline const PagedAttn8Args& fresh_args(const PagedAttn8Args&)
{
    auto p = (const PagedAttn8Args __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const PagedAttn8Args*)p;
}

__device__ inline const PagedMixed8Args& fresh_args(const PagedMixed8Args&)
{
    auto p = (const PagedMixed8Args __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const PagedMixed8Args*)p;
}
static_assert(sizeof(PagedMixed8Args) == sizeof(PagedAttn8Args) + sizeof(PagedFew8Args), "the second part follows the first");
__device__ inline const PagedFew8Args& fresh_args(const PagedFew8Args&)
{
    auto p = (const char __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr() + sizeof(PagedAttn8Args);
    asm volatile("" : "+s"(p));
    return *(const PagedFew8Args*)p;
}

// A sequence's units among the tiles' items: those with few tokens are the
// decode kernel's (its line has the others' complement).
__device__ inline bool few_rows(const PagedAttn8Args& a, const PagedSeq& s) { return a.gmax * s.nq <= a.few; }
__device__ inline uint64_t seq_units(const PagedAttn8Args& a, const PagedSeq& s)
{
    return few_rows(a, s) ? 0 : seq_units(static_cast<const PagedAttnArgs&>(a), s);
}
struct Paged8Line {
    static __device__ uint64_t units(const PagedAttnArgs& a, const PagedSeq& s)
    {
        return seq_units(static_cast<const PagedAttn8Args&>(a), s);
    }
};

// first byte and number (0: outside the pool) of the scales of kv head kvh's part of a page; its codes are D times both
struct Paged8Tile {
    uint64_t at;
    uint32_t bytes;
};
__device__ inline Paged8Tile paged8_tile(const PagedAttnArgs& a, uint32_t page, uint32_t kvh)
{
    const bool in = page < a.n_blocks;
    return Paged8Tile{(uint64_t)(in ? page * a.n_kv + kvh : 0u) << a.shift, in ? 1u << a.shift : 0u};
}

// bit k: among the values of dimension d + k that a query at position pos sees of keys lo .. end - 1 is a NaN
template <int D>
__device__ uint32_t nan_dims(const PagedAttn8Args& a, uint32_t seq, uint32_t kvh, uint32_t d, int pos, uint32_t lo, int end)
{
    uint32_t found = 0;
#pragma unroll 1
    for (uint32_t k = lo; (int)k < end && (int)k <= pos; ++k) {
        const Paged8Tile t = paged8_tile(a, (uint32_t)a.table[(size_t)seq * a.table_stride + (k >> a.shift)], kvh);
        if (t.bytes == 0) continue;
        const uint32_t off = k & ((1u << a.shift) - 1u);
        const uint8_t* p = reinterpret_cast<const uint8_t*>(a.vc) + t.at * D + (size_t)(off & ~63u) * D + d * kV8Tile + (off & 63u);
#pragma unroll 1
        for (uint32_t e = 0; e < 4; ++e) found |= (p[e * kV8Tile] & 0x7f) == 0x7f ? 1u << e : 0u;
    }
    return found;
}

}  // namespace
}  // namespace yhip
