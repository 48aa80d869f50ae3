// paged_chunks.hpp -- into how many chunks of how many units the line of a
// paged attention launch is cut (paged_items.hpp).
#pragma once

#include <stdint.h>

namespace yhip {

struct PagedChunks {
    uint32_t units, n;  // of a chunk; chunks
};

// A line of `total` units (below 2^38, checked on the host) for n_wg
// workgroups: equal chunks of at least min_units, one per workgroup at most.
// Below 2^31 units by the shorter 32-bit divisions (from there on, total plus
// n_wg or a chunk could pass 32 bits).
constexpr PagedChunks paged_chunks(uint64_t total, uint32_t n_wg, uint32_t min_units)
{
    const bool small = (total >> 31) == 0;
    const uint32_t t = (uint32_t)total;
    uint64_t even = small ? (t + n_wg - 1) / n_wg : (total + n_wg - 1) / n_wg;
    if (even > 0x7fffffffu) even = 0x7fffffffu;
    const uint32_t units = even > min_units ? (uint32_t)even : min_units;
    return PagedChunks{units, small ? (t + units - 1) / units : (uint32_t)((total + units - 1) / units)};
}

}  // namespace yhip
