// paged_decode8_lds.hpp -- a wave's share of the LDS in paged_decode8.hpp.
#pragma once

namespace yhip {

constexpr int kDecode8Rows = 16;  // of a block

// Floats of a share: a wave's O rows [16][D + 4], their maxima and sums, a flag
// (padded); the first wave's before that the queries as f16 [parts][16][D + 8],
// hi and lo parts of fp32 ones (PREC), which need the more: at head_dim 256
// 16896 bytes beside 16784.
template <int D>
constexpr int kDecode8Out = kDecode8Rows * (D + 4) + 2 * kDecode8Rows + 4;
template <int D, bool PREC>
constexpr int kDecode8Queries = (PREC ? 2 : 1) * kDecode8Rows * (D + 8) / 2;
template <int D, bool PREC>
constexpr int kDecode8Lds =
    kDecode8Out<D> > kDecode8Queries<D, PREC> ? kDecode8Out<D> : kDecode8Queries<D, PREC>;

}  // namespace yhip
