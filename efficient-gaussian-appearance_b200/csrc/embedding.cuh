// Rows of embedding indices (embedding.cu) as sort keys (sort.cu).
#pragma once

#include <cstdint>

namespace fgs {

// row of an index: the row itself, kNoRow (a negative or the padding index) or kBadRow (past the table)
constexpr uint32_t kNoRow = 0xFFFFFFFFu, kBadRow = 0xFFFFFFFEu;
template <typename I>
__device__ inline uint32_t row_of(I index, int64_t rows, int64_t padding) {
    const int64_t i = static_cast<int64_t>(index);
    if (i < 0 || i == padding) return kNoRow;
    return i < rows ? static_cast<uint32_t>(i) : kBadRow;
}

// its sort key: the row, or `rows` for indices that add to none
template <typename I>
__device__ inline uint32_t row_key(I index, int64_t rows, int64_t padding) {
    const uint32_t r = row_of(index, rows, padding);
    return r < kBadRow ? r : static_cast<uint32_t>(rows);
}

}  // namespace fgs
