// dh_vocab_range.hpp -- how far the vocabulary products' loads may reach.  Plain C++, so that it can be
// checked without a GPU.
#pragma once
#include <cstdint>

namespace dh {

// An operand's columns (of m, n or k) in whole 16-byte chunks, in which it is loaded: that many values
// of a row must be readable.  Rows of the workspace are padded; a table read in place has whole chunks.
constexpr int chunk_end(int extent) { return (extent + 7) / 8 * 8; }

// The range in bytes of `rows` rows of ld 16-bit values, from column t0 of the first: to the end of the last
// row's `extent` columns and not to the end of its ld, which a matrix inside a wider one does not have.
constexpr uint32_t range_bytes(int rows, int ld, int extent, int t0) {
    return rows <= 0 ? 0u : 2u * ((uint32_t)(rows - 1) * (uint32_t)ld + (uint32_t)(chunk_end(extent) - t0));
}

}  // namespace dh
