// What an embedding lookup does with a token, for the kernel (embedding.hip) and for its check on the CPU (tests/cpp/table_row_test.cpp).
#pragma once

#include <cstdint>

#if defined(__HIPCC__) || defined(__HIP__)
#define FERRITE_ROW __host__ __device__ constexpr
#else
#define FERRITE_ROW constexpr
#endif

namespace ferrite {

constexpr int64_t kNoRow = -1;    // a row of NaN
constexpr int64_t kStopRow = -2;  // the program stops

// The table's row of token t. As indexing, negative tokens count from the table's end, and one outside the table is the program's error: it
// stops, as it does in a tensor library's indexing and in the kernels of small vocabularies (layout.hip).
FERRITE_ROW int64_t table_row(int64_t t, int64_t vocab, bool indexing) {
  const int64_t row = indexing && t < 0 ? t + vocab : t;
  return row >= 0 && row < vocab ? row : indexing ? kStopRow : kNoRow;
}

}  // namespace ferrite

#undef FERRITE_ROW
