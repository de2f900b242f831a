// Host-side checks of ferrite-tpu_amd/csrc/table_row.h: a lookup's row, its row of NaN, and where it stops the program.
#include "../../ferrite-tpu_amd/csrc/table_row.h"

#include <cstdio>
#include <initializer_list>

using namespace ferrite;

static int failures = 0;
#define CHECK(c)                                                \
  do {                                                          \
    if (!(c)) {                                                 \
      std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #c); \
      ++failures;                                               \
    }                                                           \
  } while (0)

int main() {
  const int64_t far[] = {INT64_MIN, INT64_MIN + 1, -((int64_t)1 << 40), (int64_t)1 << 40, INT64_MAX};
  const int64_t vocabs[] = {1, 5, 3000, 0x7ffffffe};
  for (int64_t vocab : vocabs) {
    for (int64_t t : {(int64_t)0, vocab / 2, vocab - 1}) {
      CHECK(table_row(t, vocab, false) == t);
      CHECK(table_row(t, vocab, true) == t);
      CHECK(table_row(t - vocab, vocab, true) == t);
      CHECK(table_row(t - vocab, vocab, false) == kNoRow);
    }
    CHECK(table_row(vocab, vocab, false) == kNoRow);
    CHECK(table_row(vocab, vocab, true) == kStopRow);
    CHECK(table_row(-vocab - 1, vocab, true) == kStopRow);
    for (int64_t t : far) {
      CHECK(table_row(t, vocab, false) == kNoRow);
      CHECK(table_row(t, vocab, true) == kStopRow);
    }
  }
  if (failures) return 1;
  std::printf("all checks passed\n");
}
