// Rows of the biased softmax's groups (kernels/positions.cuh, RowTurns) against 64-bit arithmetic.
#include <cstdio>
#include <initializer_list>

#include "kernels/positions.cuh"

int main() {
  long checked = 0;
  for (int32_t rows : {1, 2, 31, 32, 33, 4096, 2146900000, 2147330000, 2147483646, 2147483647})
    for (int32_t step : {1, 32, 4096, 148 * 32, 148 * 6 * 32, 148 * 16 * 32, 8 * 148 * 16 * 32, 2147483647}) {
      if (rows > 10000 && step < 4096) continue;
      for (int32_t first : {0, 1, 31, step / 2, step - 1}) {
        if (first < 0 || first >= step) continue;
        cs::RowTurns t(rows, first, step);
        int64_t i = first;
        for (; t.inside(); t.next(), i += step, ++checked) {
          const int64_t row = rows - 1 - i, next = row - step;
          if (row < 0 || t.row() != row || t.here() != row || t.last() != (next < 0) || t.next_row() != (next < 0 ? 0 : next))
            return std::printf("rows %d step %d first %d turn %lld\n", rows, step, first, (long long)i), 1;
        }
        if (i < rows) return std::printf("rows %d step %d first %d ends early\n", rows, step, first), 1;
        if (first >= rows && t.row() != 0) return std::printf("outside\n"), 1;
      }
    }
  std::printf("ok %ld\n", checked);
  return 0;
}
