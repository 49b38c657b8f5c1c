// row_tail (tinytrain_b200/csrc/row_span.h) for every row of small tensors and the
// ends of larger ones: the whole words stay inside the tensor, and with the
// floats after them they cover the row. Prints "ok" and exits 0 on success.
#include <cstdio>
#include <initializer_list>

#include "row_span.h"

int main() {
    int bad = 0;
    for (int64_t D = 1; D <= 70; ++D)
        for (int64_t R : {1, 2, 3, 4, 5, 6, 7, 8, 9, 31, 4096, 4099})
            for (int64_t row = R > 16 ? R - 16 : 0; row < R; ++row) {
                const int off = static_cast<int>(row * D & 3);
                const int64_t first = row * D - off;  // the first word's first float
                const int end = off + static_cast<int>(D);
                const int tail = ttk::row_tail(row, ttk::first_cut_row(R, D), end);
                const int words = (end - tail + 3) / 4;  // copied whole
                const bool inside = words >= 0 && first + 4 * words <= R * D;
                const bool covers = tail >= 0 && tail <= 3 && 4 * words >= end - tail;
                if (!inside || !covers) {
                    std::printf("R %lld D %lld row %lld: %d words from %lld, end %d\n", (long long)R,
                                (long long)D, (long long)row, words, (long long)first, end);
                    ++bad;
                }
            }
    if (!bad)
        std::printf("ok\n");
    return bad != 0;
}
