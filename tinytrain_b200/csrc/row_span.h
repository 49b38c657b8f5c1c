// What a bulk copy may move of one row of a dense tensor whose rows are no whole
// number of 16-byte words. Plain C++, so that it can be checked on the host.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define TTK_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TTK_HOST_DEVICE inline
#endif

namespace ttk {

// A row of D floats begins `off` floats into its first word (off = row * D mod 4,
// the tensor starting on a word). `words` words from that one on are copied whole,
// with what they hold of the neighbouring rows; the row's floats from 4 * words
// to its end (at off + D) lie in a word that the tensor's end cuts short (R rows),
// which no copy of whole words may touch. Rows before the last one can end in
// that word too: those of width 1.
struct RowSpan {
    int words, end;
};

TTK_HOST_DEVICE RowSpan row_span(int64_t row, int64_t R, int64_t D, int off) {
    const int end = off + static_cast<int>(D), words = (end + 3) / 4;
    const bool cut = (R - row) * D + off < 4 * words;  // the tensor ends inside the last word
    return {cut ? words - 1 : words, end};
}

}  // namespace ttk
