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
// the tensor starting on a word) and ends at off + D. Words are copied whole, with
// what they hold of the neighbouring rows, but for a word that the tensor's end cuts
// short, which no such copy may touch.

// The first row that may end in that word: the last one, or with width 1 all that
// share it.
TTK_HOST_DEVICE int64_t first_cut_row(int64_t R, int64_t D) { return D == 1 ? R - R % 4 : R - 1; }

// How many floats before `end` = off + D lie in it.
TTK_HOST_DEVICE int row_tail(int64_t row, int64_t first_cut, int end) {
    return row >= first_cut ? end % 4 : 0;
}

}  // namespace ttk
