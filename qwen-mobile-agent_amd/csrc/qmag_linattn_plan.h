// qmag_linattn_plan.h -- how linear attention over packed sequences is cut into chunks
// and windows, and where a chunk's results lie: arithmetic without device code, so that
// a host program can walk through it for sums of any kind.
//
// A call is taken in windows of rows, so that its workspace has a bound; a sequence that
// goes on behind its window hands its state on.  Within a window a sequence of more than
// LA_SHORT rows is cut into chunks of LA_CHUNK; shorter ones go token by token.  The
// chunks of the i-th long sequence are numbered from (first row >> 6) + i on:
// ceil(n / 64) <= (n >> 6) + 1, so that no two share a number.
#pragma once

#include <stdint.h>

#include "qmag_seq.h"

namespace qmag {

constexpr int LA_CHUNK = 64, LA_SHIFT = 6, LA_SHORT = 16;

// a sequence's rows within the window [r0, r1)
struct LaRows {
    int first, n;
    bool begun, goes_on;      // rows ahead of the window, and behind it
};
constexpr LaRows la_rows(int cu0, int cu1, int T, int r0, int r1)
{
    const int a = seq_row(cu0, T), b = seq_row(cu1, T);
    const int first = a < r0 ? r0 : a, last = b > r1 ? r1 : b;
    return {first, last > first ? last - first : 0, a < r0, b > r1};
}
constexpr bool la_long(int n) { return n > LA_SHORT; }
constexpr int la_tile0(int first, int r0, int rank) { return ((first - r0) >> LA_SHIFT) + rank; }
constexpr bool la_room(int tile0, int chunks, int most) { return tile0 + chunks <= most; }

// numbers of a window of `rows` rows: its long sequences are at most n_seq, and have
// LA_SHORT + 1 rows each
constexpr int la_most_tiles(int rows, int n_seq)
{
    const int most = rows / (LA_SHORT + 1) + 1;
    return (rows >> LA_SHIFT) + (n_seq < most ? n_seq : most);
}

}  // namespace qmag
