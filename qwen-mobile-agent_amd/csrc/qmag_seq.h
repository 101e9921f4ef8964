// qmag_seq.h -- packed sequences cut into tiles of tokens: which tile a workgroup
// has, from the sums of the lengths on the device.  The arithmetic is free of device
// code, so that a host program can walk through it for sums of any kind.
//
// Sequence i is rows cu[i] .. cu[i + 1] - 1; its tiles, of 2^shift tokens each, are
// numbered from (cu[i] >> shift) + i on.  ceil(n / 2^shift) <= (n >> shift) + 1, so
// that no two sequences share a number, and all of T rows have less than
// (T >> shift) + n_seq: no prefix sums over the sequences are needed, and a number
// names its sequence by a search over cu.
#pragma once

#include <stdint.h>

namespace qmag {

// cu as the kernels take it: a row within [0, T]
constexpr int seq_row(int cu, int T) { return cu < 0 ? 0 : cu > T ? T : cu; }
constexpr int seq_tile0(int row, int i, int shift) { return (row >> shift) + i; }
constexpr int seq_tiles(int n, int shift) { return n > 0 ? ((n - 1) >> shift) + 1 : 0; }
constexpr int seq_most_tiles(int T, int n_seq, int shift) { return (T >> shift) + n_seq; }

struct SeqTile {
    int seq;        // -1: none has this number
    int tile;       // which of its tiles
    int first, n;   // its first row, and how many it has
};

// Tile number j: the last sequence that begins at or ahead of it, if it reaches j.
// n_seq >= 1; cu(i) gives the sum at i, vote(f) the bits f(0) .. f(63), all of which a
// wave asks at once: 4096 sequences in two rounds.
template <class F, class V>
constexpr SeqTile seq_find(F cu, V vote, int n_seq, int T, int shift, int j)
{
    int lo = 0;
    for (int left = n_seq; left > 1;) {
        const int step = (left - 1) / 64 + 1;
        const uint64_t ahead = vote([&](int i) {
            const int at = lo + (i * step < left ? i * step : 0);
            return i * step < left && seq_tile0(seq_row(cu(at), T), at, shift) <= j;
        });
        const int hit = ahead ? 63 - __builtin_clzll(ahead) : 0;
        lo += hit * step;
        left = left - hit * step < step ? left - hit * step : step;
    }
    const int first = seq_row(cu(lo), T), n = seq_row(cu(lo + 1), T) - first;
    const int tile = j - seq_tile0(first, lo, shift);
    if (tile < 0 || tile >= seq_tiles(n, shift)) return {-1, 0, 0, 0};
    return {lo, tile, first, n};
}

}  // namespace qmag
