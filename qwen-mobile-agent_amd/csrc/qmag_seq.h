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
// n_seq >= 1; cu(i) gives the sum at i.
template <class F>
constexpr SeqTile seq_find(F cu, int n_seq, int T, int shift, int j)
{
    int lo = 0, hi = n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (seq_tile0(seq_row(cu(mid), T), mid, shift) <= j) lo = mid;
        else hi = mid - 1;
    }
    const int first = seq_row(cu(lo), T), n = seq_row(cu(lo + 1), T) - first;
    const int tile = j - seq_tile0(first, lo, shift);
    if (tile < 0 || tile >= seq_tiles(n, shift)) return {-1, 0, 0, 0};
    return {lo, tile, first, n};
}

}  // namespace qmag
