// qmag_linattn_plan.h -- how linear attention over packed sequences is cut into chunks
// and windows, and where a chunk's results lie: arithmetic without device code, so that
// a host program can walk through it for sums of any kind.
//
// A call is taken in windows of rows, so that its workspace has a bound; a sequence that
// goes on behind its window hands its state on.  Within a window a sequence of more than
// `brief` rows is cut into chunks of LA_CHUNK; those as brief go token by token.  The
// chunks of the i-th long sequence are numbered from (first row >> 6) + i on:
// ceil(n / 64) <= (n >> 6) + 1, so that no two share a number.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "qmag_seq.h"

namespace qmag {

constexpr int LA_CHUNK = 64, LA_SHIFT = 6;

// Up to how many rows a sequence goes token by token, for the waves that this takes, 16
// columns of a head and sequence each.  Few waves wait for one another's sums, some 0.7 us
// a token, and a chunk takes 26 us whatever rows it has (one sequence of 32 heads and 128
// channels fp32, tokens and a chunk: 27 us and 26 for 32 rows, 50 and 26 for 64).  Where
// the chip is full a token costs what it computes, and a chunk what its type's bf16 parts
// (3, 2 or 1) make of it.  Sequences alike, us token by token (4 to 15 more where the call
// is cut all the same) and in chunks:
//   heads, channels           fp32 64 rows  96 rows   fp16 48 rows  56 rows   bf16 40 rows  48 rows
//   64 of 32 over 16, 64         187  278  274  368      145  173  166  178     123  155  148  155
//   64 of 32 over 16, 128        480  624  699  826      381  523  446  525     330  330  381  330
//   64 of 8 over 4, 256          452  442  641  691      339  349  395  340     294  271  335  272
//   16 of 32 over 16, 64          64   77   93   93       51   57   59   57      42   52   49   52
//   16 of 32 over 16, 128        144  150  208  189      116  132  132  133      99   92  117   92
//   16 of 8 over 4, 256          131  129  186  175      100  107  115  108      86   87  100   86
constexpr int la_brief(int64_t waves, int parts) { return waves <= 1024 ? 32 : parts == 3 ? 96 : parts == 2 ? 48 : 40; }
// Whether a call is cut: its sequences have more rows than that on average, or one of them
// may have many more, the others a row each.  A prompt of 512 tokens beside 31 single
// ones takes 81 us, token by token 436; where none is long after all, the launches that
// find nothing take 64 sequences of 8 tokens from 88 us to 92.
constexpr bool la_cut(int T, int n_seq, int brief)
{
    return T > (int64_t)brief * n_seq || (int64_t)T - n_seq >= (brief <= 32 ? 64 : 128);
}

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
constexpr bool la_long(int n, int brief) { return n > brief; }
constexpr int la_tile0(int first, int r0, int rank) { return ((first - r0) >> LA_SHIFT) + rank; }

// A window's long sequences, each of brief + 1 rows or more, and their chunks' numbers.  (Sequences that lap over one
// another may be more, or have more: what is behind these goes token by token.)
constexpr int la_most_long(int rows, int n_seq, int brief)
{
    const int most = rows / (brief + 1);
    return n_seq < most ? n_seq : most;
}
constexpr int la_most_tiles(int rows, int n_seq, int brief) { return (rows >> LA_SHIFT) + la_most_long(rows, n_seq, brief); }
constexpr bool la_room(int rank, int tile0, int chunks, int most_long, int most_tiles)
{
    return rank < most_long && tile0 + chunks <= most_tiles;
}


// ------------------------------------------------------------- workspace --
// What a chunk has there, in bytes: for each key head K's and Q's parts (three bf16 of an fp32 value, two of an fp16 one,
// one of a bf16 one); for each head the triangle's inverse and P, three parts of 6 operands of 1 KB each, 1280 bytes of
// vectors, and 64 for a row's place in each of up to 16 slices of columns.
constexpr size_t la_key_bytes(int parts, int dim_k) { return (size_t)2 * parts * LA_CHUNK * dim_k * 2; }
constexpr size_t LA_HEAD_BYTES = 2 * 6 * 3 * 1024 + 1280;
constexpr size_t la_tile_bytes(int parts, int dim_k, int n_key, int n_head)
{
    return (size_t)n_key * la_key_bytes(parts, dim_k) + (size_t)n_head * (LA_HEAD_BYTES + 64);
}

// A call's workspace is at most this; calls of more rows than it holds the chunks of go window by window, and have two
// states of `state` bytes there to hand on.
constexpr size_t LA_WORKSPACE = (size_t)1 << 30;
constexpr size_t la_workspace(int window, int T, int n_seq, int brief, size_t tile, size_t state)
{
    return (size_t)la_most_tiles(window, n_seq, brief) * tile + (T > window ? 2 * state : 0);
}
// The rows of a window, whole chunks; 0: not even two chunks are held (heads by the thousand, whose sequences fill the
// chip token by token, which takes no workspace).
constexpr int la_window(int T, int n_seq, int brief, size_t tile, size_t state)
{
    int window = ((int64_t)T + LA_CHUNK - 1) / LA_CHUNK < (1 << 20) ? (T + LA_CHUNK - 1) / LA_CHUNK * LA_CHUNK : 1 << 26;
    while (window > 0 && la_workspace(window, T, n_seq, brief, tile, state) > LA_WORKSPACE) window = window / (2 * LA_CHUNK) * LA_CHUNK;
    return window >= 2 * LA_CHUNK || window >= T ? window : 0;
}

}  // namespace qmag
