// qmag_attn_plan.h -- how a call over the 4-bit cache is cut into workgroups, and
// where a workgroup's partial results lie: arithmetic without device code, so that
// a host program can walk through every place that any lengths lead to.
//
// Sequence i has nq rows of q times G heads in groups of RG rows, and its `len`
// tokens in n_split chunks; an item is one group against one chunk, of one kv head.
// The host knows T, the rows of all sequences, and allots max_items; the lengths
// are the device's, and the caller's data.
#pragma once

#include <stdint.h>

namespace qmag {

// Lengths as the kernels take them: rows within [0, T], tokens within the table.
constexpr int ak_row(int cu, int T) { return cu < 0 ? 0 : cu > T ? T : cu; }
constexpr int ak_len(int len, int max_blocks, int shift)
{
    return len < 0 ? 0 : len > max_blocks << shift ? max_blocks << shift : len;
}

// groups of rows of a sequence (the host allots less than 2^23 of a call)
constexpr int ak_groups(int nq, int G, int RG) { return (int)(((int64_t)nq * G + RG - 1) / RG); }

// What a sequence adds to the call's cost, and the chunk that cuts the sum of it
// into `target` items: whole steps, more than cost / target and at least min_chunk.
constexpr float ak_cost(int groups, int len) { return (float)groups * (float)len; }
constexpr int ak_chunk(float cost, int target, int step, int min_chunk)
{
    const float c = cost / (float)target < 1073741824.0f ? cost / (float)target : 1073741824.0f;
    const int whole = (int)c / step * step + step;
    return whole > min_chunk ? whole : min_chunk;
}
constexpr int AK_UNSPLIT = 1 << 30;       // no sequence is longer

constexpr int ak_split(int len, int chunk)
{
    const int n = (int)(((unsigned)len + (unsigned)chunk - 1u) / (unsigned)chunk);
    return n > 1 ? n : 1;
}

// Items of a sequence.  (The cap only meets lengths that are none, and keeps the
// sums of them in range.)
constexpr int ak_items(int groups, int split)
{
    const int64_t n = (int64_t)groups * split;
    return n < (1 << 23) ? (int)n : 1 << 23;
}

// What the host allots: items of a kv head.  Row groups at most `groups`; of split
// sequences sum groups_i ceil(len_i / chunk) <= groups + sum groups_i len_i / chunk,
// chunk more than cost / target.  (cost is a sum in fp32, off by less than 2^-17 of
// it: less than an item of a target of some thousand.)
constexpr int64_t ak_most_groups(int T, int G, int RG, int n_seq) { return (int64_t)T * G / RG + (T < n_seq ? T : n_seq); }
constexpr int64_t ak_most_items(int64_t groups, int target, int64_t parts)
{
    return groups * parts < groups + target ? groups * parts : groups + target;
}

// Whether a sequence has all its items, which begin with item0.  Lengths that lap
// over one another make more of them than the host allots; one whose parts would
// end behind those is left out whole (the first of its items may still lie before
// the end, but a row's parts are apart by its other rows').
constexpr bool ak_room(int item0, int items, int max_items) { return item0 + items <= max_items; }

// Where row r of group `group` of a sequence whose items begin with item0 has its
// partial results, in rows, and the first place behind kv head kvh: a row's parts
// one behind another.
constexpr int64_t ak_part_row(int kvh, int max_items, int item0, int group, int n_split, int RG, int r)
{
    return ((int64_t)kvh * max_items + item0 + (int64_t)group * n_split) * RG + (int64_t)r * n_split;
}

}  // namespace qmag
