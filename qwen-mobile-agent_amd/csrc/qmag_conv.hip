// qmag_conv.hip -- short causal convolution of a recurrent layer (the role of
// conv1d_layer, src/nn.c:717): each channel by its own 2 to 4 taps over packed
// sequences, the last inputs of each kept in a state.
//
//   y[t][c] = bias[c] + sum_w weight[c][w] x[t - W + 1 + w][c],  out = y or y / (1 + e^-y)
//
// A thread takes the channels of 16 bytes and walks down a tile of tokens, the
// W - 1 inputs behind it in registers, so that a value is read once but for a
// tile's first W - 1 rows.  Tiles are of 4 tokens or more: only a sequence's first
// tile reaches ahead of its rows, so that the thread that reads a channel's state
// is the one that replaces it, and no other looks at it.
//
// Bound by memory: 4096 tokens of 8192 fp32 channels and 4 taps take 58.5 us, of
// which reading and writing them alone is 56 at the 4.8 TB/s of a copy; 5003 tokens
// of 4100 bf16 channels 23.6 us (3.5 TB/s; no row begins at 16 bytes, and a tile of 8
// tokens reads 10 rows).  Five tokens take 3.9 us, a launch and four loads that wait
// for one another: cu, the slot, the state, the rows.
#include "qmag_rows.h"
#include "qmag_seq.h"

namespace qmag {

struct ConvArgs {
    const void *x;
    void *out;
    int64_t xs, os;
    const float *weight, *bias;
    float *state;
    const int *slot, *len, *cu;
    int n_channel, n_slot, n_seq, T, shift, n_tile, across, silu;
};

// V values from p, or only the first n of them, the others zero
template <class T, int V, bool FULL>
__device__ __forceinline__ void load_some(const typename T::S *p, int n, float (&o)[V])
{
    if constexpr (FULL) {
        load_row<T, V>(p, o);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = i < n ? T::up(p[i]) : 0.0f;
    }
}
template <class T, int V, bool FULL>
__device__ __forceinline__ void store_some(typename T::S *p, int n, const float (&v)[V])
{
    if constexpr (FULL) {
        store_row<T, V>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) p[i] = T::down(v[i]);
    }
}

// y / (1 + e^-y), e^-y as a square, so that it does not leave fp32's range where the result is above its smallest normal
// number (y of -92), both sides times 2^-8, so that what is divided by has a normal reciprocal there; y itself loses
// digits to that below 2^-118 only, 2^-143 at most.  (Two scales chosen by a comparison: 24.4 us for 5003 tokens of 4100
// bf16 channels against 23.)
__device__ __forceinline__ float conv_silu(float y)
{
    const float half = __builtin_amdgcn_exp2f(y * -0.72134752044448170368f) * 0x1p-4f;      // e^(-y/2) / 16
    return (y * 0x1p-8f) * __builtin_amdgcn_rcpf(fmaf(half, half, 0x1p-8f));
}

// a tile's channels from c0 on: V of them, or the row's last nc.  Rows are asked for 16 values ahead of those at work:
// 32 of bf16 ones take so many registers that three waves fit where four do (26.4 us against 23.6).
template <class T, int W, bool FULL>
__device__ __forceinline__ void conv_tile(const ConvArgs &A, const SeqTile &s, int c0, int nc)
{
    using S = typename T::S;
    constexpr int V = 16 / (int)sizeof(S), AT_ONCE = 16 / V;
    const S *x = (const S *)A.x + c0;
    S *out = (S *)A.out + c0;
    const int tokens = 1 << A.shift;
    const int64_t row = (int64_t)s.first + ((int64_t)s.tile << A.shift);
    const int n = min(tokens, s.n - (s.tile << A.shift));
    float v[AT_ONCE][V], past[W - 1][V], w[V * W], bias[V];
#pragma unroll
    for (int u = 0; u < AT_ONCE; u++) load_some<T, V, FULL>(x + (row + min(u, n - 1)) * A.xs, nc, v[u]);
    load_some<TF32, V * W, FULL>(A.weight + (int64_t)c0 * W, nc * W, w);
    if (A.bias) {
        load_some<TF32, V, FULL>(A.bias + c0, nc, bias);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) bias[i] = 0.0f;
    }
    const int slot = A.slot ? __builtin_amdgcn_readfirstlane(ldg(A.slot + s.seq)) : -1;
    const bool held = s.tile == 0 && slot >= 0 && slot < A.n_slot;
    float *state = A.state + (int64_t)(held ? slot : 0) * (W - 1) * A.n_channel + c0;
    if (s.tile > 0) {
#pragma unroll
        for (int k = 0; k < W - 1; k++) load_some<T, V, FULL>(x + (row - (W - 1) + k) * A.xs, nc, past[k]);
    } else if (held && !(A.len && __builtin_amdgcn_readfirstlane(ldg(A.len + s.seq)) <= 0)) {
#pragma unroll
        for (int k = 0; k < W - 1; k++) load_some<TF32, V, FULL>(state + (int64_t)k * A.n_channel, nc, past[k]);
    } else {
#pragma unroll
        for (int k = 0; k < W - 1; k++)
#pragma unroll
            for (int i = 0; i < V; i++) past[k][i] = 0.0f;
    }
    for (int t0 = 0; t0 < n; t0 += AT_ONCE) {
        // (asked for behind the tile's end too, its last row: a load in a branch is waited for at the branch's end)
        float next[AT_ONCE][V];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) load_some<T, V, FULL>(x + (row + min(t0 + AT_ONCE + u, n - 1)) * A.xs, nc, next[u]);
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            if (t0 + u >= n) break;
            float y[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                float a = bias[i];
#pragma unroll
                for (int k = 0; k < W - 1; k++) a = fmaf(w[i * W + k], past[k][i], a);
                a = fmaf(w[i * W + W - 1], v[u][i], a);
                y[i] = A.silu ? conv_silu(a) : a;
#pragma unroll
                for (int k = 0; k + 1 < W - 1; k++) past[k][i] = past[k + 1][i];
                past[W - 2][i] = v[u][i];
            }
            store_some<T, V, FULL>(out + (row + t0 + u) * A.os, nc, y);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
            for (int i = 0; i < V; i++) v[u][i] = next[u][i];
    }
    if (held) {
        // a sequence longer than its first tile: its last rows; else what the tile ends with
        if (s.n > tokens) {
#pragma unroll
            for (int k = 0; k < W - 1; k++)
                load_some<T, V, FULL>(x + ((int64_t)s.first + s.n - (W - 1) + k) * A.xs, nc, past[k]);
        }
#pragma unroll
        for (int k = 0; k < W - 1; k++) store_some<TF32, V, FULL>(state + (int64_t)k * A.n_channel, nc, past[k]);
    }
}

template <class T, int W>
__global__ void __launch_bounds__(256, 4) conv_kernel(ConvArgs A)
{
    constexpr int V = 16 / (int)sizeof(typename T::S);
    const int c0 = (int)(blockIdx.x % A.across * blockDim.x + threadIdx.x) * V;
    for (int j = blockIdx.x / A.across; j < A.n_tile; j += gridDim.x / A.across) {
        const SeqTile s = seq_find([&](int i) { return ldg(A.cu + i); }, [&](auto f) { return __ballot(f(lane_id())); },
                                   A.n_seq, A.T, A.shift, j);
        if (s.seq < 0) continue;
        if (c0 + V <= A.n_channel) conv_tile<T, W, true>(A, s, c0, V);
        else if (c0 < A.n_channel) conv_tile<T, W, false>(A, s, c0, A.n_channel - c0);
    }
}

}  // namespace qmag

using namespace qmag;

extern "C" int qmag_conv_dev(const qmag_conv *c, int type, const void *x, int64_t x_stride, void *out, int64_t out_stride,
                             const int *slot, const int *len, const int *cu, int n_seq, int T)
{
    if (!c) return fail(QMAG_ERR_ARG, "conv: null descriptor");
    const int size = attn_type_size(type);
    if (!size) return fail(QMAG_ERR_ARG, "conv: type %d", type);
    if (c->n_channel < 1 || c->n_channel > QMAG_CONV_MAX_CHANNEL || c->width < 2 || c->width > 4 || c->n_slot < 0)
        return fail(QMAG_ERR_ARG, "conv: %d channels, width %d, %d slots", c->n_channel, c->width, c->n_slot);
    if (T < 0 || n_seq < 0 || n_seq > QMAG_KV_MAX_SEQ) return fail(QMAG_ERR_ARG, "conv: T=%d n_seq=%d", T, n_seq);
    if (!c->weight || (((uintptr_t)c->weight | (uintptr_t)c->bias | (uintptr_t)c->state) % 4) || (c->n_slot && !c->state))
        return fail(QMAG_ERR_ARG, "conv: a null or unaligned weight or state");
    if (n_seq > 0 && (!cu || (c->n_slot && !slot) || (((uintptr_t)cu | (uintptr_t)slot | (uintptr_t)len) % 4)))
        return fail(QMAG_ERR_ARG, "conv: cu or slot is null or unaligned");
    const int C = c->n_channel;
    const qmag_heads hx = {(void *)x, 1, x_stride, 0}, ho = {out, 1, out_stride, 0};
    int st;
    if ((st = check_heads("conv x", &hx, type, C, T, false))) return st;
    if ((st = check_heads("conv out", &ho, type, C, T, true))) return st;
    const size_t row = sizeof(float) * (size_t)C, held = (size_t)c->n_slot * (size_t)(c->width - 1) * row;
    const struct { const void *p; size_t n; } reads[] = {
        {c->weight, row * (size_t)c->width}, {c->bias, c->bias ? row : 0}, {slot, slot ? sizeof(int) * (size_t)n_seq : 0},
        {len, len ? sizeof(int) * (size_t)n_seq : 0}, {cu, n_seq ? sizeof(int) * ((size_t)n_seq + 1) : 0}};
    if (heads_overlap(&ho, &hx, size, C, T)) return fail(QMAG_ERR_ARG, "conv: out overlaps x");
    if (heads_meet(&ho, size, C, T, c->state, held) || heads_meet(&hx, size, C, T, c->state, held))
        return fail(QMAG_ERR_ARG, "conv: x or out overlaps the state");
    for (const auto &r : reads)
        if (heads_meet(&ho, size, C, T, r.p, r.n) || ranges_meet(c->state, held, r.p, r.n))
            return fail(QMAG_ERR_ARG, "conv: out or the state overlaps an input");
    if ((st = require_ready())) return st;
    if (T == 0 || n_seq == 0) return QMAG_OK;

    ConvArgs A = {x, out, x_stride, out_stride, c->weight, c->bias, c->state, c->n_slot ? slot : nullptr, len, cu,
                  C, c->n_slot, n_seq, T, 2, 0, 0, c->silu};
    const int per = 16 / size, threads = (C + per - 1) / per;
    // workgroups of up to four waves, as few of which are empty as may be
    const int waves = (threads + 63) / 64, across = (waves + 3) / 4, wg = (waves + across - 1) / across * 64;
    // tiles as long as leave the chip its waves: longer ones read fewer rows twice, shorter ones keep more loads on
    // their way (4100 bf16 channels: 23.6 us from 4096 waves on, 26.1 from 2048, 25.2 from 8192; 8192 fp32: 58.5, 58.5, 57.7)
    while (A.shift < 5 && (int64_t)seq_most_tiles(T, n_seq, A.shift + 1) * across * (wg / 64) >= 4096) A.shift++;
    A.n_tile = seq_most_tiles(T, n_seq, A.shift);
    A.across = across;                                // a tile's workgroups side by side: rows are read whole (80 us else)
    DeviceScope dev;
    if (dev.st) return dev.st;
    hipStream_t s = ctx().stream;
    const int most = (1 << 22) / across + 1;          // a launch holds fewer than 2^32 threads
    const unsigned grid = (unsigned)(A.n_tile < most ? A.n_tile : most) * (unsigned)across;
    prof_begin(PROF_CONV, s);
    with_type(type, [&](auto t) {
        using TT = decltype(t);
        if (c->width == 2) conv_kernel<TT, 2><<<grid, wg, 0, s>>>(A);
        else if (c->width == 3) conv_kernel<TT, 3><<<grid, wg, 0, s>>>(A);
        else conv_kernel<TT, 4><<<grid, wg, 0, s>>>(A);
        return 0;
    });
    prof_end(PROF_CONV, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}
