// qmag_rope.hip -- rotary positions with one to four axes on the heads of a
// projection (the role of rope_imrope, src/nn.c:841-861).
//
// Pair i of a head turns by a = pos[axis(i)][t] * theta^(-2 i / n_rot):
//   y_i = x_i cos a - x_j sin a,   y_j = x_i sin a + x_j cos a.
// Far positions make a large: it is formed in turns (a / 2 pi) in 64 bits and its
// whole turns dropped exactly.  The fraction goes to fp32, and what that leaves of it
// (up to 2 pi 2^-26, much beside a sine near half a turn) is added to first order.
//
// A workgroup takes one token and some of its heads: the token's cosines and
// sines go to LDS once, then each thread turns 16 bytes of pairs.  Memory
// bound beyond a few hundred tokens: 4096 of 32 + 8 heads of 128 in bf16 15.1 us, 5.6
// TB/s (84 MB, part of which stays in the caches); one token is a launch, 3.4 us.
#include <math.h>

#include "qmag_attn.h"

namespace qmag {

constexpr int ROPE_MAX_PAIRS = 128;

struct RopeArgs {
    double turns[ROPE_MAX_PAIRS];     // theta^(-2 i / n_rot) / 2 pi
    uint8_t axis[ROPE_MAX_PAIRS];
    struct {
        const void *src;
        void *dst;
        int64_t st, sh, dt, dh;       // strides of a token and of a head
        int n;
    } view[2];
    const int *pos;
    int T, dim, pairs;
    int heads_per_wg;                 // over both views
    int unit_shift;                   // threads of a head, a power of two
    int copy;                         // values beyond n_rot are copied
};

// V values to a thread and step, 1 where alignment or sizes do not allow 16 bytes
template <class T, int V, bool ADJ>
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs A)
{
    using S = typename T::S;
    struct alignas(V * sizeof(S)) Vec { S v[V]; };
    __shared__ float2 cs[ROPE_MAX_PAIRS];
    const int tid = threadIdx.x;
    const int h0 = blockIdx.y * A.heads_per_wg, h1 = min(h0 + A.heads_per_wg, A.view[0].n + A.view[1].n);
    const int per = 256 >> A.unit_shift;
    const int rot_units = (ADJ ? 2 * A.pairs : A.pairs) / V;
    const int units = rot_units + (A.copy ? (A.dim - 2 * A.pairs) / V : 0);
    for (int64_t t = blockIdx.x; t < A.T; t += gridDim.x) {
        if (tid < A.pairs) {
            double r = (double)A.pos[A.axis[tid] * (int64_t)A.T + t] * A.turns[tid];
            r -= rint(r);
            const float f = (float)r, rest = (float)((r - (double)f) * (2.0 * M_PI));
            float s, c;
            sincospif(2.0f * f, &s, &c);
            cs[tid] = make_float2(fmaf(-rest, s, c), fmaf(rest, c, s));
        }
        __syncthreads();
        for (int h = h0 + (tid >> A.unit_shift); h < h1; h += per) {
            const int w = h >= A.view[0].n, hh = w ? h - A.view[0].n : h;
            const auto &v = A.view[w];
            const S *src = (const S *)v.src + t * v.st + hh * v.sh;
            S *dst = (S *)v.dst + t * v.dt + hh * v.dh;
            for (int u = tid & ((1 << A.unit_shift) - 1); u < units; u += 1 << A.unit_shift) {
                if (u >= rot_units) {
                    const int i = 2 * A.pairs + (u - rot_units) * V;
                    *reinterpret_cast<Vec *>(dst + i) = *reinterpret_cast<const Vec *>(src + i);
                } else if constexpr (ADJ && V >= 2) {
                    Vec x = *reinterpret_cast<const Vec *>(src + u * V);
    #pragma unroll
                    for (int k = 0; k < V; k += 2) {
                        const float2 f = cs[(u * V + k) / 2];
                        const float a = T::up(x.v[k]), b = T::up(x.v[k + 1]);
                        x.v[k] = T::down(a * f.x - b * f.y);
                        x.v[k + 1] = T::down(a * f.y + b * f.x);
                    }
                    *reinterpret_cast<Vec *>(dst + u * V) = x;
                } else if constexpr (ADJ) {
                    if (u & 1) continue;
                    const float2 f = cs[u / 2];
                    const float a = T::up(src[u]), b = T::up(src[u + 1]);
                    dst[u] = T::down(a * f.x - b * f.y);
                    dst[u + 1] = T::down(a * f.y + b * f.x);
                } else {
                    Vec x = *reinterpret_cast<const Vec *>(src + u * V);
                    Vec y = *reinterpret_cast<const Vec *>(src + A.pairs + u * V);
    #pragma unroll
                    for (int k = 0; k < V; k++) {
                        const float2 f = cs[u * V + k];
                        const float a = T::up(x.v[k]), b = T::up(y.v[k]);
                        x.v[k] = T::down(a * f.x - b * f.y);
                        y.v[k] = T::down(a * f.y + b * f.x);
                    }
                    *reinterpret_cast<Vec *>(dst + u * V) = x;
                    *reinterpret_cast<Vec *>(dst + A.pairs + u * V) = y;
                }
            }
        }
        __syncthreads();      // the next token's angles
    }
}

}  // namespace qmag

using namespace qmag;

extern "C" int qmag_rope_dev(const qmag_rope *r, const int *pos, int T, int type, const qmag_heads *src,
                             const qmag_heads *dst, int n_views)
{
    int st;
    if (!r || (!pos && T > 0) || !src || !dst) return fail(QMAG_ERR_ARG, "rope: null pointer");
    if (T < 0 || n_views < 1 || n_views > 2) return fail(QMAG_ERR_ARG, "rope: T=%d n_views=%d", T, n_views);
    const int size = attn_type_size(type);
    if (!size) return fail(QMAG_ERR_ARG, "rope: type %d", type);
    if (r->head_dim < 2 || r->head_dim > QMAG_ROPE_MAX_DIM || r->n_rot < 2 || r->n_rot % 2 || r->n_rot > r->head_dim ||
        r->n_rot > 2 * ROPE_MAX_PAIRS)
        return fail(QMAG_ERR_ARG, "rope: head_dim=%d n_rot=%d", r->head_dim, r->n_rot);
    if (r->n_axes < 1 || r->n_axes > 4) return fail(QMAG_ERR_ARG, "rope: n_axes=%d", r->n_axes);
    if (!(r->theta > 0.0) || !isfinite(r->theta)) return fail(QMAG_ERR_ARG, "rope: theta=%g", r->theta);
    int left[4] = {0, 0, 0, 0};
    long sum = 0;
    for (int a = 0; a < r->n_axes; a++) {
        if (r->sections[a] < 0) return fail(QMAG_ERR_ARG, "rope: sections[%d]=%d", a, r->sections[a]);
        left[a] = r->sections[a];
        sum += left[a];
    }
    if (sum != r->n_rot / 2) return fail(QMAG_ERR_ARG, "rope: sections hold %ld pairs of %d", sum, r->n_rot / 2);
    if ((uintptr_t)pos % 4) return fail(QMAG_ERR_ARG, "rope: pos is not aligned");

    RopeArgs A = {};
    A.pairs = r->n_rot / 2;
    for (int i = 0, a = 0; i < A.pairs; i++) {
        // pairs to the axes in runs, or in turns that pass over an axis with none left
        while (!left[a]) a = (a + 1) % r->n_axes;
        A.axis[i] = (uint8_t)a;
        left[a]--;
        if (r->interleaved) a = (a + 1) % r->n_axes;
        A.turns[i] = pow(r->theta, -2.0 * i / r->n_rot) / (2.0 * M_PI);
        if (!isfinite(A.turns[i] * 2147483648.0)) return fail(QMAG_ERR_ARG, "rope: theta=%g, whose angles leave 64 bits", r->theta);
    }
    A.pos = pos;
    A.T = T;
    A.dim = r->head_dim;
    bool vec = true;
    for (int v = 0; v < n_views; v++) {
        if ((st = check_heads("rope src", &src[v], type, r->head_dim, T, false))) return st;
        if ((st = check_heads("rope dst", &dst[v], type, r->head_dim, T, true))) return st;
        if (src[v].n_head != dst[v].n_head)
            return fail(QMAG_ERR_ARG, "rope: %d heads to %d", src[v].n_head, dst[v].n_head);
        const bool same = src[v].ptr == dst[v].ptr && src[v].token_stride == dst[v].token_stride &&
                          src[v].head_stride == dst[v].head_stride;
        if (!same && heads_overlap(&src[v], &dst[v], size, r->head_dim, T))
            return fail(QMAG_ERR_ARG, "rope: view %d's destination overlaps its source without being it", v);
        A.copy |= !same;
        vec = vec && heads_aligned(&src[v], type) && heads_aligned(&dst[v], type);
        A.view[v] = {src[v].ptr, dst[v].ptr, src[v].token_stride, src[v].head_stride, dst[v].token_stride,
                     dst[v].head_stride, src[v].n_head};
    }
    // one view's destination over the other's source or destination would be a race
    if (n_views == 2 && (heads_overlap(&dst[0], &src[1], size, r->head_dim, T) ||
                         heads_overlap(&dst[0], &dst[1], size, r->head_dim, T) ||
                         heads_overlap(&src[0], &dst[1], size, r->head_dim, T)))
        return fail(QMAG_ERR_ARG, "rope: the views overlap");
    const int n = A.view[0].n + A.view[1].n;
    if ((st = require_ready())) return st;
    if (n == 0 || T == 0) return QMAG_OK;
    const int V = 16 / size;
    vec = vec && r->head_dim % V == 0 && (r->adjacent ? r->n_rot : A.pairs) % V == 0;
    const int v = vec ? V : 1;
    const int units = ((r->adjacent ? 2 : 1) * A.pairs + (A.copy ? r->head_dim - 2 * A.pairs : 0)) / v;
    while ((1 << A.unit_shift) < units && A.unit_shift < 8) A.unit_shift++;
    // a head to every 256 >> unit_shift threads; one token's heads go to
    // several workgroups until there are enough of those for every CU
    const int per = 256 >> A.unit_shift;
    int wgs = (n + per - 1) / per;
    while (wgs > 1 && (int64_t)T * wgs > 2048) wgs = (wgs + 1) / 2;
    A.heads_per_wg = (n + wgs - 1) / wgs;
    wgs = (n + A.heads_per_wg - 1) / A.heads_per_wg;

    DeviceScope dev;
    if (dev.st) return dev.st;
    hipStream_t s = ctx().stream;
    const dim3 grid((unsigned)(T < 1 << 20 ? T : 1 << 20), (unsigned)wgs);
    prof_begin(PROF_ROPE, s);
    with_type(type, [&](auto t) {
        using TT = decltype(t);
        constexpr int VV = 16 / (int)sizeof(typename TT::S);
        if (vec && r->adjacent) rope_kernel<TT, VV, true><<<grid, 256, 0, s>>>(A);
        else if (vec) rope_kernel<TT, VV, false><<<grid, 256, 0, s>>>(A);
        else if (r->adjacent) rope_kernel<TT, 1, true><<<grid, 256, 0, s>>>(A);
        else rope_kernel<TT, 1, false><<<grid, 256, 0, s>>>(A);
        return 0;
    });
    prof_end(PROF_ROPE, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}
