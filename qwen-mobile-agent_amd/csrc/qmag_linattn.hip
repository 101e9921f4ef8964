// qmag_linattn.hip -- linear attention with a decay for each head, plain or by the
// delta rule (the role of gdn_worker, src/nn.c:784), one state S [dim_k][dim_v] a head
// and sequence.  A token, as a recurrence:
//
//   S <- a S;  u = b (v - delta S^T k);  S <- S + k u^T;  o = scale S^T q,  a = e^g
//
// The columns of S have nothing to do with one another.  A wave takes 16 of them: lane
// l rows (l % 16) dim_k / 16 .. of columns 4 (l / 16) .., all in registers for as
// many tokens as there are.  With S0 the state ahead of a token,
//   S^T q = a S0^T q + (k . q) u,
// so that both of a token's products with the state are formed from S0, side by side,
// and one exchange over 16 lanes sums them.
#include <math.h>

#include "qmag_rows.h"
#include "qmag_seq.h"

namespace qmag {

constexpr int LA_WG = 256;

struct LaHeads {
    const void *p;
    int64_t ts, hs;
};

struct LaArgs {
    LaHeads q, k, v;
    void *out;
    int64_t ots, ohs;
    const float *decay, *beta;
    float *state;
    const int *slot, *len, *cu;
    int n_head, share, turns, dim_v, n_slot, n_seq, T;
    float norm_eps, scale;
};

// e^g: at most 1, nothing left of what a fp32 weight does not hold; a NaN stays
__device__ __forceinline__ float la_decay(float g)
{
    return g > 0.0f ? 1.0f : expf(g);
}

template <class T, int N>
struct LaToken {
    float k[N], q[N], v[4], a, b;
};

// A sequence's rows, one after another, of one head and 16 columns, by one wave.
template <class T, int DK, bool DELTA>
__device__ void la_recurrence(const LaArgs &A, int seq, int head, int c0, int first, int n)
{
    using S = typename T::S;
    constexpr int N = DK / 16;
    const int lane = lane_id(), rg = lane & 15, col = c0 + 4 * (lane >> 4);
    const int kh = A.turns ? head % A.share : head / A.share;
    const int slot = A.slot ? ldg(A.slot + seq) : -1;
    const bool held = slot >= 0 && slot < A.n_slot;
    float *state = A.state + (((int64_t)(held ? slot : 0) * A.n_head + head) * DK + rg * N) * A.dim_v + col;
    float s[N][4];
    if (held && !(A.len && ldg(A.len + seq) <= 0)) {
#pragma unroll
        for (int r = 0; r < N; r++) load_row<TF32, 4>(state + (int64_t)r * A.dim_v, s[r]);
    } else {
#pragma unroll
        for (int r = 0; r < N; r++)
#pragma unroll
            for (int c = 0; c < 4; c++) s[r][c] = 0.0f;
    }
    const S *kp = (const S *)A.k.p + first * A.k.ts + kh * A.k.hs + rg * N;
    const S *qp = (const S *)A.q.p + first * A.q.ts + kh * A.q.hs + rg * N;
    const S *vp = (const S *)A.v.p + first * A.v.ts + head * A.v.hs + col;
    S *op = (S *)A.out + first * A.ots + head * A.ohs + col;
    const float *gp = A.decay ? A.decay + (int64_t)first * A.n_head + head : nullptr;
    const float *bp = A.beta ? A.beta + (int64_t)first * A.n_head + head : nullptr;
    auto load = [&](int t, LaToken<T, N> &x) {
        load_row<T, N>(kp + t * A.k.ts, x.k);
        load_row<T, N>(qp + t * A.q.ts, x.q);
        load_row<T, 4>(vp + t * A.v.ts, x.v);
        x.a = gp ? ldg(gp + (int64_t)t * A.n_head) : 0.0f;
        x.b = bp ? ldg(bp + (int64_t)t * A.n_head) : 1.0f;
    };
    LaToken<T, N> x;
    load(0, x);
    for (int t = 0; t < n; t++) {
        LaToken<T, N> next;
        if (t + 1 < n) load(t + 1, next);
        if (A.norm_eps > 0.0f) {
            // ahead of the products: a large key's would leave fp32's range
            float kk = 0.0f, qq = 0.0f;
#pragma unroll
            for (int r = 0; r < N; r++) {
                kk = fmaf(x.k[r], x.k[r], kk);
                qq = fmaf(x.q[r], x.q[r], qq);
            }
            const float rk = rsqrtf(group_sum<16>(kk) + A.norm_eps), rq = rsqrtf(group_sum<16>(qq) + A.norm_eps);
#pragma unroll
            for (int r = 0; r < N; r++) x.k[r] *= rk, x.q[r] *= rq;
        }
        float kq = 0.0f, ks[4] = {0.0f, 0.0f, 0.0f, 0.0f}, qs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < N; r++) {
            kq = fmaf(x.k[r], x.q[r], kq);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if constexpr (DELTA) ks[c] = fmaf(x.k[r], s[r][c], ks[c]);
                qs[c] = fmaf(x.q[r], s[r][c], qs[c]);
            }
        }
        kq = group_sum<16>(kq);
        const float a = la_decay(x.a);
        float u[4], o[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if constexpr (DELTA) u[c] = x.b * fmaf(-a, group_sum<16>(ks[c]), x.v[c]);
            else u[c] = x.b * x.v[c];
            o[c] = A.scale * fmaf(kq, u[c], a * group_sum<16>(qs[c]));
        }
#pragma unroll
        for (int r = 0; r < N; r++)
#pragma unroll
            for (int c = 0; c < 4; c++) s[r][c] = fmaf(x.k[r], u[c], a * s[r][c]);
        if (rg == 0) store_row<T, 4>(op + t * A.ots, o);
        x = next;
    }
    if (held) {
#pragma unroll
        for (int r = 0; r < N; r++) store_row<TF32, 4>(state + (int64_t)r * A.dim_v, s[r]);
    }
}

template <class T, int DK, bool DELTA>
__global__ void __launch_bounds__(LA_WG) linattn_step_kernel(LaArgs A)
{
    const int slices = A.dim_v / 16;
    const int64_t jobs = (int64_t)A.n_seq * A.n_head * slices;
    for (int64_t j = (int64_t)blockIdx.x * (LA_WG / 64) + (threadIdx.x >> 6); j < jobs; j += (int64_t)gridDim.x * (LA_WG / 64)) {
        const int64_t sh = j / slices;
        const int seq = __builtin_amdgcn_readfirstlane((int)(sh / A.n_head)), head = __builtin_amdgcn_readfirstlane((int)(sh % A.n_head));
        const int c0 = __builtin_amdgcn_readfirstlane((int)(j % slices) * 16);
        const int first = seq_row(ldg(A.cu + seq), A.T), n = seq_row(ldg(A.cu + seq + 1), A.T) - first;
        if (n > 0) la_recurrence<T, DK, DELTA>(A, seq, head, c0, first, n);
    }
}

template <class F>
static int with_dim_k(int dim, F f)
{
    if (dim == 64) return f(std::integral_constant<int, 64>{});
    if (dim == 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}

}  // namespace qmag

using namespace qmag;

extern "C" int qmag_linattn_dev(const qmag_linattn *a, int type, const qmag_heads *q, const qmag_heads *k,
                                const qmag_heads *v, const qmag_heads *out, const float *decay, const float *beta,
                                const int *slot, const int *len, const int *cu, int n_seq, int T, float scale)
{
    if (!a || !q || !k || !v || !out) return fail(QMAG_ERR_ARG, "linattn: null descriptor");
    const int size = attn_type_size(type);
    if (!size) return fail(QMAG_ERR_ARG, "linattn: type %d", type);
    if ((a->dim_k != 64 && a->dim_k != 128 && a->dim_k != 256) || a->dim_v < 16 || a->dim_v > 256 || a->dim_v % 16)
        return fail(QMAG_ERR_ARG, "linattn: dim_k=%d (64, 128 or 256) dim_v=%d (a multiple of 16 to 256)", a->dim_k, a->dim_v);
    if (a->n_head < 1 || a->n_head > QMAG_MAX_HEADS || a->n_slot < 0 || !(a->norm_eps >= 0.0f) || !isfinite(a->norm_eps) || !isfinite(scale))
        return fail(QMAG_ERR_ARG, "linattn: %d heads, %d slots, norm_eps=%g, scale=%g", a->n_head, a->n_slot, a->norm_eps, scale);
    if (T < 0 || n_seq < 0 || n_seq > QMAG_KV_MAX_SEQ) return fail(QMAG_ERR_ARG, "linattn: T=%d n_seq=%d", T, n_seq);
    if ((uintptr_t)a->state % 16 || (a->n_slot && !a->state)) return fail(QMAG_ERR_ARG, "linattn: state is null or not 16-byte aligned");
    if (n_seq > 0 && (!cu || (a->n_slot && !slot) || (((uintptr_t)cu | (uintptr_t)slot | (uintptr_t)len) % 4)))
        return fail(QMAG_ERR_ARG, "linattn: cu or slot is null or unaligned");
    if (((uintptr_t)decay | (uintptr_t)beta) % 4) return fail(QMAG_ERR_ARG, "linattn: decay or beta is not aligned");
    int st;
    if ((st = check_heads("linattn q", q, type, a->dim_k, T, false))) return st;
    if ((st = check_heads("linattn k", k, type, a->dim_k, T, false))) return st;
    if ((st = check_heads("linattn v", v, type, a->dim_v, T, false))) return st;
    if ((st = check_heads("linattn out", out, type, a->dim_v, T, true))) return st;
    if (v->n_head != a->n_head || out->n_head != a->n_head || q->n_head != k->n_head || q->n_head < 1 || a->n_head % q->n_head)
        return fail(QMAG_ERR_ARG, "linattn: %d, %d, %d and %d heads of q, k, v and out for %d", q->n_head, k->n_head, v->n_head,
                    out->n_head, a->n_head);
    const size_t held = sizeof(float) * (size_t)a->n_slot * (size_t)a->n_head * (size_t)a->dim_k * (size_t)a->dim_v;
    const size_t gates = sizeof(float) * (size_t)T * (size_t)a->n_head;
    const struct { const void *p; size_t n; } reads[] = {
        {decay, decay ? gates : 0}, {beta, beta ? gates : 0}, {slot, slot ? sizeof(int) * (size_t)n_seq : 0},
        {len, len ? sizeof(int) * (size_t)n_seq : 0}, {cu, n_seq ? sizeof(int) * ((size_t)n_seq + 1) : 0}};
    const struct { const qmag_heads *h; int dim; } views[] = {{q, a->dim_k}, {k, a->dim_k}, {v, a->dim_v}};
    if (heads_meet(out, size, a->dim_v, T, a->state, held)) return fail(QMAG_ERR_ARG, "linattn: out overlaps the state");
    for (const auto &r : reads)
        if (heads_meet(out, size, a->dim_v, T, r.p, r.n) || ranges_meet(a->state, held, r.p, r.n))
            return fail(QMAG_ERR_ARG, "linattn: out or the state overlaps an input");
    for (const auto &x : views) {
        if (heads_meet(x.h, size, x.dim, T, a->state, held)) return fail(QMAG_ERR_ARG, "linattn: q, k or v overlaps the state");
        if (heads_overlap(out, x.h, size, a->dim_v, T, x.dim)) return fail(QMAG_ERR_ARG, "linattn: out overlaps q, k or v");
    }
    if ((st = require_ready())) return st;
    if (T == 0 || n_seq == 0) return QMAG_OK;

    LaArgs A = {};
    A.q = {q->ptr, q->token_stride, q->head_stride};
    A.k = {k->ptr, k->token_stride, k->head_stride};
    A.v = {v->ptr, v->token_stride, v->head_stride};
    A.out = out->ptr, A.ots = out->token_stride, A.ohs = out->head_stride;
    A.decay = decay, A.beta = beta, A.state = a->state;
    A.slot = a->n_slot ? slot : nullptr, A.len = len, A.cu = cu;
    A.n_head = a->n_head, A.turns = a->turns, A.share = a->turns ? q->n_head : a->n_head / q->n_head;
    A.dim_v = a->dim_v, A.n_slot = a->n_slot, A.n_seq = n_seq, A.T = T;
    A.norm_eps = a->norm_eps, A.scale = scale;
    DeviceScope dev;
    if (dev.st) return dev.st;
    hipStream_t s = ctx().stream;
    const int64_t wgs = ((int64_t)n_seq * a->n_head * (a->dim_v / 16) + LA_WG / 64 - 1) / (LA_WG / 64);
    const unsigned grid = (unsigned)(wgs < 1 << 23 ? wgs : 1 << 23);
    prof_begin(PROF_LINATTN, s);
    with_type(type, [&](auto t) {
        return with_dim_k(a->dim_k, [&](auto d) {
            if (a->delta) linattn_step_kernel<decltype(t), decltype(d)::value, true><<<grid, LA_WG, 0, s>>>(A);
            else linattn_step_kernel<decltype(t), decltype(d)::value, false><<<grid, LA_WG, 0, s>>>(A);
            return 0;
        });
    });
    prof_end(PROF_LINATTN, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}
