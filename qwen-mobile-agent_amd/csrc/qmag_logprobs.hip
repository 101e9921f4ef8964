// qmag_logprobs.hip -- log probabilities of given tokens, the entropy and the most
// likely tokens of rows of logits, beside the sampler, in one pass over the logits.
//
// A thread keeps the largest value m it has met, s = sum e^(x - m) and
// t = sum e^(x - m) (x - m), moved to a new m as s' = s c, t' = c (t + s (m - m')),
// c = e^(m - m'); threads, waves and parts of a row join the same way.  Then
//   ln sum e^x = m + ln s,   entropy = ln s - t / s.
// A thread adds its values in groups of eight, and keeps what a sum's rounding
// leaves: beside a token that stands out the others are each less than half a step
// of the sum, and a thousand of them count (1e-6 of a row's result without).
// Where the most likely tokens are asked for, a wave keeps the 64 best keys (a
// value's order above its complemented place, so that no two are equal) sorted, one
// to a lane; of a tile of values those above the k-th best wait in LDS (few after the
// first tiles: a random row of n has about k ln(n / k)), and k that wait are sorted
// and merged in.
//
// A row is one workgroup's, or, where there are few, several workgroups' and joined
// by a second launch.
//
// Bound by vector instructions where there are many rows: 1024 of 151936 bf16 logits with
// the best token take 87 us, in which a SIMD has 39000 of them, 16.4 a value, 156000 of
// 219000 cycles at four each and more for the exponentials; 311 MB of logits at 3.6 TB/s
// are half of what a streaming read reaches (6.4).  One row, fp32,
// 20 tokens: 7.2 us and 7.3 for the join, sorts of 64 keys one after another in both;
// 77 rows of 32003 fp16, 5 tokens: 12.8 and 5.0.
#include <float.h>

#include "qmag_rows.h"
#include "qmag_wavesort.h"

namespace qmag {

constexpr int LP_WG = 256, LP_WAVES = LP_WG / 64;
constexpr int LP_PER = 8;                        // values of a thread in a tile
constexpr int LP_TILE = 64 * LP_PER;             // a wave's tile
constexpr int LP_AHEAD = 4;                      // tiles asked for ahead (8: 92 us for 1024 rows against 87)
constexpr int LP_ROOM = 64 + LP_TILE;           // keys that wait: fewer than k ahead of a tile, all of its values

struct LpArgs {
    const void *x;
    int64_t stride;
    const int *token;
    float *logprob, *entropy, *top_logprob;
    int *top_id;
    float *stat;             // parts: [T][parts][4] m, s, t
    uint64_t *keys;          // [T][parts][64]
    int n_vocab, T, top_k, parts, part_len;
};

constexpr uint32_t LP_KEY_NONE = 0x007FFFFFu;    // samp_key(-inf)
constexpr float LOG2E = 1.44269504088896340736f;

// the largest of three; not as fmaxf has it where one is a NaN, which then costs an instruction for each operand
__device__ __forceinline__ float lp_max(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

struct LpSum {
    float m, s, t, rs, rt;            // rs, rt: what s and t are above their sums
    __device__ void clear() { m = -FLT_MAX, s = 0.0f, t = 0.0f, rs = 0.0f, rt = 0.0f; }
    __device__ void add(float es, float et)
    {
        const float ys = es - rs, yt = et - rt, ns = s + ys, nt = t + yt;
        rs = (ns - s) - ys;
        rt = (nt - t) - yt;
        s = ns;
        t = nt;
    }
    // to a maximum of at least m: a sum of nothing stays one
    __device__ void move(float to)
    {
        const float d = fmaxf(m - to, -200.0f), c = __builtin_amdgcn_exp2f(d * LOG2E);
        t = s == 0.0f ? 0.0f : c * fmaf(s, d, t);
        rt = s == 0.0f ? 0.0f : c * fmaf(rs, d, rt);
        s *= c;
        rs *= c;
        m = to;
    }
    __device__ void join(float m2, float s2, float t2)
    {
        LpSum o;
        o.clear();
        o.m = m2, o.s = s2, o.t = t2;
        const float to = fmaxf(m, m2);
        move(to);
        o.move(to);
        s += o.s;
        t += o.t;
    }
};

__device__ __forceinline__ LpSum lp_wave_join(LpSum a)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const float m = __uint_as_float(xor_lane(__float_as_uint(a.m), d)), s = __uint_as_float(xor_lane(__float_as_uint(a.s), d)),
                    t = __uint_as_float(xor_lane(__float_as_uint(a.t), d));
        a.join(m, s, t);
    }
    return a;
}

// keys sorted descending and others ascending: the 64 largest of both, descending
__device__ __forceinline__ uint64_t lp_merge(uint64_t best, uint64_t ascending)
{
    return wave_clean64(best > ascending ? best : ascending);
}

// a wave's best keys
struct LpTop {
    uint64_t best;        // one to a lane, descending
    float bound;          // the k-th best value
    bool full;            // there are k numbers: what is not above the bound is none of the best
    int n;                // keys waiting in LDS
    __device__ void clear() { best = 0, bound = 0.0f, full = false, n = 0; }
    // the last of those that wait, up to 64 of them
    __device__ void take(const uint64_t *wait, int k)
    {
        const int from = max(n - 64, 0);
        __builtin_amdgcn_wave_barrier();
        const uint64_t v = from + lane_id() < n ? wait[from + lane_id()] : 0ull;
        __builtin_amdgcn_wave_barrier();
        best = lp_merge(best, ~wave_sort64(~v));
        n = from;
        const uint64_t kth = readlane64(best, k - 1);
        full = (uint32_t)(kth >> 32) > 1u;           // 0: no key, 1: NaN
        bound = samp_value(kth);
    }
    // What of a tile may be among the best, hi being the lane's largest value in it: values above the bound, or,
    // while there is none, keys from the k-th best of the lanes' largest on (k lanes hold one of that size).  It holds
    // for the whole tile, whose values do not come in the order of their places.
    // (odd: a NaN among the lane's values, which may be its largest)
    __device__ bool filter(float hi, bool odd, int k, uint32_t *from) const
    {
        if (full) {
            *from = 0;
            return __ballot(hi > bound || odd) != 0;
        }
        *from = (uint32_t)__builtin_amdgcn_readlane((int)wave_sort64_u32(samp_key(hi)), k - 1);
        if (*from <= LP_KEY_NONE) *from = 0;             // a lane's largest may be no value of the row
        return true;
    }
    // a value of each lane joins those that wait
    __device__ __forceinline__ void add(float v, int id, bool in, bool first, uint32_t from, uint64_t *wait)
    {
        const uint32_t key = samp_key(v);
        const uint64_t who = __ballot(in && (first ? key >= from : v > bound));
        const int at = __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
        if ((who >> lane_id()) & 1u) wait[n + at] = samp_comp(key, id, v);
        n += __popcll(who);
    }
};

// The results of a row from its sums, by one wave; key: its best keys, one to a lane.
template <class T>
__device__ __forceinline__ void lp_finish(const LpArgs &A, int64_t row, LpSum a, uint64_t key)
{
    const int lane = lane_id();
    const float nan = __builtin_nanf("");
    // a NaN among the sums is one among the logits, or an infinite maximum
    const bool ok = a.s > 0.0f && a.m < INFINITY;
    const float ln = logf(a.s);
    if (lane == 0 && A.logprob) {
        const int tok = A.token[row];
        float lp = 0.0f;
        if (tok >= 0 && tok < A.n_vocab) lp = ok ? (T::up(((const typename T::S *)A.x)[row * A.stride + tok]) - a.m) - ln : nan;
        A.logprob[row] = lp;
    }
    if (lane == 0 && A.entropy) A.entropy[row] = ok ? fmaxf(ln - a.t / a.s, 0.0f) : nan;
    if (lane < A.top_k) {
        A.top_id[row * A.top_k + lane] = samp_id(key);
        A.top_logprob[row * A.top_k + lane] = ok ? (samp_value(key) - a.m) - ln : nan;
    }
}

// a thread's values of a tile as they are read
template <class T>
struct LpRaw {
    static constexpr int N = LP_PER * (int)sizeof(typename T::S) / 16, PER = LP_PER / N;
    uint4 r[N];
    __device__ __forceinline__ void load(const typename T::S *p)
    {
#pragma unroll
        for (int i = 0; i < N; i++) r[i] = ld16((const uint8_t *)(p + i * PER));
    }
    // (what is made of them is not moved up to where they were asked for, which would wait for them there)
    __device__ __forceinline__ void get(float (&v)[LP_PER])
    {
#pragma unroll
        for (int i = 0; i < N; i++) {
            asm volatile("" : "+v"(r[i].x), "+v"(r[i].y), "+v"(r[i].z), "+v"(r[i].w));
            union { uint4 u; typename T::S s[PER]; } x;
            x.u = r[i];
#pragma unroll
            for (int e = 0; e < PER; e++) v[i * PER + e] = T::up(x.s[e]);
        }
    }
};

template <class T, bool TOP>
__global__ void __launch_bounds__(LP_WG) logprobs_kernel(LpArgs A)
{
    using S = typename T::S;
    __shared__ uint64_t s_wait[TOP ? LP_WAVES : 1][LP_ROOM];
    __shared__ float s_sum[LP_WAVES][3];
    const int lane = lane_id(), w = threadIdx.x >> 6;
    uint64_t *wait = s_wait[TOP ? w : 0];
    for (int64_t job = blockIdx.x; job < (int64_t)A.T * A.parts; job += gridDim.x) {
        const int64_t row = job / A.parts;
        const int part = (int)(job - row * A.parts);
        const int v0 = part * A.part_len, v1 = (int)min((int64_t)v0 + A.part_len, (int64_t)A.n_vocab);
        const S *x = (const S *)A.x + row * A.stride;
        LpSum a;
        a.clear();
        LpTop top;
        top.clear();
        auto tile = [&](const float (&v)[LP_PER], int64_t i0) {
            const float hi = lp_max(lp_max(v[0], v[1], v[2]), lp_max(v[3], v[4], v[5]), lp_max(v[6], v[7], v[7]));
            if (hi > a.m) a.move(hi);
            float es = 0.0f, et = 0.0f;
#pragma unroll
            for (int i = 0; i < LP_PER; i++) {
                const float d = v[i] - a.m, e = __builtin_amdgcn_exp2f(d * LOG2E);
                es += e;                                              // a NaN stays
                et = fmaf(e, fmaxf(d, -200.0f), et);
            }
            a.add(es, et);
            if constexpr (TOP) {
                uint32_t from;
                const bool first = !top.full;
                if (top.filter(hi, es != es, A.top_k, &from)) {
#pragma unroll
                    for (int i = 0; i < LP_PER; i++) top.add(v[i], (int)(i0 + i), i0 + i < v1, first, from, wait);
                    // (as many as are asked for move the bound; waiting for 64 lets half of all tiles through at k = 1)
                    while (top.n >= A.top_k || (first && top.n > 0)) top.take(wait, A.top_k);
                }
            }
        };
        // whole tiles, several asked for ahead: a CU's share of the memory is some 16 KB for each microsecond of a load
        const int64_t w0 = (int64_t)v0 + w * LP_TILE;
        const int whole = v1 - w0 >= LP_TILE ? (int)((v1 - w0 - LP_TILE) / (LP_WAVES * LP_TILE)) + 1 : 0;
        constexpr int64_t STEP = LP_WAVES * LP_TILE;
        LpRaw<T> raw[LP_AHEAD];
        const S *from = x + w0 + lane * LP_PER;
        const int groups = whole / LP_AHEAD * LP_AHEAD;
        if (groups > 0) {
#pragma unroll
            for (int u = 0; u < LP_AHEAD; u++) raw[u].load(from + u * STEP);
            for (int k = 0; k < groups; k += LP_AHEAD) {
#pragma unroll
                for (int u = 0; u < LP_AHEAD; u++) {
                    float v[LP_PER];
                    raw[u].get(v);
                    raw[u].load(from + min(k + u + LP_AHEAD, whole - 1) * STEP);
                    tile(v, w0 + (k + u) * STEP + lane * LP_PER);
                }
            }
        }
        for (int k = groups; k < whole; k++) {
            float v[LP_PER];
            raw[0].load(from + k * STEP);
            raw[0].get(v);
            tile(v, w0 + k * STEP + lane * LP_PER);
        }
        const int64_t rest = w0 + whole * STEP;
        if (rest < v1) {
            const int64_t i0 = rest + lane * LP_PER;
            float v[LP_PER];
#pragma unroll
            for (int i = 0; i < LP_PER; i++) v[i] = i0 + i < v1 ? T::up(x[i0 + i]) : -INFINITY;
            tile(v, i0);
        }
        if constexpr (TOP) {
            if (top.n > 0) top.take(wait, A.top_k);
            wait[lane] = top.best;
        }
        a = lp_wave_join(a);
        if (lane == 0) s_sum[w][0] = a.m, s_sum[w][1] = a.s, s_sum[w][2] = a.t;
        __syncthreads();
        if (w == 0) {
#pragma unroll
            for (int o = 1; o < LP_WAVES; o++) a.join(s_sum[o][0], s_sum[o][1], s_sum[o][2]);
            uint64_t key = top.best;
            if constexpr (TOP)
                for (int o = 1; o < LP_WAVES; o++) key = lp_merge(key, s_wait[o][63 - lane]);
            if (A.parts == 1) {
                lp_finish<T>(A, row, a, key);
            } else {
                if (lane == 0) {
                    float *st = A.stat + job * 4;
                    st[0] = a.m, st[1] = a.s, st[2] = a.t;
                }
                if constexpr (TOP) A.keys[job * 64 + lane] = key;
            }
        }
        __syncthreads();                 // the next job's sums
    }
}

// Parts of a row: a wave takes every 16th, four asked for at once, then the waves' results in pairs.
constexpr int LP_JOIN = 1024, LP_JOINERS = LP_JOIN / 64;
template <class T, bool TOP>
__global__ void __launch_bounds__(LP_JOIN) logprobs_join_kernel(LpArgs A)
{
    __shared__ uint64_t s_key[TOP ? LP_JOINERS : 1][64];
    __shared__ float s_sum[LP_JOINERS][3];
    const int lane = lane_id(), w = threadIdx.x >> 6;
    for (int64_t row = blockIdx.x; row < A.T; row += gridDim.x) {
        LpSum a;
        a.clear();
        uint64_t key = 0;
        for (int p = w + LP_JOINERS * lane; p < A.parts; p += LP_JOIN) {
            const float *st = A.stat + (row * A.parts + p) * 4;
            a.join(st[0], st[1], st[2]);
        }
        if constexpr (TOP) {
            for (int p = w; p < A.parts; p += 4 * LP_JOINERS) {
                uint64_t k[4];
#pragma unroll
                for (int u = 0; u < 4; u++)
                    k[u] = p + u * LP_JOINERS < A.parts ? A.keys[(row * A.parts + p + u * LP_JOINERS) * 64 + 63 - lane] : 0ull;
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (p + u * LP_JOINERS < A.parts) key = lp_merge(key, k[u]);
            }
            s_key[w][lane] = key;
        }
        a = lp_wave_join(a);
        if (lane == 0) s_sum[w][0] = a.m, s_sum[w][1] = a.s, s_sum[w][2] = a.t;
        __syncthreads();
        if constexpr (TOP) {
#pragma unroll
            for (int half = LP_JOINERS / 2; half > 0; half >>= 1) {
                if (w < half && w + half < A.parts) {
                    key = lp_merge(key, s_key[w + half][63 - lane]);
                    s_key[w][lane] = key;
                }
                if (half > 1) __syncthreads();
            }
        }
        if (w == 0) {
            LpSum b;
            b.clear();
            if (lane < LP_JOINERS) b.m = s_sum[lane][0], b.s = s_sum[lane][1], b.t = s_sum[lane][2];
            lp_finish<T>(A, row, lp_wave_join(b), key);
        }
        __syncthreads();
    }
}

}  // namespace qmag

using namespace qmag;

extern "C" int qmag_logprobs_dev(int n_vocab, int type, const void *logits, int64_t stride, const int *token, int T,
                                 int top_k, float *logprob, float *entropy, int *top_id, float *top_logprob)
{
    const int size = attn_type_size(type);
    if (!size) return fail(QMAG_ERR_ARG, "logprobs: type %d", type);
    if (n_vocab < 1 || T < 0 || top_k < 0 || top_k > QMAG_LOGPROBS_MAX_TOP || top_k > n_vocab)
        return fail(QMAG_ERR_ARG, "logprobs: n_vocab=%d T=%d top_k=%d", n_vocab, T, top_k);
    if (((uintptr_t)token | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_id | (uintptr_t)top_logprob) % 4)
        return fail(QMAG_ERR_ARG, "logprobs: an unaligned pointer");
    if (T > 0 && ((logprob && !token) || (top_k > 0 && (!top_id || !top_logprob))))
        return fail(QMAG_ERR_ARG, "logprobs: logprob without token, or top_k=%d without its results", top_k);
    const qmag_heads hx = {(void *)logits, 1, stride, 0};
    int st = check_heads("logprobs logits", &hx, type, n_vocab, T, false);
    if (st) return st;
    const size_t n = sizeof(float) * (size_t)T;
    const struct { const void *p; size_t n; } out[] = {{logprob, logprob ? n : 0}, {entropy, entropy ? n : 0},
                                                       {top_id, n * (size_t)top_k}, {top_logprob, n * (size_t)top_k}};
    for (int i = 0; i < 4; i++) {
        if (heads_meet(&hx, size, n_vocab, T, out[i].p, out[i].n) || ranges_meet(out[i].p, out[i].n, token, logprob ? n : 0))
            return fail(QMAG_ERR_ARG, "logprobs: a result overlaps an input");
        for (int j = 0; j < i; j++)
            if (ranges_meet(out[i].p, out[i].n, out[j].p, out[j].n)) return fail(QMAG_ERR_ARG, "logprobs: results overlap");
    }
    if ((st = require_ready())) return st;
    if (T == 0 || (!logprob && !entropy && top_k == 0)) return QMAG_OK;

    LpArgs A = {logits, stride, token, logprob, entropy, top_logprob, top_id, nullptr, nullptr, n_vocab, T, top_k, 1, n_vocab};
    // rows in parts while there are fewer than 1024 of them (2048: 102 us and 16 for the join, for 1024 rows, against 87),
    // parts of 2048 values and more
    const int64_t want = (1024 + (int64_t)T - 1) / T, fit = ((int64_t)n_vocab + LP_WAVES * LP_TILE - 1) / (LP_WAVES * LP_TILE);
    A.parts = (int)(want < fit ? want : fit);
    if (A.parts > 1) {
        const int64_t tiles = (fit + A.parts - 1) / A.parts;
        A.part_len = (int)(tiles * LP_WAVES * LP_TILE);
        A.parts = (int)((fit + tiles - 1) / tiles);
    }
    DeviceScope dev;
    if (dev.st) return dev.st;
    hipStream_t s = ctx().stream;
    if (A.parts > 1) {
        const size_t jobs = (size_t)T * (size_t)A.parts;
        uint8_t *p = (uint8_t *)workspace(WS_LOGPROBS, jobs * (16 + (top_k ? 512 : 0)), &st);
        if (st) return st;
        A.keys = (uint64_t *)p;
        A.stat = (float *)(p + jobs * (top_k ? 512 : 0));
    }
    const int64_t jobs = (int64_t)T * A.parts, most = 1 << 23;
    const unsigned grid = (unsigned)(jobs < most ? jobs : most), rows = (unsigned)(T < most ? T : most);
    prof_begin(PROF_LOGPROBS, s);
    with_type(type, [&](auto t) {
        using TT = decltype(t);
        if (top_k) logprobs_kernel<TT, true><<<grid, LP_WG, 0, s>>>(A);
        else logprobs_kernel<TT, false><<<grid, LP_WG, 0, s>>>(A);
        if (A.parts > 1 && top_k) logprobs_join_kernel<TT, true><<<rows, LP_JOIN, 0, s>>>(A);
        else if (A.parts > 1) logprobs_join_kernel<TT, false><<<rows, LP_JOIN, 0, s>>>(A);
        return 0;
    });
    prof_end(PROF_LOGPROBS, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}
