// qmag_attn_kv4.hip -- attention of a sequence's newest tokens over its paged
// 4-bit cache (the role of attn_worker over kvq records, src/nn.c:1215-1453).
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - max),
//   k_t = d_t code_t + m_t per 64 channels, v_t alike.
//
// The codes go to the matrix cores as fp16 whole numbers: a nibble below the
// exponent of 1024 (or, from the upper half of a byte, of 64) is that number plus
// the code, and one subtraction for two values leaves code - 8.  No code is
// rounded, and no step or minimum touches the operand.  The 8 keeps the two sums
// below small: with codes from 0 to 15 they were each tens of times the result,
// which cost a digit (1e-5 of the result against 1e-6).  (The nibble alone is an
// fp16 subnormal, two instructions less for four values, but the matrix cores
// align subnormal products as if their leading zeros were digits: the sums came
// out 10 bits short, 3e-4 of the result.)
//   scores   S = K Q^T per 64 channels on codes, then d S + (m + 8 d) sum(q) in fp32;
//   output   O^T = V^T P'^T with P' = p d: the step of a token and group is
//            folded into the softmax weight, the rest adds sum_t p (m + 8 d).
// q and P' are fp16 after an exact scaling by a power of two; fp32 calls split
// them into two fp16 parts (22 bits), 16-bit calls take one (11 bits, no less
// than the type itself holds).
//
// S^T comes out of v_mfma_f32_16x16x32_f16 with a lane holding one query row and
// the tokens 4 h .. 4 h + 3 of each 16 (h = lane / 16), which is just what the
// second product wants as its operand when V's tokens are taken in that order:
// neither scores nor weights ever cross lanes, and the loop uses no LDS.
//
// Rows are the queries of the heads that share a kv head.  The work is (kv head,
// sequence, group of rows, chunk of the cache); every workgroup finds its own
// from the lengths on the device.  The chunk is the same for all sequences, so
// that a long one among short ones is spread over the chip; partial results of
// split sequences are joined by a second launch.
#include "qmag_attn.h"

namespace qmag {

constexpr int AK_WG = 256;

struct AkArgs {
    const uint8_t *data;
    const int *table, *cu, *len;
    const void *q;
    void *out;
    int64_t qt, qh, ot, oh;               // strides of a token and of a head
    float *part, *ml;                     // partial outputs [n_kv][max_items][RG][D], their (max, sum)
    int64_t half;
    int n_seq, max_blocks, shift, n_block, n_kv, G, T;
    int max_items, target;                // items of a kv head: at most; aimed at
    int min_chunk;                        // 0: sequences are not split
    float scale;                          // times log2 e
    int q_vec, o_vec;
};

// What a workgroup finds about its sequence.
struct AkPlan {
    int seq, q0, nq, len;                 // its rows of q, its tokens in the cache
    int chunk, n_split, item0;            // its first item
};

__device__ __forceinline__ void ak_seq(const AkArgs &A, int i, int *q0, int *nq, int *len)
{
    const int a = min(max(A.cu[i], 0), A.T), b = min(max(A.cu[i + 1], 0), A.T);
    *q0 = a;
    *nq = max(b - a, 0);
    *len = min(max(A.len[i], 0), A.max_blocks << A.shift);
}

__device__ __forceinline__ int ak_groups(const AkArgs &A, int nq, int RG)
{
    return (int)(((int64_t)nq * A.G + RG - 1) / RG);
}

// The sequence of item `want` (by_token: of row `want` of q), found by the
// calling wave alone.  False if there is none.
template <int RG, int STEP>
__device__ __forceinline__ bool ak_find(const AkArgs &A, int want, bool by_token, AkPlan *P)
{
    const int lane = lane_id();
    unsigned long long cost = 0;
    int q0, nq, len;
    P->chunk = 1 << 30;                            // no sequence is longer
    if (A.min_chunk) {
        for (int i = lane; i < A.n_seq; i += 64) {
            ak_seq(A, i, &q0, &nq, &len);
            cost += (unsigned long long)ak_groups(A, nq, RG) * (unsigned)len;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) cost += __shfl_xor(cost, d);
        const unsigned long long c = (cost + A.target - 1) / (unsigned)A.target;
        const unsigned long long r = (max(c, (unsigned long long)A.min_chunk) + STEP - 1) / STEP * STEP;
        P->chunk = (int)min(r, 1ull << 30);
    }
    long long items = 0;
    for (int base = 0; base < A.n_seq; base += 64) {
        const int i = base + lane;
        q0 = nq = len = 0;
        if (i < A.n_seq) ak_seq(A, i, &q0, &nq, &len);
        const int split = max(1, (int)(((unsigned)len + (unsigned)P->chunk - 1u) / (unsigned)P->chunk));
        const long long mine = (long long)ak_groups(A, nq, RG) * split;
        long long incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const long long v = __shfl_up(incl, d);
            if (lane >= d) incl += v;
        }
        const bool here = by_token ? want >= q0 && want < q0 + nq : want < items + incl;
        const unsigned long long hit = __ballot(here);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            P->seq = base + at;
            P->q0 = __builtin_amdgcn_readlane(q0, at);
            P->nq = __builtin_amdgcn_readlane(nq, at);
            P->len = __builtin_amdgcn_readlane(len, at);
            P->n_split = __builtin_amdgcn_readlane(split, at);
            // lengths that overlap make more items than there are workgroups
            if (items + __shfl(incl, at) > A.max_items && by_token) return false;
            P->item0 = (int)(items + __shfl(incl - mine, at));
            return true;
        }
        items += __shfl(incl, 63);
    }
    return false;
}

// max and sum over the four lanes that hold a row
__device__ __forceinline__ float row_max(float v)
{
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ int row_max_i(int v)
{
    auto p = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = max((int)p[0], (int)p[1]);
    p = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    return max((int)p[0], (int)p[1]);
}
__device__ __forceinline__ float row_sum(float v)
{
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

union Frag {
    uint32_t u[4];
    half8 h;
};

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Nibbles 0 and 4 of w (of each half dword), or 1 and 5, less 8, as fp16.
__device__ __forceinline__ uint32_t even_codes(uint32_t w)
{
    const half2v v = __builtin_bit_cast(half2v, (w & 0x000F000Fu) | 0x64006400u) - (half2v){(_Float16)1032.0f, (_Float16)1032.0f};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t odd_codes(uint32_t w)
{
    const half2v v = __builtin_bit_cast(half2v, (w & 0x00F000F0u) | 0x54005400u) - (half2v){(_Float16)72.0f, (_Float16)72.0f};
    return __builtin_bit_cast(uint32_t, v);
}

// Eight nibbles as eight fp16 values, in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ half8 k_frag(uint32_t w)
{
    Frag f;
    f.u[0] = even_codes(w);
    f.u[1] = odd_codes(w);
    f.u[2] = even_codes(w >> 8);
    f.u[3] = odd_codes(w >> 8);
    return f.h;
}

// d, and m + 8 d, the value of code 8
__device__ __forceinline__ float step_of(uint32_t dm) { return h2f(dm & 0xFFFFu); }
__device__ __forceinline__ float mid_of(uint32_t dm) { return fmaf(8.0f, h2f(dm & 0xFFFFu), h2f(dm >> 16)); }

// (hi, lo) fp16 parts of eight values; NS == 1: hi alone, to nearest
template <int NS>
__device__ __forceinline__ void split8(const float (&x)[8], half8 *hi, half8 *lo)
{
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = NS == 2 ? rounded(x[i]) : x[i];
        (*hi)[i] = (_Float16)v;
        if constexpr (NS == 2) (*lo)[i] = (_Float16)(v - (float)(*hi)[i]);
    }
}

// N dwords from p, in loads of up to 16 bytes (p is aligned to them)
template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t *p, uint32_t (&o)[N])
{
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *(const uint4 *)(p + 4 * i);
            o[i] = v.x, o[i + 1] = v.y, o[i + 2] = v.z, o[i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = *(const uint2 *)p;
        o[0] = v.x, o[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = *(const uint32_t *)(p + 4 * i);
    }
}

// SPLITW: the four waves take the tiles of a chunk in turn for the same 16
// rows and join at the end; otherwise each has 16 rows of its own.
template <class T, int D, bool SPLITW>
__global__ void __launch_bounds__(AK_WG, 2) attn_kv4_kernel(AkArgs A)
{
    using S = typename T::S;
    constexpr int NS = sizeof(S) == 4 ? 2 : 1;
    constexpr int NG = D / 64;
    constexpr int RG = SPLITW ? 16 : 64;
    constexpr int VD = (D + 127) / 128;            // dwords of a lane's V codes of a token
    constexpr int LROW = D + 4;                    // LDS row of the join
    __shared__ float join[SPLITW ? 4 * 16 * LROW : 1];
    __shared__ float join_m[4][16], join_l[4][16];

    const int kvh = blockIdx.y, item = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = lane_id(), n = lane & 15, h = lane >> 4;
    AkPlan P;
    if (!ak_find<RG, SPLITW ? 128 : 32>(A, item, false, &P)) return;
    const int local = item - P.item0, split = local % P.n_split, group = local / P.n_split;
    const int rows = P.nq * A.G;
    const int r0 = group * RG + (SPLITW ? 0 : wave * 16);
    if (!SPLITW && r0 >= rows) return;

    // ---- queries
    const int row = r0 + n, j = min(row, rows - 1) / A.G, gh = min(row, rows - 1) - j * A.G;
    const bool live = row < rows;
    half8 qh[NG][2], ql[NS == 2 ? NG : 1][2];
    float qs[NG], rs;
    {
        const S *qp = (const S *)A.q + (P.q0 + j) * A.qt + (kvh * A.G + gh) * A.qh;
        float x[NG][2][8], top = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                load8<T>(qp + g * 64 + s * 32 + h * 8, A.q_vec, x[g][s]);
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[g][s][i]));
            }
        // the row's largest value to 2^14 .. 2^15: exact, and undone by rs
        const int e = min(max((int)(__float_as_uint(row_max(top)) >> 23) - 127, -100), 127);
        const float up = exp2i(14 - e);
        rs = exp2i(e - 14) * A.scale;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float sum = 0.0f;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[g][s][i] *= up;
                    sum += x[g][s][i];
                    f[2 * (i & 3) + (i >> 2)] = x[g][s][i];         // nibble i's place in a fragment
                }
                split8<NS>(f, &qh[g][s], &ql[NS == 2 ? g : 0][s]);
            }
            qs[g] = row_sum(sum);
        }
    }

    // ---- the range of tokens
    const int past = P.len - P.nq;                 // tokens before the first query's own
    const int lim = live ? past + j : INT32_MAX;   // the last token the row sees
    const int j_last = (min(r0 + 16, rows) - 1) / A.G, open = past + r0 / A.G;
    int c0 = split * P.chunk;
    const int c1 = min(min(P.len, c0 + P.chunk), past + j_last + 1);
    if (SPLITW) c0 += 32 * wave;
    constexpr int STEP = SPLITW ? 128 : 32;
    const int *table = A.table + P.seq * (int64_t)A.max_blocks;
    const int64_t block_stride = 2 * A.half * A.n_kv;
    const uint8_t *head = A.data + kvh * 2 * A.half;
    const int64_t codes = (int64_t)(D / 2) << A.shift;

    f32x4 o[NG][4];
    float vs[NG], l = 0.0f, m = -INFINITY;
    int ve = -1;                                   // the row's weights carry 2^(21 - ve)
#pragma unroll
    for (int g = 0; g < NG; g++) {
        vs[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) o[g][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (int t0 = c0; t0 < c1; t0 += STEP) {
        // two halves of 16 tokens, each within one block
        const uint8_t *kb[2];
        bool there[2];
        int off[2];
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const int t = t0 + 16 * a;
            const int id = table[min(t >> A.shift, A.max_blocks - 1)];
            there[a] = id >= 0 && id < A.n_block;
            kb[a] = head + (there[a] ? id : 0) * block_stride;
            off[a] = t & ((1 << A.shift) - 1);
        }
        uint32_t kc[2][D / 32], kdm[8][NG], vdm[8][NG], vc[8][VD];
#pragma unroll
        for (int a = 0; a < 2; a++) load_dwords(kb[a] + (off[a] + n) * (D / 2) + h * (D / 8), kc[a]);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int a = i >> 2, tk = off[a] + 4 * h + (i & 3);
            load_dwords(kb[a] + codes + tk * (NG * 4), kdm[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int a = i >> 2, tk = off[a] + 4 * h + (i & 3);
            const uint8_t *vb = kb[a] + A.half;
            if constexpr (D == 64) vc[i][0] = *(const uint16_t *)(vb + tk * (D / 2) + n * 2);
            else load_dwords(vb + tk * (D / 2) + n * (D / 32), vc[i]);
            load_dwords(vb + codes + tk * (NG * 4), vdm[i]);
        }

        // ---- scores
        float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int g = 0; g < NG; g++) {
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    const half8 kf = k_frag(kc[a][2 * g + st]);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[g][st], acc, 0, 0, 0);
                    if constexpr (NS == 2) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[g][st], acc, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float d = step_of(kdm[4 * a + r][g]), mid = mid_of(kdm[4 * a + r][g]);
                    s[4 * a + r] = fmaf(d, acc[r], fmaf(mid, qs[g], s[4 * a + r]));
                }
            }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] *= rs;
        if (!there[0] || !there[1] || t0 + 31 > open) {
            // a token the row does not see has no weight, whatever the cache holds there
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int a = i >> 2, tk = t0 + 16 * a + 4 * h + (i & 3);
                const bool seen = tk <= lim && tk < c1 && there[a];
                s[i] = seen ? s[i] : -INFINITY;
#pragma unroll
                for (int g = 0; g < NG; g++) vdm[i][g] = seen ? vdm[i][g] : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, s[i]);
        top = row_max(top);

        // ---- running maximum: moved only when a weight would pass 2^8
        if (__any(top > m + 8.0f)) {
            const float mn = fmaxf(m, top);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                vs[g] *= f;
#pragma unroll
                for (int i = 0; i < 4; i++) o[g][i] *= f;
            }
        }
        const float ms = m == -INFINITY ? 0.0f : m;
        // ---- the largest step the row has seen sets the power of two of its weights
        typedef short s16x2 __attribute__((ext_vector_type(2)));
        s16x2 dt = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int g = 0; g < NG; g++) dt = __builtin_elementwise_max(dt, __builtin_bit_cast(s16x2, vdm[i][g]));
        const int de = row_max_i(min((int)dt[0] >> 10, 30));
        if (__any(de > ve)) {
            const int en = max(de, ve);
            const float f = ve < 0 ? 0.0f : exp2i(ve - en);
            ve = en;
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[g][i] *= f;
        }
        const float pf = exp2i(21 - ve);
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[i] = __builtin_amdgcn_exp2f(s[i] - ms);
            l += p[i];
        }

        // ---- output
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = p[i] * pf * step_of(vdm[i][g]);
                vs[g] = fmaf(p[i], mid_of(vdm[i][g]), vs[g]);
            }
            half8 ph, pl;
            split8<NS>(x, &ph, &pl);
#pragma unroll
            for (int b = 0; b < 2; b++) {
                // byte b of group g: channels 4 n + 2 b and the next of every token
                Frag even, odd;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int at = 2 * (g & 1) + b;
                    const uint32_t w = __builtin_amdgcn_perm(vc[2 * k + 1][g >> 1], vc[2 * k][g >> 1],
                                                             0x0C040C00u + 0x00010001u * (uint32_t)at);
                    even.u[k] = even_codes(w);
                    odd.u[k] = odd_codes(w);
                }
                o[g][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even.h, ph, o[g][2 * b], 0, 0, 0);
                o[g][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd.h, ph, o[g][2 * b + 1], 0, 0, 0);
                if constexpr (NS == 2) {
                    o[g][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even.h, pl, o[g][2 * b], 0, 0, 0);
                    o[g][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd.h, pl, o[g][2 * b + 1], 0, 0, 0);
                }
            }
        }
    }

    // ---- a lane's row: channels 64 g + 4 (4 h + r) + i in o[g][i][r]
    l = row_sum(l);
    const float back = exp2i(max(ve, 0) - 21);
    float y[NG][4][4];                             // [g][r][i]
    float scale_w = 1.0f;
    if constexpr (SPLITW) {
        if (h == 0) {
            join_m[wave][n] = m;
            join_l[wave][n] = l;
        }
        __syncthreads();
        float all = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; w++) all = fmaxf(all, join_m[w][n]);
        scale_w = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - all);
        // a NaN weight leaves m at -inf: let it through
        if (m == -INFINITY && l != 0.0f) scale_w = l;
    }
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const float add = row_sum(vs[g]);
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                y[g][r][i] = fmaf(o[g][i][r], back, add) * scale_w;
    }
    const int64_t slot = ((int64_t)kvh * A.max_items + item) * RG;
    if constexpr (SPLITW) {
        float *mine = join + (wave * 16 + n) * LROW;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(float4 *)(mine + 64 * g + 4 * (4 * h + r)) = make_float4(y[g][r][0], y[g][r][1], y[g][r][2], y[g][r][3]);
        __syncthreads();
        // 16 threads a row, four channels at a time
        const int rr = threadIdx.x >> 4, cc = threadIdx.x & 15;
        if (r0 + rr >= rows) return;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) M = fmaxf(M, join_m[w][rr]);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float mw = join_m[w][rr], lw = join_l[w][rr];
            L += mw == -INFINITY ? (lw != 0.0f ? lw : 0.0f) : lw * __builtin_amdgcn_exp2f(mw - M);
        }
        const int jj = (r0 + rr) / A.G, hh = r0 + rr - jj * A.G;
        S *op = (S *)A.out + (P.q0 + jj) * A.ot + (kvh * A.G + hh) * A.oh;
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int c = 0; c < D; c += 64) {
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float4 f = *(const float4 *)(join + (w * 16 + rr) * LROW + c + 4 * cc);
                v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
            }
            if (P.n_split == 1) {
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] *= inv;
                store4<T>(op + c + 4 * cc, A.o_vec, v);
            } else {
                store4<TF32>(A.part + (slot + rr) * D + c + 4 * cc, true, v);
            }
        }
        if (P.n_split > 1 && cc == 0) {
            A.ml[2 * (slot + rr)] = M;
            A.ml[2 * (slot + rr) + 1] = L;
        }
    } else {
        if (!live) return;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        S *op = (S *)A.out + (P.q0 + j) * A.ot + (kvh * A.G + gh) * A.oh;
        const int64_t at = slot + wave * 16 + n;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int c = 64 * g + 4 * (4 * h + r);
                if (P.n_split == 1) {
#pragma unroll
                    for (int i = 0; i < 4; i++) y[g][r][i] *= inv;
                    store4<T>(op + c, A.o_vec, y[g][r]);
                } else {
                    store4<TF32>(A.part + at * D + c, true, y[g][r]);
                }
            }
        if (P.n_split > 1 && h == 0) {
            A.ml[2 * at] = m;
            A.ml[2 * at + 1] = l;
        }
    }
}

// Joins the partial results of the rows whose sequence was split: a workgroup
// for a head of a token, its waves the parts in turn.
template <class T, int D, int RG, int STEP>
__global__ void __launch_bounds__(AK_WG) attn_kv4_join_kernel(AkArgs A)
{
    using S = typename T::S;
    constexpr int C = D / 64;                       // channels of a lane
    __shared__ float sum[4][D], sl[4];
    const int t = blockIdx.x, head = blockIdx.y, kvh = head / A.G, gh = head - kvh * A.G;
    const int wave = threadIdx.x >> 6, lane = lane_id();
    AkPlan P;
    if (!ak_find<RG, STEP>(A, t, true, &P) || P.n_split == 1) return;
    const int row = (t - P.q0) * A.G + gh;
    const int64_t first = ((int64_t)kvh * A.max_items + P.item0 + row / RG * P.n_split) * RG + row % RG;
    float M = -INFINITY;
    for (int i = lane; i < P.n_split; i += 64) M = fmaxf(M, A.ml[2 * (first + (int64_t)i * RG)]);
    M = group_max<64>(M);
    float acc[C], L = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c++) acc[c] = 0.0f;
#pragma unroll 4
    for (int i = wave; i < P.n_split; i += 4) {
        const int64_t at = first + (int64_t)i * RG;
        const float mi = A.ml[2 * at], li = A.ml[2 * at + 1];
        const float f = mi == -INFINITY ? (li != 0.0f ? li : 0.0f) : __builtin_amdgcn_exp2f(mi - M);
        L += mi == -INFINITY ? f : f * li;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const float v = A.part[at * D + 64 * c + lane];
            // a part without a token seen: nothing was summed there
            acc[c] += f == 0.0f ? 0.0f : f * v;
        }
    }
#pragma unroll
    for (int c = 0; c < C; c++) sum[wave][64 * c + lane] = acc[c];
    if (lane == 0) sl[wave] = L;
    __syncthreads();
    L = sl[0] + sl[1] + sl[2] + sl[3];
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    S *op = (S *)A.out + t * A.ot + head * A.oh;
    for (int c = threadIdx.x; c < D; c += AK_WG) op[c] = T::down((sum[0][c] + sum[1][c] + sum[2][c] + sum[3][c]) * inv);
}

template <class T, int D, bool SPLITW>
static int ak_launch(AkArgs A, hipStream_t s)
{
    constexpr int RG = SPLITW ? 16 : 64, STEP = SPLITW ? 128 : 32;
    // Row groups at most; two workgroups for every CU are aimed at.
    const int64_t groups = (int64_t)A.T * A.G / RG + A.n_seq;
    const int64_t goal = 2 * (int64_t)ctx().n_cu;
    A.target = (int)((goal + A.n_kv - 1) / A.n_kv);
    // enough row groups to fill the chip twice over: nothing is split
    A.min_chunk = ((int64_t)A.T * A.G / RG) * A.n_kv >= 2 * goal ? 0 : 256;
    const int64_t items = groups + (A.min_chunk ? A.target : 0);
    if (items > INT32_MAX / AK_WG) return fail(QMAG_ERR_ARG, "attn_kv4: %lld groups of rows", (long long)items);
    A.max_items = (int)items;
    if (A.min_chunk) {
        int st;
        const size_t rows = (size_t)A.n_kv * A.max_items * RG;
        A.part = (float *)workspace(WS_ATTN, rows * (D + 2) * sizeof(float), &st);
        if (st) return st;
        A.ml = A.part + rows * D;
    }
    attn_kv4_kernel<T, D, SPLITW><<<dim3((unsigned)items, (unsigned)A.n_kv), AK_WG, 0, s>>>(A);
    if (A.min_chunk)
        attn_kv4_join_kernel<T, D, RG, STEP><<<dim3((unsigned)A.T, (unsigned)(A.n_kv * A.G)), AK_WG, 0, s>>>(A);
    return QMAG_OK;
}

template <class T, int D>
static int ak_pick(const AkArgs &A, hipStream_t s)
{
    // few rows to a sequence: the waves share them and split the tokens
    if ((int64_t)A.T * A.G <= 32 * (int64_t)A.n_seq) return ak_launch<T, D, true>(A, s);
    return ak_launch<T, D, false>(A, s);
}

}  // namespace qmag

using namespace qmag;

extern "C" int qmag_attn_kv4_dev(const qmag_kv4 *c, const qmag_kv_table *t, int type, const qmag_heads *q,
                                 const qmag_heads *out, const int *cu, const int *len, int T, float scale)
{
    int st = check_kv4(c);
    if (st) return st;
    if (!t || !q || !out) return fail(QMAG_ERR_ARG, "attn_kv4: null pointer");
    if (T < 0 || T > QMAG_ATTN_MAX_TOKENS || t->n_seq < 0 || t->n_seq > QMAG_KV_MAX_SEQ)
        return fail(QMAG_ERR_ARG, "attn_kv4: T=%d n_seq=%d", T, t->n_seq);
    if (t->block_size != c->block_size || t->n_block != c->n_block)
        return fail(QMAG_ERR_ARG, "attn_kv4: a table of %d blocks of %d for a cache of %d of %d", t->n_block, t->block_size,
                    c->n_block, c->block_size);
    if ((st = check_heads("attn_kv4 q", q, type, c->head_dim, T, false))) return st;
    if ((st = check_heads("attn_kv4 out", out, type, c->head_dim, T, true))) return st;
    if (q->n_head < 1 || q->n_head != out->n_head || q->n_head % c->n_kv)
        return fail(QMAG_ERR_ARG, "attn_kv4: %d query and %d output heads over %d kv heads", q->n_head, out->n_head, c->n_kv);
    if (t->max_blocks < 1 || (int64_t)t->max_blocks * t->block_size > 1 << 30)
        return fail(QMAG_ERR_ARG, "attn_kv4: rows of %d blocks of %d tokens", t->max_blocks, t->block_size);
    if (T > 0 && t->n_seq > 0 && (!cu || !len || !t->table || ((uintptr_t)cu | (uintptr_t)len | (uintptr_t)t->table) % 4))
        return fail(QMAG_ERR_ARG, "attn_kv4: a null or unaligned pointer");
    if (heads_overlap(q, out, attn_type_size(type), c->head_dim, T))
        return fail(QMAG_ERR_ARG, "attn_kv4: the output overlaps the queries");
    if ((st = require_ready())) return st;
    if (T == 0 || t->n_seq == 0) return QMAG_OK;
    DeviceScope dev;
    if (dev.st) return dev.st;
    AkArgs A = {};
    A.data = (const uint8_t *)c->data;
    A.table = t->table;
    A.cu = cu;
    A.len = len;
    A.q = q->ptr;
    A.out = out->ptr;
    A.qt = q->token_stride, A.qh = q->head_stride, A.ot = out->token_stride, A.oh = out->head_stride;
    A.half = kv4_half_bytes(c->block_size, c->head_dim);
    A.n_seq = t->n_seq;
    A.max_blocks = t->max_blocks;
    while ((1 << A.shift) < c->block_size) A.shift++;
    A.n_block = c->n_block;
    A.n_kv = c->n_kv;
    A.G = q->n_head / c->n_kv;
    A.T = T;
    A.scale = scale * 1.44269504088896340736f;
    A.q_vec = heads_aligned(q, type);
    A.o_vec = heads_aligned(out, type);
    hipStream_t s = ctx().stream;
    prof_begin(PROF_ATTN, s);
    st = with_type(type, [&](auto ty) {
        using TT = decltype(ty);
        if (c->head_dim == 64) return ak_pick<TT, 64>(A, s);
        if (c->head_dim == 128) return ak_pick<TT, 128>(A, s);
        return ak_pick<TT, 256>(A, s);
    });
    prof_end(PROF_ATTN, s);
    if (st) return st;
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}
