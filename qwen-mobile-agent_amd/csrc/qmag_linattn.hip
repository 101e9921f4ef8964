// qmag_linattn.hip -- linear attention with a decay for each head, plain or by the
// delta rule (the role of gdn_worker, src/nn.c:784), one state S [dim_k][dim_v] a head
// and sequence.  A token, as a recurrence:
//
//   S <- a S;  u = b (v - delta S^T k);  S <- S + k u^T;  o = scale S^T q,  a = e^g
//
// The columns of S have nothing to do with one another.  Two forms:
//
// Token by token (la_recurrence).  A wave takes 16 columns: lane l rows
// (l % 16) dim_k / 16 .. of columns 4 (l / 16) .., all in registers for as many tokens
// as there are.  With S0 the state ahead of a token,
//   S^T q = a S0^T q + (k . q) u,
// so that both of a token's products with the state are formed from S0, side by side,
// and one exchange over 16 lanes sums them.
//
// In chunks of 64 tokens, for prompts.  With G the sums of g from a chunk's start and S0
// the state ahead of it,
//   (I + L) U = b (V - e^G K S0),  L_ij = b_i (k_i . k_j) e^(G_i - G_j), j < i  (delta)
//   O = scale (e^G Q S0 + P U),    P_ij = (q_i . k_j) e^(G_i - G_j), j <= i
//   S1 = e^G_63 S0 + sum_j e^(G_63 - G_j) k_j u_j^T.
// P and (I + L)^-1 do not depend on the state: a first kernel forms them for all chunks
// at once, a second walks down each sequence's chunks, 16 columns of a head to a
// workgroup.  Sums of g are held in 64 bits, since their differences count.
//
// Products are the bf16 matrix cores': an fp32 operand is three bf16 parts (24 bits, the
// range of fp32; fp16 values are two exactly, bf16 ones one), and of the products of
// parts those are formed whose places add up to less than three (2^-24 of the operands).
// An accumulator holds four rows of a column in a lane, which is half of what the next
// product's operand holds of 32 rows.  Products over tokens take their 32 terms in the
// order [4 g .. 4 g + 3, 16 + 4 g ..] for lane group g, products over channels a group's
// eight side by side, the state's rows being laid out for it: neither moves between lanes.
//
// What they are bound by (32 heads over 16 key heads, 128 channels both):
//   a token each of 96 sequences, bf16: 89 us for 403 MB of states, 4.5 TB/s, memory.
//   one token of one sequence: 5.3 us; 61 tokens of 13 sequences: 16.2.  Some 0.7 us a
//   token for two sums over 16 lanes and what hangs on them; where the chip is full, 250
//   instructions for each token and wave.  Not kept: more tokens asked for ahead and
//   normalised early (registers for three waves where four were: 96 sequences 118 us),
//   half the columns a wave (18.7 us for the 61 tokens), a quarter (27).
//   prompts, fp32, 4096 tokens: 54 us for all chunks' matrices, 179 MB written and read
//   back, and 183 for the walk, 64 chunks in a row of 2.9 us: three products of 6 pairs
//   of parts that wait for one another through LDS, with a barrier after each.
//   8192 tokens of 7 prompts, bf16: 65 and 237 us, the chip full of chunks of two
//   workgroups to a CU at 3.7 us each (two parts of what a 16-bit result is made of: 206).
//   Not kept in the walk, at 200 us for fp32 and 245 for bf16: operands by transfers
//   straight to LDS, by 4 waves more (227, 325); Q and K split into parts there (244, 395).
#include <float.h>
#include <math.h>

#include "qmag_rows.h"
#include "qmag_linattn_plan.h"

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
    int n_head, n_key, share, turns, dim_v, n_slot, n_seq, T;
    float norm_eps, scale;
    // the chunked form
    int r0, r1;               // the window's rows
    int n_tile, n_long, brief;
    uint8_t *keys, *heads;    // what chunks have for each key head, and for each head
    int *left;                // [n_tile][n_head][dim_v / 16] of a sequence's first chunk: the first row the walk did not do
    const float *carry_in;    // [n_head][dim_k][dim_v]: the state of a sequence begun ahead of the window
    float *carry_out;
};

// the key head of a head, and the i-th head of a key head
__device__ __forceinline__ int la_key_of(const LaArgs &A, int head) { return A.turns ? head % A.n_key : head / A.share; }
__device__ __forceinline__ int la_head_of(const LaArgs &A, int key, int i) { return A.turns ? key + i * A.n_key : key * A.share + i; }

// e^g: at most 1, nothing left of what a fp32 weight does not hold; a NaN stays
__device__ __forceinline__ float la_decay(float g)
{
    return g > 0.0f ? 1.0f : expf(g);
}

__device__ __forceinline__ int la_one(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Where a sequence's state comes from and goes to, at row 0 and column 0 of a head; null: nowhere.
struct LaState {
    const float *from;
    float *to;
};
__device__ __forceinline__ LaState la_state(const LaArgs &A, int seq, int head, int dim_k, bool begun, bool goes_on)
{
    const int64_t size = (int64_t)dim_k * A.dim_v;
    const int slot = A.slot ? la_one(ldg(A.slot + seq)) : -1, behind = A.len ? la_one(ldg(A.len + seq)) : 1;
    float *own = slot >= 0 && slot < A.n_slot ? A.state + ((int64_t)slot * A.n_head + head) * size : nullptr;
    LaState s;
    s.from = begun ? A.carry_in + head * size : own && behind > 0 ? own : nullptr;
    s.to = goes_on ? A.carry_out + head * size : own;
    return s;
}

template <int N>
struct LaToken {
    float k[N], q[N], v[4], a, b;
};

// n rows from `first` on, one after another, of one head and 16 columns, by one wave.  The
// first `quiet` rows' results are there already.
template <class T, int DK, bool DELTA>
__device__ void la_recurrence(const LaArgs &A, int head, int c0, int first, int n, int quiet, LaState st)
{
    using S = typename T::S;
    constexpr int N = DK / 16;
    const int lane = lane_id(), rg = lane & 15, col = c0 + 4 * (lane >> 4);
    const int kh = la_key_of(A, head);
    float s[N][4];
#pragma unroll
    for (int r = 0; r < N; r++) {
        if (st.from) {
            load_row<TF32, 4>(st.from + (int64_t)(rg * N + r) * A.dim_v + col, s[r]);
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) s[r][c] = 0.0f;
        }
    }
    const S *kp = (const S *)A.k.p + first * A.k.ts + kh * A.k.hs + rg * N;
    const S *qp = (const S *)A.q.p + first * A.q.ts + kh * A.q.hs + rg * N;
    const S *vp = (const S *)A.v.p + first * A.v.ts + head * A.v.hs + col;
    S *op = (S *)A.out + first * A.ots + head * A.ohs + col;
    const float *gp = A.decay ? A.decay + (int64_t)first * A.n_head + head : nullptr;
    const float *bp = A.beta ? A.beta + (int64_t)first * A.n_head + head : nullptr;
    auto load = [&](int t, LaToken<N> &x) {
        load_row<T, N>(kp + t * A.k.ts, x.k);
        load_row<T, N>(qp + t * A.q.ts, x.q);
        load_row<T, 4>(vp + t * A.v.ts, x.v);
        x.a = gp ? ldg(gp + (int64_t)t * A.n_head) : 0.0f;
        x.b = bp ? ldg(bp + (int64_t)t * A.n_head) : 1.0f;
    };
    LaToken<N> x;
    load(0, x);
    for (int t = 0; t < n; t++) {
        LaToken<N> next;
        load(min(t + 1, n - 1), next);
        if (A.norm_eps > 0.0f) {
            // ahead of the products: a large key's would leave fp32's range
            float kk = 0.0f, qq = 0.0f;
            auto squares = [&]() {
                kk = qq = 0.0f;
#pragma unroll
                for (int r = 0; r < N; r++) {
                    kk = fmaf(x.k[r], x.k[r], kk);
                    qq = fmaf(x.q[r], x.q[r], qq);
                }
                kk = group_sum<16>(kk);
                qq = group_sum<16>(qq);
            };
            squares();
            float ek = A.norm_eps, eq = A.norm_eps;
            if (__ballot(!(kk + qq <= FLT_MAX))) {
                // a row whose squares do so themselves is taken times 2^-70, and its eps with it
                const float fk = kk <= FLT_MAX ? 1.0f : 0x1p-70f, fq = qq <= FLT_MAX ? 1.0f : 0x1p-70f;
#pragma unroll
                for (int r = 0; r < N; r++) x.k[r] *= fk, x.q[r] *= fq;
                ek = ek * fk * fk;
                eq = eq * fq * fq;
                squares();
            }
            const float rk = rsqrtf(kk + ek), rq = rsqrtf(qq + eq);
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
        if (rg == 0 && t >= quiet) store_row<T, 4>(op + t * A.ots, o);
        x = next;
    }
    if (st.to) {
#pragma unroll
        for (int r = 0; r < N; r++) store_row<TF32, 4>(st.to + (int64_t)(rg * N + r) * A.dim_v + col, s[r]);
    }
}

// ------------------------------------------------------------ in chunks --

// bf16 parts of a value of the type; what is formed of them is fp32, three parts, for results of any type: a 16-bit one
// is rounded once, from what the recurrence in fp32 has.
template <class T> constexpr int LA_PARTS = 3;
template <> constexpr int LA_PARTS<TF16> = 2;
template <> constexpr int LA_PARTS<TBF16> = 1;

// What the chunks' products hold; anything else goes token by token, from the row that has it or, for a state, the chunk
// ahead of which it has grown so.  K and Q are multiplied as they are read, their norms' inverses come after, so that
//   K S, Q S          |k| |s| sqrt(dim_k) <= 2^(40 + 80 + 4)
// is what stays in fp32's range by the least.  With k', q' the keys and queries that the formula has (normalised or not),
// and b |k'|^2 <= 2.01 for the delta rule, whose b |k'| is then 2^10.5 at most, and whose state so at most doubles in a chunk:
//   U                 b (|v| + |k'| |S|) <= 2^96 (2^60 without the delta rule); its terms in T X 64 times 2^97
//   u_j |k'_j|        2^86 (2^80), and as much is added to the state; divided by |k_j|, as it meets K, 2^116
//   P U               64 scale |q'| 2^86 <= 2^122
// and none of it is above 2^124.  From the smallest k', q' and scale on P's third part is above bf16's smallest, 2^-133.
constexpr float LA_MOST_ROW = 0x1p80f;           // |k|^2, |q|^2 as they are read
constexpr float LA_MOST_KEY = 0x1p40f, LA_LEAST_KEY = 0x1p-80f;      // |k'|^2, |q'|^2 that are not 0
constexpr float LA_LEAST_ROW = 0x1p-60f;         // with the norm, |k|^2 and |q|^2 that are not 0: squares lose digits
constexpr float LA_MOST_BETA = 0x1p20f, LA_MOST_V = 0x1p40f, LA_MOST_STATE = 0x1p80f;
constexpr float LA_MOST_SCALE = 0x1p10f, LA_LEAST_SCALE = 0x1p-30f;

// Operands lie in the workspace as the matrix cores take them: 64 lanes of 16 bytes.
constexpr int LA_FRAG = 1024;
constexpr int LA_TRI = 6;             // operands of a lower triangle: 16 rows by 32 columns, those all above it left out
constexpr int la_tri(int rt, int tb) { return rt < 2 ? rt : 2 * rt - 2 + tb; }
// What a chunk has for each key head: the parts of K, rows of whole 16 bytes whose places are exchanged so that 16 rows'
// lie in different banks, and of Q as operands, [16 rows: 4][DK / 32][parts].
template <class T, int DK>
struct LaKeys {
    static constexpr int K = 0, PLANE = 64 * DK * 2, Q = LA_PARTS<T> * PLANE, BYTES = 2 * Q;
    static_assert(BYTES == la_key_bytes(LA_PARTS<T>, DK));
};
// Where 16 bytes of a row of K lie, in 16 bytes: 16 rows' of one piece in different banks, and so four rows' of four
// pieces side by side, which a transposing read takes.
template <int DK>
__host__ __device__ constexpr int la_place(int row, int piece)
{
    return piece ^ (DK == 64 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3));
}
// What a chunk has for each head: (I + L)^-1 and P [LA_TRI][parts], then rows of 64 that the chunk's tokens are
// multiplied by.
struct LaLayout {
    static constexpr int TI = 0, P = LA_TRI * 3 * LA_FRAG, VEC = P + LA_TRI * 3 * LA_FRAG, QD = VEC + 1024;
    static constexpr int KD = 0, KE = 64, B = 128, END = 192, BAD = 193;     // floats of VEC; END: e^G_63; BAD: the first row the form does not hold, 64: none
    static constexpr int HEAD_BYTES = QD + 256;
};
static_assert(LaLayout::HEAD_BYTES == LA_HEAD_BYTES);

// x as N parts, the first the nearest bf16 to it, each other to what those ahead leave
template <int N, int V>
__device__ __forceinline__ void la_split(const float (&x)[V], __bf16 (&o)[N][V])
{
#pragma unroll
    for (int i = 0; i < V; i++) {
        float r = x[i];
#pragma unroll
        for (int p = 0; p < N; p++) {
            o[p][i] = (__bf16)r;
            r -= (float)o[p][i];
        }
    }
}
template <int N>
__device__ __forceinline__ void la_split8(const float (&x)[8], bf168 (&o)[N])
{
    __bf16 s[N][8];
    la_split<N, 8>(x, s);
#pragma unroll
    for (int p = 0; p < N; p++)
#pragma unroll
        for (int i = 0; i < 8; i++) o[p][i] = s[p][i];
}

// c += a b, of the products of parts those of places adding up to less than three, the smallest first
template <int NA, int NB>
__device__ __forceinline__ void la_mac(const bf168 (&a)[NA], const bf168 (&b)[NB], f32x4 &c)
{
#pragma unroll
    for (int places = 2; places >= 0; places--)
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int j = places - i;
            if (j >= 0 && j < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], c, 0, 0, 0);
        }
}

template <int N>
__device__ __forceinline__ void la_load(const uint8_t *p, bf168 (&o)[N])
{
    const uint32_t at = (uint32_t)lane_id() * 16;
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = *(const QMAG_GLOBAL bf168 *)(p + i * LA_FRAG + at);
}
template <int N>
__device__ __forceinline__ void la_store(uint8_t *p, const bf168 (&x)[N])
{
    const int at = lane_id() * 16;
#pragma unroll
    for (int i = 0; i < N; i++) *(QMAG_GLOBAL bf168 *)(p + i * LA_FRAG + at) = x[i];
}

// sums over the four lanes of a column (or row)
__device__ __forceinline__ float la_sum4(float v)
{
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// A wave looks for long sequences: of chunk number j the sequence (-1: none), its rows and which of its chunks.
struct LaTile {
    LaRows rows;
    int chunk;
    bool any;
};
__device__ LaTile la_find(const LaArgs &A, int j)
{
    const int lane = lane_id();
    int rank = 0;
    for (int s0 = 0; s0 < A.n_seq; s0 += 64) {
        const int i = s0 + lane;
        LaRows x = {0, 0, false, false};
        if (i < A.n_seq) x = la_rows(ldg(A.cu + i), ldg(A.cu + i + 1), A.T, A.r0, A.r1);
        const uint64_t is_long = __ballot(la_long(x.n, A.brief));
        const int tile0 = la_tile0(x.first, A.r0, rank + __popcll(is_long & ((1ull << lane) - 1)));
        const uint64_t hit = __ballot(la_long(x.n, A.brief) && j >= tile0 && j < tile0 + seq_tiles(x.n, LA_SHIFT));
        if (hit) {
            const int at = __ffsll((unsigned long long)hit) - 1;
            x.first = __builtin_amdgcn_readlane(x.first, at);
            x.n = __builtin_amdgcn_readlane(x.n, at);
            return {x, j - __builtin_amdgcn_readlane(tile0, at), true};
        }
        rank += __popcll(is_long);
    }
    return {{0, 0, false, false}, 0, false};
}
// how many long sequences are ahead of one
__device__ int la_rank(const LaArgs &A, int seq)
{
    const int lane = lane_id();
    int rank = 0;
    for (int s0 = 0; s0 < seq; s0 += 64) {
        const int i = s0 + lane;
        bool is_long = false;
        if (i < seq) is_long = la_long(la_rows(ldg(A.cu + i), ldg(A.cu + i + 1), A.T, A.r0, A.r1).n, A.brief);
        rank += __popcll(__ballot(is_long));
    }
    return rank;
}
// the long sequence that has `rank` ahead of it; -1: none
__device__ int la_ranked(const LaArgs &A, int rank)
{
    const int lane = lane_id();
    for (int s0 = 0; s0 < A.n_seq; s0 += 64) {
        const int i = s0 + lane;
        bool is_long = false;
        if (i < A.n_seq) is_long = la_long(la_rows(ldg(A.cu + i), ldg(A.cu + i + 1), A.T, A.r0, A.r1).n, A.brief);
        uint64_t m = __ballot(is_long);
        const int n = __popcll(m);
        if (rank < n) {
            for (; rank > 0; rank--) m &= m - 1;
            return s0 + __ffsll((unsigned long long)m) - 1;
        }
        rank -= n;
    }
    return -1;
}

// Token by token: whole calls, or what the walk down a window's chunks leaves, sequences of few rows and those with
// values that its products do not hold, from their first row on.
template <class T, int DK, bool DELTA, bool REST>
__global__ void __launch_bounds__(LA_WG) linattn_step_kernel(LaArgs A)
{
    const uint32_t slices = (uint32_t)A.dim_v / 16, jobs = (uint32_t)A.n_seq * (uint32_t)A.n_head * slices;
    for (uint32_t j = blockIdx.x * (LA_WG / 64) + (uint32_t)la_one(threadIdx.x >> 6); j < jobs; j += gridDim.x * (LA_WG / 64)) {
        const uint32_t sh = j / slices;
        const int seq = (int)(sh / (uint32_t)A.n_head), head = (int)(sh % (uint32_t)A.n_head), c0 = (int)(j % slices) * 16;
        const LaRows rows = la_rows(la_one(ldg(A.cu + seq)), la_one(ldg(A.cu + seq + 1)), A.T, A.r0, A.r1);
        if (rows.n <= 0) continue;
        int quiet = 0;
        if (REST && la_long(rows.n, A.brief)) {
            const int rank = la_rank(A, seq), tile0 = la_tile0(rows.first, A.r0, rank);
            if (la_room(rank, tile0, seq_tiles(rows.n, LA_SHIFT), A.n_long, A.n_tile)) quiet = ldg(A.left + ((int64_t)tile0 * A.n_head + head) * slices + c0 / 16);
            if (quiet < 0) continue;
        }
        la_recurrence<T, DK, DELTA>(A, head, c0, rows.first, rows.n, quiet, la_state(A, seq, head, DK, rows.begun, rows.goes_on));
    }
}

// What a chunk of a key head and its heads has that does not depend on the state: a wave takes 16 of the chunk's rows.
// 54 us for 4096 tokens of 16 key heads and 32 heads in fp32, 96 KB of K and Q and twice 37 KB of matrices for each chunk
// and key head: 179 MB written and 64 read, 4.5 TB/s, the memory's rate.
// Products of rows j with rows i leave lane group g with j = 4 g .. of a row i: as P and the inverse are operands.
constexpr double LOG2E = 1.4426950408889634;
__device__ __forceinline__ float la_power(double x) { return __builtin_amdgcn_exp2f((float)x); }

// workgroups to a CU, as many as their LDS leaves, three at most: more than two waves to a SIMD take fewer registers than
// the compiler would (8192 tokens bf16, three: 146 registers, two: 159, which leave three workgroups their places too and
// take as long, 65 us; with more than 168 they took 72)
template <class T, int DK>
constexpr int LA_CHUNK_WGS = 160 * 1024 / (LA_PARTS<T> * 128 * (DK + 8) + 28 * 1024) < 3 ? 160 * 1024 / (LA_PARTS<T> * 128 * (DK + 8) + 28 * 1024) : 3;

template <class T, int DK, bool DELTA>
__global__ void __launch_bounds__(256, (LA_CHUNK_WGS<T, DK>)) linattn_chunk_kernel(LaArgs A)
{
    using S = typename T::S;
    using Y = LaLayout;
    constexpr int NP = LA_PARTS<T>, NKB = DK / 32, ROW = DK + 8;
    __shared__ __attribute__((aligned(16))) __bf16 s_k[NP][64][ROW];
    __shared__ __attribute__((aligned(16))) float s_lt[64][68];           // L, rows and columns exchanged
    __shared__ __attribute__((aligned(16))) float s_dt[4][16][20];        // inverses of its diagonal blocks, exchanged
    __shared__ double s_g[4][64];
    __shared__ float s_fk[64], s_fq[64], s_kk[64], s_b[4][64];
    __shared__ int s_odd[4], s_good[4];
    const int lane = lane_id(), w = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4, g4 = g * 4;
    const int tile = blockIdx.x / A.n_key, key = blockIdx.x % A.n_key;
    const LaTile at = la_find(A, tile);
    if (!at.any) return;
    const int n = min(64, at.rows.n - 64 * at.chunk);
    const int64_t row0 = at.rows.first + 64 * (int64_t)at.chunk;

    uint8_t *mine = A.keys + ((int64_t)tile * A.n_key + key) * LaKeys<T, DK>::BYTES;
    // rows of K and Q as operands, their sums of squares, and the bits that any of their values has
    bf168 kf[NKB][NP], qf[NKB][NP];
    float kk = 0.0f, qq = 0.0f;
    uint32_t kn = 0, qn = 0;
    const int my = 16 * w + l16;
    const S *kp = (const S *)A.k.p + (row0 + min(my, n - 1)) * A.k.ts + key * A.k.hs + 8 * g;
    const S *qp = (const S *)A.q.p + (row0 + min(my, n - 1)) * A.q.ts + key * A.q.hs + 8 * g;
    float kx[NKB][8], qx[NKB][8];
#pragma unroll
    for (int kb = 0; kb < NKB; kb++) {
        load_row<T, 8>(kp + 32 * kb, kx[kb]);
        load_row<T, 8>(qp + 32 * kb, qx[kb]);
    }
#pragma unroll
    for (int kb = 0; kb < NKB; kb++) {
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = my < n ? kx[kb][e] : 0.0f, y[e] = my < n ? qx[kb][e] : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            kk = fmaf(x[e], x[e], kk);
            qq = fmaf(y[e], y[e], qq);
            kn |= __float_as_uint(x[e]);
            qn |= __float_as_uint(y[e]);
        }
        la_split8<NP>(x, kf[kb]);
        la_split8<NP>(y, qf[kb]);
#pragma unroll
        for (int p = 0; p < NP; p++) {
            *(bf168 *)&s_k[p][my][32 * kb + 8 * g] = kf[kb][p];
            *(QMAG_GLOBAL bf168 *)(mine + p * LaKeys<T, DK>::PLANE + my * DK * 2 + la_place<DK>(my, 4 * kb + g) * 16) = kf[kb][p];
        }
        la_store<NP>(mine + LaKeys<T, DK>::Q + (w * NKB + kb) * NP * LA_FRAG, qf[kb]);
    }
    kk = la_sum4(kk);
    qq = la_sum4(qq);
    const bool norm = A.norm_eps > 0.0f;
    // whether the row, which four lanes have, is other than zeros (whose squares' sum is 0 too where they are small)
    constexpr uint64_t ROW_LANES = 0x0001000100010001ull;
    const bool some_k = (__ballot(kn << 1 != 0) >> l16 & ROW_LANES) != 0, some_q = (__ballot(qn << 1 != 0) >> l16 & ROW_LANES) != 0;
    if (lane < 16) {
        // (a key of zeros adds nothing whatever it is multiplied by)
        s_kk[my] = norm ? kk / (kk + A.norm_eps) : kk;
        s_fk[my] = !some_k ? 0.0f : norm ? rsqrtf(kk + A.norm_eps) : 1.0f;
        s_fq[my] = !some_q ? 0.0f : norm ? rsqrtf(qq + A.norm_eps) : 1.0f;
    }
    // From a row that is not held on the chunk goes token by token; the rows ahead of it are as if there were none behind.
    auto held = [&](float sum, bool some) {
        const float key = norm ? sum / (sum + A.norm_eps) : sum;
        return !some || (sum <= LA_MOST_ROW && (!norm || sum >= LA_LEAST_ROW) && key <= LA_MOST_KEY && key >= LA_LEAST_KEY);
    };
    const uint64_t odd = __ballot(!held(kk, some_k) || !held(qq, some_q));
    if (lane == 0) s_odd[w] = odd ? 16 * w + (__ffsll((unsigned long long)odd) - 1) % 16 : 64;
    __syncthreads();
    const int even = min(min(s_odd[0], s_odd[1]), min(s_odd[2], s_odd[3]));

    f32x4 ck[4], cq[4];
#pragma unroll
    for (int ct = 0; ct < 4; ct++) {
        if (ct > w) continue;
        ck[ct] = cq[ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) {
            bf168 a[NP];
#pragma unroll
            for (int p = 0; p < NP; p++) a[p] = *(const bf168 *)&s_k[p][16 * ct + l16][32 * kb + 8 * g];
            if constexpr (DELTA) la_mac(a, kf[kb], ck[ct]);
            la_mac(a, qf[kb], cq[ct]);
        }
    }
    const int sharing = A.n_head / A.n_key;
    for (int i = 0; i < sharing; i++) {
        // the gates of four heads at once, a wave to each
        if (i % 4 == 0 && i + w < sharing) {
            const int head = la_head_of(A, key, i + w);
            uint8_t *to = A.heads + ((int64_t)tile * A.n_head + head) * Y::HEAD_BYTES;
            float g = 0.0f, b = 0.0f;
            if (lane < n) {
                g = A.decay ? ldg(A.decay + (row0 + lane) * A.n_head + head) : 0.0f;
                b = A.beta ? ldg(A.beta + (row0 + lane) * A.n_head + head) : 1.0f;
            }
            const bool none = g != g;
            g = g > 0.0f ? 0.0f : g < -200.0f ? -200.0f : g;              // e^-200 is 0 in fp32
            double sum = g;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_up(sum, d);
                if (lane >= d) sum += o;
            }
            sum *= LOG2E;
            const double all = __shfl(sum, 63);
            const float bk = b * s_kk[lane];
            // the delta rule grows past b |k|^2 = 2, and its inverse with it
            const bool out = none || !(fabsf(b) <= LA_MOST_BETA) || (DELTA && !(bk >= 0.0f && bk <= 2.01f));
            const uint64_t bad = __ballot(out);
            s_g[w][lane] = sum;
            s_b[w][lane] = b;
            const int good = bad ? min(even, __ffsll((unsigned long long)bad) - 1) : even;
            float *vec = (float *)(to + Y::VEC);
            const float now = la_power(sum), fk = s_fk[lane];
            vec[Y::KD + lane] = now * fk;
            ((float *)(to + Y::QD))[lane] = A.scale * s_fq[lane] * now;
            vec[Y::KE + lane] = la_power(all - sum) * fk;
            vec[Y::B + lane] = b;
            if (lane == 0) {
                vec[Y::END] = la_power(all);
                ((int *)vec)[Y::BAD] = s_good[w] = good;
            }
        }
        if (i % 4 == 0) __syncthreads();
        const int head = la_head_of(A, key, i), gate = i % 4;
        uint8_t *to = A.heads + ((int64_t)tile * A.n_head + head) * Y::HEAD_BYTES;
        const double gi = s_g[gate][my];
        const bool row = my < s_good[gate];
        const float pq = A.scale * s_fq[my], lk = s_b[gate][my] * s_fk[my];
        float pv[4][4];
#pragma unroll
        for (int ct = 0; ct < 4; ct++) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                pv[ct][r] = 0.0f;
                if (ct > w) continue;
                const int j = 16 * ct + g4 + r;
                const float e = s_fk[j] * la_power(gi - s_g[gate][j]);
                pv[ct][r] = row && j <= my ? pq * (cq[ct][r] * e) : 0.0f;
                if constexpr (DELTA) s_lt[j][my] = row && j < my ? lk * (ck[ct][r] * e) : 0.0f;
            }
        }
#pragma unroll
        for (int tb = 0; tb < 2; tb++) {
            if (2 * tb > w) continue;
            float x[8];
            bf168 p[3];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = pv[2 * tb + (e >> 2)][e & 3];
            la_split8<3>(x, p);
            la_store<3>(to + Y::P + la_tri(w, tb) * 3 * LA_FRAG, p);
        }
        if constexpr (DELTA) {
            // the inverse of the wave's diagonal block, a column to a lane (four lanes the same)
            __builtin_amdgcn_wave_barrier();
            float d[16];
#pragma unroll
            for (int r = 0; r < 16; r++) d[r] = r == l16 ? 1.0f : 0.0f;
#pragma unroll
            for (int m = 0; m < 15; m++)
#pragma unroll
                for (int r = m + 1; r < 16; r++) d[r] = fmaf(-s_lt[16 * w + m][16 * w + r], d[m], d[r]);
            if (lane < 16) {
#pragma unroll
                for (int r = 0; r < 16; r += 4) *(f32x4 *)&s_dt[w][l16][r] = f32x4{d[r], d[r + 1], d[r + 2], d[r + 3]};
            }
            __syncthreads();
            // row w of the inverse, from the diagonal on: T_wb = -(sum over c in b + 1 .. w of T_wc L_cb) T_bb
            f32x4 t[4];
#pragma unroll
            for (int b = 3; b >= 0; b--) {
                t[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (b > w) continue;
                if (b == w) {
#pragma unroll
                    for (int r = 0; r < 4; r++) t[b][r] = s_dt[w][g4 + r][l16];
                    continue;
                }
                f32x4 m = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = b + 1; c < 4; c++) {
                    if (c > w) continue;
                    const f32x4 a = *(const f32x4 *)&s_lt[16 * b + l16][16 * c + g4];
#pragma unroll
                    for (int r = 0; r < 4; r++) m = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], t[c][r], m, 0, 0, 0);
                }
                const f32x4 a = *(const f32x4 *)&s_dt[b][l16][g4];
#pragma unroll
                for (int r = 0; r < 4; r++) t[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(-a[r], m[r], t[b], 0, 0, 0);
            }
#pragma unroll
            for (int tb = 0; tb < 2; tb++) {
                if (2 * tb > w) continue;
                float x[8];
                bf168 p[3];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = t[2 * tb + (e >> 2)][e & 3];
                la_split8<3>(x, p);
                la_store<3>(to + Y::TI + la_tri(w, tb) * 3 * LA_FRAG, p);
            }
        }
        __syncthreads();                    // the next head's gates and L
    }
}

// Down a sequence's chunks: one head, 16 columns of the state, by 8 waves.  Waves 0 .. 3 form U and the next state, 16
// of the chunk's rows and a quarter of the state's each; what a wave forms the others take from LDS as operands.  Waves
// 4 .. 7 form the results, and bring LDS what the first four read of a chunk, ahead of them: a CU takes in some 40
// bytes a clock, and a wave that asks for its own operands waits in line with all others.
template <class T, int DK>
struct LaRoom {
    static constexpr int K = LaKeys<T, DK>::Q, REST = DK / 32 * 3 * LA_FRAG + 2 * 9 * LA_FRAG + 5 * LA_FRAG + 64;
    static constexpr int BUFS = 2 * K + REST <= 160 * 1024 ? 2 : 1;      // chunks of K in LDS
    // two workgroups to a CU, where their LDS allows it and half the registers do: each waits most of its time for a
    // product or a move through LDS.  (fp32's three parts of Q and K ahead do not fit 128: 4096 tokens, 32 heads and 64
    // channels 367 us against 165.)
    static constexpr int WGS = sizeof(typename T::S) == 2 && 2 * (2 * K + REST) <= 160 * 1024 ? 2 : 1;
};

// a value as if it were new in every turn of a loop, so that places formed from it are not kept (and then spilled)
__device__ __forceinline__ void la_fresh(uint32_t &v) { asm volatile("" : "+v"(v)); }

template <class T, int DK, bool DELTA>
__global__ void __launch_bounds__(512, (2 * LaRoom<T, DK>::WGS)) linattn_chain_kernel(LaArgs A)
{
    using S = typename T::S;
    using Y = LaLayout;
    using M = LaRoom<T, DK>;
    using X = LaKeys<T, DK>;
    constexpr int NP = LA_PARTS<T>, NKB = DK / 32, BUFS = M::BUFS;
    constexpr int OWN = (NKB + 3) / 4;                    // blocks of 32 rows of the state that a wave holds
    __shared__ __attribute__((aligned(16))) uint8_t s_k[BUFS][X::Q];
    __shared__ __attribute__((aligned(16))) uint8_t s_s[NKB][3][LA_FRAG];
    __shared__ __attribute__((aligned(16))) uint8_t s_x[DELTA ? 2 : 1][3][LA_FRAG], s_u[2][3][LA_FRAG], s_e[2][3][LA_FRAG];
    __shared__ __attribute__((aligned(16))) float s_vec[256], s_v[1024];
    __shared__ __attribute__((aligned(16))) int s_bad[4];         // each wave's first row that the form does not hold, 64: none
    const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4, g4 = g * 4;
    const bool chain = w < 4;
    const int rt = w & 3;
    uint32_t at = lane * 16, half = at + 8 * (rt & 1);
    // workgroups go round the 8 XCDs: the slices of a key head's heads on one of them, a sequence's key heads on all
    const uint32_t slices = (uint32_t)A.dim_v / 16, each = (uint32_t)A.share * slices, units = (uint32_t)A.n_long * (uint32_t)A.n_key;
    for (uint32_t b = blockIdx.x; b < (units + 7) / 8 * 8 * each; b += gridDim.x) {
        const uint32_t unit = (b >> 3) / each * 8 + (b & 7);
        if (unit >= units) continue;
        const int rank = la_one((int)(unit / (uint32_t)A.n_key)), seq = la_one(la_ranked(A, rank));
        if (seq < 0) break;
        const int key = la_one((int)(unit % (uint32_t)A.n_key)), part = la_one((int)((b >> 3) % each));
        const int head = la_head_of(A, key, part / (int)slices), c0 = la_one(part % (int)slices * 16);
        // (what the workgroup has in common in scalar registers, places formed from it too)
        const LaRows rows = la_rows(la_one(ldg(A.cu + seq)), la_one(ldg(A.cu + seq + 1)), A.T, A.r0, A.r1);
        const int chunks = seq_tiles(rows.n, LA_SHIFT), tile0 = la_one(la_tile0(rows.first, A.r0, rank));
        if (!la_room(rank, tile0, chunks, A.n_long, A.n_tile)) continue;
        const LaState st = la_state(A, seq, head, DK, rows.begun, rows.goes_on);
        __syncthreads();                                  // the job before has left LDS
        // a wave's block kb of the state holds rows 32 kb + 8 g + 4 h + r
        f32x4 s[OWN][2];
        bool odd = false;
#pragma unroll
        for (int o = 0; o < OWN; o++) {
            const int kb = rt + 4 * o;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    s[o][h][r] = 0.0f;
                    if (chain && kb < NKB && st.from) s[o][h][r] = ldg(st.from + (int64_t)(32 * kb + 8 * g + 4 * h + r) * A.dim_v + c0 + l16);
                    odd |= !(fabsf(s[o][h][r]) <= LA_MOST_STATE);
                }
        }
        auto publish = [&]() {
#pragma unroll
            for (int o = 0; o < OWN; o++) {
                const int kb = rt + 4 * o;
                if (!chain || kb >= NKB) continue;
                float x[8];
                bf168 p[3];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = s[o][e >> 2][e & 3];
                la_split8<3>(x, p);
#pragma unroll
                for (int i = 0; i < 3; i++) *(bf168 *)&s_s[kb][i][at] = p[i];
            }
        };
        publish();
        int c = 0, upto = 0;                              // the first chunk that is not done, the first such row of it
        bool wide = false;                                // the wave's part of the state is not held any more
        const bool go = !__syncthreads_or(odd);
        auto heads = [&](int i) { return A.heads + ((int64_t)(tile0 + min(i, chunks - 1)) * A.n_head + head) * Y::HEAD_BYTES; };
        auto keys = [&](int i) { return A.keys + ((int64_t)(tile0 + min(i, chunks - 1)) * A.n_key + key) * X::BYTES; };
        // a row of chunk i, or the sequence's last
        auto row_of = [&](int i, int row) { return (int64_t)rows.first + min(64 * i + row, rows.n - 1); };
        if (chain && go) {
            // places in K that differ by more than a constant: a row's blocks, the wave's rows of K^T
            constexpr int KINDS = NKB < 4 ? NKB : 4;
            int row_at[KINDS];
#pragma unroll
            for (int i = 0; i < KINDS; i++) row_at[i] = (16 * rt + l16) * DK * 2 + la_place<DK>(l16, 4 * i + g) * 16;
            bf168 tf[2][3];                               // the wave's rows of the inverse, a chunk ahead
            auto ask_t = [&](int i) {
#pragma unroll
                for (int tb = 0; tb < 2; tb++) la_load<3>(heads(i) + Y::TI + la_tri(rt, rt < 2 ? 0 : tb) * 3 * LA_FRAG, tf[tb]);
            };
            if constexpr (DELTA) ask_t(0);
            const int tok = g4 + (l16 >> 2);
            const int col_at = tok * DK * 2 + la_place<DK>(tok, 4 * min(rt, NKB - 1) + (l16 & 3)) * 16;
            __syncthreads();
            for (; c < chunks; c++) {
                la_fresh(at);
                la_fresh(half);
                const uint8_t *K = s_k[c % BUFS];
                f32x4 acc;
                if constexpr (DELTA) {
                    f32x4 ks[2] = {};
#pragma unroll
                    for (int kb = 0; kb < NKB; kb++) {
                        bf168 a[NP], b[3];
#pragma unroll
                        for (int i = 0; i < 3; i++) b[i] = *(const bf168 *)&s_s[kb][i][at];
#pragma unroll
                        for (int i = 0; i < NP; i++) a[i] = *(const bf168 *)(K + row_at[kb % KINDS] + i * X::PLANE + kb / KINDS * 256);
                        la_mac(a, b, ks[kb & 1]);
                    }
                    acc = ks[0] + ks[1];
                }
                const f32x4 kd = *(const f32x4 *)&s_vec[Y::KD + 16 * rt + g4], bt = *(const f32x4 *)&s_vec[Y::B + 16 * rt + g4],
                            ke = *(const f32x4 *)&s_vec[Y::KE + 16 * rt + g4], v = *(const f32x4 *)&s_v[256 * rt + 4 * lane];
                const float end = s_vec[Y::END];
                const int good = ((const int *)s_vec)[Y::BAD], left = min(rows.n - 64 * c, good);
                float x[4];
                bool odd = good < 64;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    // (b is 0 behind the sequence's end)
                    x[r] = bt[r] * (DELTA ? fmaf(-kd[r], acc[r], v[r]) : v[r]);
                    odd |= !(fabsf(v[r]) <= LA_MOST_V);
                }
                int bad = 64;
                if (__ballot(odd)) {
                    bad = good;
#pragma unroll
                    for (int r = 3; r >= 0; r--) {
                        const int row = 16 * rt + g4 + r;
                        const bool fine = fabsf(v[r]) <= LA_MOST_V;
                        if (row < left && !fine) bad = min(bad, row);
                        if (row >= left || !fine) x[r] = 0.0f;              // not even times 0 in the rows ahead
                    }
                    bad = group_min_i<64>(bad);
                }
                if constexpr (DELTA) {
                    __bf16 p[3][4];
                    la_split<3, 4>(x, p);
#pragma unroll
                    for (int i = 0; i < 3; i++) *(s16x4 *)&s_x[rt >> 1][i][half] = *(const s16x4 *)p[i];
                }
                if (lane == 0) s_bad[rt] = wide ? 0 : bad;            // a chunk from a state that is not held is left out
                if constexpr (DELTA) {
                    __syncthreads();
                    f32x4 us[2] = {};
#pragma unroll
                    for (int tb = 0; tb < 2; tb++) {
                        if (2 * tb > rt) continue;
                        bf168 b[3];
#pragma unroll
                        for (int i = 0; i < 3; i++) b[i] = *(const bf168 *)&s_x[tb][i][at];
                        la_mac(tf[tb], b, us[tb]);
                    }
                    ask_t(c + 1);
                    const f32x4 u = us[0] + us[1];
#pragma unroll
                    for (int r = 0; r < 4; r++) x[r] = u[r];
                }
                {
                    __bf16 p[3][4], pe[3][4];
                    float xe[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) xe[r] = x[r] * ke[r];
                    la_split<3, 4>(x, p);
                    la_split<3, 4>(xe, pe);
#pragma unroll
                    for (int i = 0; i < 3; i++) {
                        *(s16x4 *)&s_u[rt >> 1][i][half] = *(const s16x4 *)p[i];
                        *(s16x4 *)&s_e[rt >> 1][i][half] = *(const s16x4 *)pe[i];
                    }
                }
                __syncthreads();
                upto = min(min(s_bad[0], s_bad[1]), min(s_bad[2], s_bad[3]));
                if (upto < 64) break;
#pragma unroll
                for (int o = 0; o < OWN; o++)
#pragma unroll
                    for (int h = 0; h < 2; h++) s[o][h] *= end;
#pragma unroll
                for (int tb = 0; tb < 2; tb++) {
                    bf168 b[3];
#pragma unroll
                    for (int i = 0; i < 3; i++) b[i] = *(const bf168 *)&s_e[tb][i][at];
#pragma unroll
                    for (int o = 0; o < OWN; o++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            // K^T by transposing reads: 16 lanes take 4 tokens by 4 times 4 channels, and lane n gets
                            // the tokens of the n-th
                            union { s16x4 half[2]; bf168 v; } a[NP];
                            bf168 av[NP];
#pragma unroll
                            for (int i = 0; i < NP; i++) {
#pragma unroll
                                for (int u = 0; u < 2; u++)
                                    a[i].half[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                        (__attribute__((address_space(3))) s16x4 *)(K + col_at + i * X::PLANE + (32 * tb + 16 * u) * DK * 2 + 256 * o + 8 * h));
                                av[i] = a[i].v;
                            }
                            la_mac(av, b, s[o][h]);
                        }
                }
                float most = 0.0f;
#pragma unroll
                for (int o = 0; o < OWN; o++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int r = 0; r < 4; r++) most = fmaxf(most, fabsf(s[o][h][r]));
                wide = __ballot(most > LA_MOST_STATE) != 0;
                publish();
                __syncthreads();
                if constexpr (BUFS == 1) __syncthreads();
            }
        } else if (go) {
            // All that a chunk is taken from is asked for a chunk and more ahead, and goes on to LDS as soon as its
            // place there is free: K beside the last one's, V and what it is multiplied by once the first barrier has
            // passed.
            constexpr int MINE = X::Q / LA_FRAG / 4;
            // (256 fp32 channels: Q where it is used, or registers spill: 2 x 2048 tokens of 4 heads 355 us against 577)
            constexpr bool HOLD = NKB * NP <= 16;
            bf168 qf[NKB][NP], pf[2][3];
            f32x4 qd, kr[MINE], vec;
            float v[4];
            auto ask_q = [&](int i) {
                if (!HOLD) return;
                const uint8_t *p = keys(i) + X::Q + rt * NKB * NP * LA_FRAG;
#pragma unroll
                for (int kb = 0; kb < NKB; kb++) la_load<NP>(p + kb * NP * LA_FRAG, qf[kb]);
            };
            auto ask_p = [&](int i) {
                const uint8_t *p = heads(i);
                qd = *(const QMAG_GLOBAL f32x4 *)(p + Y::QD + 64 * rt + (at >> 8) * 16);
#pragma unroll
                for (int tb = 0; tb < 2; tb++) la_load<3>(p + Y::P + la_tri(rt, rt < 2 ? 0 : tb) * 3 * LA_FRAG, pf[tb]);
            };
            auto ask_k = [&](int i) {
#pragma unroll
                for (int u = 0; u < MINE; u++) kr[u] = *(const QMAG_GLOBAL f32x4 *)(keys(i) + (rt + 4 * u) * LA_FRAG + (uint32_t)at);
            };
            auto put_k = [&](int i) {
#pragma unroll
                for (int u = 0; u < MINE; u++) *(f32x4 *)(s_k[i % BUFS] + (rt + 4 * u) * LA_FRAG + at) = kr[u];
            };
            auto ask_v = [&](int i) {
                const int row = 16 * rt + (int)(at >> 8) * 4, col = (int)(at >> 4) & 15;      // (the lane's, new in every turn)
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] = T::up(*(const QMAG_GLOBAL S *)((const S *)A.v.p + row_of(i, row + r) * A.v.ts + head * A.v.hs + c0 + col));
                vec = *(const QMAG_GLOBAL f32x4 *)(heads(i) + Y::VEC + (uint32_t)at);
            };
            auto put_v = [&]() {
                *(f32x4 *)((uint8_t *)s_v + 1024 * rt + at) = f32x4{v[0], v[1], v[2], v[3]};
                if (rt == 0) *(f32x4 *)((uint8_t *)s_vec + at) = vec;
            };
            ask_k(0);
            ask_v(0);
            ask_q(0);
            ask_p(0);
            put_k(0);
            put_v();
            ask_k(1);
            ask_v(1);
            __syncthreads();
            for (; c < chunks; c++) {
                la_fresh(at);
                f32x4 qs[2] = {};
#pragma unroll
                for (int kb = 0; kb < NKB; kb++) {
                    bf168 b[3];
#pragma unroll
                    for (int i = 0; i < 3; i++) b[i] = *(const bf168 *)&s_s[kb][i][at];
                    if constexpr (!HOLD) la_load<NP>(keys(c) + X::Q + (rt * NKB + kb) * NP * LA_FRAG, qf[kb]);
                    la_mac(qf[kb], b, qs[kb & 1]);
                }
                ask_q(c + 1);
                f32x4 o = (qs[0] + qs[1]) * qd;
                if constexpr (BUFS == 2) {
                    put_k(c + 1);
                    ask_k(c + 2);
                }
                if constexpr (DELTA) {
                    __syncthreads();
                    if constexpr (BUFS == 2) {
                        put_v();
                        ask_v(c + 2);
                    }
                }
                __syncthreads();
                upto = min(min(s_bad[0], s_bad[1]), min(s_bad[2], s_bad[3]));
#pragma unroll
                for (int tb = 0; tb < 2; tb++) {
                    if (2 * tb > rt) continue;
                    bf168 b[3];
#pragma unroll
                    for (int i = 0; i < 3; i++) b[i] = *(const bf168 *)&s_u[tb][i][at];
                    la_mac(pf[tb], b, o);
                }
                ask_p(c + 1);
                if constexpr (!DELTA && BUFS == 2) {
                    put_v();
                    ask_v(c + 2);
                }
                const int t = 64 * c + 16 * rt + (int)(at >> 8) * 4, to = min(rows.n, 64 * c + upto);
                S *p = (S *)A.out + (rows.first + (int64_t)t) * A.ots + head * A.ohs + c0 + ((at >> 4) & 15);
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (t + r < to) p[r * A.ots] = T::down(o[r]);
                if (upto < 64) break;
                __syncthreads();
                if constexpr (BUFS == 1) {
                    put_k(c + 1);
                    put_v();
                    ask_k(c + 2);
                    ask_v(c + 2);
                    __syncthreads();
                }
            }
        }
        // a row with values that the products do not hold, or a state: all is left as it was from there on
        const bool grown = __syncthreads_or(wide);
        if (threadIdx.x == 0) A.left[((int64_t)tile0 * A.n_head + head) * slices + c0 / 16] = c < chunks ? 64 * c + upto : grown ? rows.n : -1;
        if (c >= chunks && !grown && chain && st.to) {
#pragma unroll
            for (int o = 0; o < OWN; o++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (rt + 4 * o < NKB) st.to[(int64_t)(32 * (rt + 4 * o) + 8 * g + 4 * h + r) * A.dim_v + c0 + l16] = s[o][h][r];
        }
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
    A.n_head = a->n_head, A.n_key = q->n_head, A.share = a->n_head / q->n_head, A.turns = a->turns;
    A.dim_v = a->dim_v, A.n_slot = a->n_slot, A.n_seq = n_seq, A.T = T;
    A.norm_eps = a->norm_eps, A.scale = scale, A.r1 = T;
    DeviceScope dev;
    if (dev.st) return dev.st;
    hipStream_t s = ctx().stream;
    const int64_t slices = (int64_t)n_seq * a->n_head * (a->dim_v / 16);
    // prompts in chunks; few tokens to a sequence one after another
    const int parts = with_type(type, [](auto t) { return LA_PARTS<decltype(t)>; });
    A.brief = la_brief(slices, parts);
    const size_t tile = la_tile_bytes(parts, a->dim_k, q->n_head, a->n_head);
    const size_t state = sizeof(float) * (size_t)a->n_head * (size_t)a->dim_k * (size_t)a->dim_v;
    const bool cut = la_cut(T, n_seq, A.brief) && fabsf(scale) >= LA_LEAST_SCALE && fabsf(scale) <= LA_MOST_SCALE;
    const int window = cut ? la_window(T, n_seq, A.brief, tile, state) : 0;
    const bool chunks = window > 0;
    if (chunks) {
        uint8_t *p = (uint8_t *)workspace(WS_LINATTN, la_workspace(window, T, n_seq, A.brief, tile, state), &st);
        if (st) return st;
        A.carry_in = (float *)p;
        A.keys = p + (T > window ? 2 * state : 0);
    }
    prof_begin(PROF_LINATTN, s);
    with_type(type, [&](auto t) {
        return with_dim_k(a->dim_k, [&](auto d) {
            using TT = decltype(t);
            constexpr int DK = decltype(d)::value;
            const int64_t step_wgs = (slices + LA_WG / 64 - 1) / (LA_WG / 64);
            const unsigned steps = (unsigned)(step_wgs < 1 << 23 ? step_wgs : 1 << 23);
            if (!chunks) {
                if (a->delta) linattn_step_kernel<TT, DK, true, false><<<steps, LA_WG, 0, s>>>(A);
                else linattn_step_kernel<TT, DK, false, false><<<steps, LA_WG, 0, s>>>(A);
                return 0;
            }
            float *carry = (float *)A.carry_in;
            for (int64_t r0 = 0, odd = 0; r0 < T; r0 += window, odd ^= 1) {
                A.r0 = (int)r0;
                A.r1 = (int)(r0 + window < T ? r0 + window : T);
                A.n_tile = la_most_tiles(A.r1 - A.r0, n_seq, A.brief);
                A.n_long = la_most_long(A.r1 - A.r0, n_seq, A.brief);
                // (a workgroup that finds no sequence ends: few of them, where none may be long enough)
                const int64_t wgs = ((int64_t)A.n_long * A.n_key + 7) / 8 * 8 * A.share * (a->dim_v / 16);
                const unsigned grid = (unsigned)(wgs < 2048 ? wgs : 2048);
                A.heads = A.keys + (size_t)A.n_tile * (size_t)A.n_key * LaKeys<TT, DK>::BYTES;
                A.left = (int *)(A.heads + (size_t)A.n_tile * (size_t)A.n_head * LaLayout::HEAD_BYTES);
                A.carry_in = carry + (odd ? state / sizeof(float) : 0);
                A.carry_out = carry + (odd ? 0 : state / sizeof(float));
                const unsigned tiles = (unsigned)A.n_tile * (unsigned)A.n_key;
                if (a->delta) {
                    if (grid) {
                        linattn_chunk_kernel<TT, DK, true><<<tiles, 256, 0, s>>>(A);
                        linattn_chain_kernel<TT, DK, true><<<grid, 512, 0, s>>>(A);
                    }
                    linattn_step_kernel<TT, DK, true, true><<<steps, LA_WG, 0, s>>>(A);
                } else {
                    if (grid) {
                        linattn_chunk_kernel<TT, DK, false><<<tiles, 256, 0, s>>>(A);
                        linattn_chain_kernel<TT, DK, false><<<grid, 512, 0, s>>>(A);
                    }
                    linattn_step_kernel<TT, DK, false, true><<<steps, LA_WG, 0, s>>>(A);
                }
            }
            return 0;
        });
    });
    prof_end(PROF_LINATTN, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}
