// qmag_attn_kv4.hip -- attention of a sequence's newest tokens over its paged
// 4-bit cache (the role of attn_worker over kvq records, src/nn.c:1215-1453).
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - max),
//   k_t = d_t code_t + m_t per 64 channels, v_t alike.
//
// The codes go to the matrix cores as fp16 whole numbers: a nibble below the
// exponent of 1024 (or, from the upper half of a byte, of 64) is that number plus
// the code, and one subtraction for two values leaves it.  No code is rounded,
// and no step or minimum touches the operand.  Two ways (Code):
//   CENTRED  fp32 and fp16 calls take code - 8, which keeps the two sums below
//            small: with codes from 0 to 15 they were each tens of times the
//            result, which cost a digit (fp32: 1e-5 of the result against 1e-6;
//            fp16: 3.6e-4 against 2.4e-4, of which its rounding is 2.0e-4);
//   PLAIN    bf16 calls take the code: a digit they do not hold anyway, and the
//            value of code 8 need not be formed.
// (The nibble alone, an fp16 subnormal, would be four instructions fewer for eight
// codes.  But the matrix cores align subnormal products as if their leading zeros
// were digits, which leaves sums of 14 bits: with a few query channels some thousand
// times the others the weights were wrong altogether.)
//   scores   S = K Q^T per 64 channels on codes, then d S + mid sum(q) in fp32,
//            mid the value of the operand 0: m, or m + 8 d;
//   output   O^T = V^T P'^T with P' = p d: the step of a token and group is
//            folded into the softmax weight, the rest adds sum_t p mid.
// q and P' are fp16 after an exact scaling by a power of two; fp32 calls split
// them into two fp16 parts (22 bits), 16-bit calls take one (11 bits, no less
// than the type itself holds).
//
// S^T comes out of v_mfma_f32_16x16x32_f16 with a lane holding one query row and
// the tokens 4 h .. 4 h + 3 of each 16 (h = lane / 16), which is just what the
// second product wants as its operand when V's tokens are taken in that order:
// neither scores nor weights ever cross lanes.
//
// Rows are the queries of the heads that share a kv head.  The work is (kv head,
// sequence, group of rows, chunk of the cache); every workgroup finds its own
// from the lengths on the device.  The chunk is the same for all sequences, so
// that a long one among short ones is spread over the chip; partial results of
// split sequences are joined by a second launch.  Two kernels: up to 256 rows to a
// sequence, and more (ak_pick).
#include <type_traits>

#include "qmag_attn.h"
#include "qmag_attn_plan.h"

namespace qmag {

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
    *q0 = ak_row(A.cu[i], A.T);
    *nq = max(ak_row(A.cu[i + 1], A.T) - *q0, 0);
    *len = ak_len(A.len[i], A.max_blocks, A.shift);
}

// The sequence of item `want` (by_token: of row `want` of q), found by the
// calling wave alone.  False if there is none, or none that has room.
template <int RG, int STEP>
__device__ __forceinline__ bool ak_find(const AkArgs &A, int want, bool by_token, AkPlan *P)
{
    const int lane = lane_id();
    int q0 = 0, nq = 0, len = 0;
    if (lane < A.n_seq) ak_seq(A, lane, &q0, &nq, &len);
    P->chunk = AK_UNSPLIT;
    if (A.min_chunk) {
        float cost = ak_cost(ak_groups(nq, A.G, RG), len);       // the same for whoever forms it
        for (int i = 64 + lane; i < A.n_seq; i += 64) {
            int x, n, l;
            ak_seq(A, i, &x, &n, &l);
            cost += ak_cost(ak_groups(n, A.G, RG), l);
        }
        P->chunk = __builtin_amdgcn_readfirstlane(ak_chunk(group_sum<64>(cost), A.target, STEP, A.min_chunk));
    }
    int items = 0;
    for (int base = 0; base < A.n_seq; base += 64) {
        if (base) {
            q0 = nq = len = 0;
            if (base + lane < A.n_seq) ak_seq(A, base + lane, &q0, &nq, &len);
        }
        const int split = ak_split(len, P->chunk), mine = ak_items(ak_groups(nq, A.G, RG), split);
        const int incl = wave_scan(mine);
        const bool here = by_token ? want >= q0 && want < q0 + nq : want < items + incl;
        const unsigned long long hit = __ballot(here);
        if (hit) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll(hit) - 1);
            P->seq = base + at;
            P->q0 = __builtin_amdgcn_readlane(q0, at);
            P->nq = __builtin_amdgcn_readlane(nq, at);
            P->len = __builtin_amdgcn_readlane(len, at);
            P->n_split = __builtin_amdgcn_readlane(split, at);
            P->item0 = items + __builtin_amdgcn_readlane(incl - mine, at);
            return ak_room(P->item0, __builtin_amdgcn_readlane(mine, at), A.max_items);
        }
        items = min(items + __builtin_amdgcn_readlane(incl, 63), 1 << 30);
    }
    return false;
}

// The workgroup's kv head and item.  Items in order, all heads of each, so that
// those that have no work are the last to start: with the heads one behind
// another the idle ones between them left some CUs two busy workgroups and others
// none (one sequence of 32,768 tokens 21.9 us so, 18.8 in order; of 32 sequences,
// where few are idle, 51.9 and 52.1).
__device__ __forceinline__ void ak_item(const AkArgs &A, int *item, int *kvh)
{
    const unsigned i = blockIdx.x / (unsigned)A.n_kv;
    *item = (int)i;
    *kvh = (int)(blockIdx.x - i * (unsigned)A.n_kv);
}

// Where row r of a group of RG rows has its partial results: a row's parts one
// behind another (16 KB apart, as the workgroups write them, they would all lie
// in one memory channel: joining 256 of them took 14 us against 3).
__device__ __forceinline__ int64_t ak_part(const AkArgs &A, const AkPlan &P, int kvh, int group, int RG, int r)
{
    return ak_part_row(kvh, A.max_items, P.item0, group, P.n_split, RG, r);
}

// max and sum over the four lanes that hold a row
__device__ __forceinline__ float row_max(float v)
{
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
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

// The maximum of a row that has seen nothing: above no score, and finite, so that
// differences from it are numbers.
constexpr float AK_NONE = -3.402823466e38f;

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// What turns nibbles into fp16: masks and exponents in registers of both kinds,
// so that the two go into one instruction.
enum Code { CENTRED, PLAIN };
struct Nibbles {
    uint32_t lo = 0x000F000Fu, hi = 0x00F000F0u, e1024 = 0x64006400u, e64 = 0x54005400u;
    __device__ __forceinline__ Nibbles()
    {
        asm("" : "+s"(lo), "+s"(hi));
        asm("" : "+v"(e1024), "+v"(e64));
    }
    // nibbles 0 and 4 of w (of each half dword), or 1 and 5, as fp16
    template <Code CODE>
    __device__ __forceinline__ uint32_t even(uint32_t w) const
    {
        const _Float16 z = (_Float16)(CODE == CENTRED ? 1032.0f : 1024.0f);
        const half2v v = __builtin_bit_cast(half2v, (w & lo) | e1024) - (half2v){z, z};
        return __builtin_bit_cast(uint32_t, v);
    }
    template <Code CODE>
    __device__ __forceinline__ uint32_t odd(uint32_t w) const
    {
        const _Float16 z = (_Float16)(CODE == CENTRED ? 72.0f : 64.0f);
        const half2v v = __builtin_bit_cast(half2v, (w & hi) | e64) - (half2v){z, z};
        return __builtin_bit_cast(uint32_t, v);
    }
};

// Eight nibbles as eight fp16 values, in the order 0 4 1 5 2 6 3 7.
template <Code CODE>
__device__ __forceinline__ half8 k_frag(const Nibbles &N, uint32_t w)
{
    Frag f;
    f.u[0] = N.template even<CODE>(w);
    f.u[1] = N.template odd<CODE>(w);
    f.u[2] = N.template even<CODE>(w >> 8);
    f.u[3] = N.template odd<CODE>(w >> 8);
    return f.h;
}

// d, and the value of the operand 0
__device__ __forceinline__ float step_of(uint32_t dm) { return h2f(dm & 0xFFFFu); }
template <Code CODE>
__device__ __forceinline__ float mid_of(uint32_t dm)
{
    return CODE == CENTRED ? fmaf(8.0f, h2f(dm & 0xFFFFu), h2f(dm >> 16)) : h2f(dm >> 16);
}

// (hi, lo) fp16 parts of eight values; NS == 1: hi alone, to nearest
template <int NS>
__device__ __forceinline__ void split8(const float (&x)[8], half8 *hi, half8 *lo)
{
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        half2v h = {(_Float16)x[i], (_Float16)x[i + 1]};
        if constexpr (NS == 2) {
            half2v l;
            split2(x[i], x[i + 1], &h, &l);
            (*lo)[i] = l[0], (*lo)[i + 1] = l[1];
        }
        (*hi)[i] = h[0], (*hi)[i + 1] = h[1];
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

// The size of a step d (bits 0 .. 15, not negative): its exponent and first two digits, an
// e with d < 2^(e - 14.5), and of a normal d at least 2^(e - 15).  NaN and infinity have 31
// and more.
__device__ __forceinline__ float ak_size(uint32_t d) { return 0.25f * (float)(d >> 8 & 255u); }

// The weights p of a lane's eight scores (of what its row does not see -inf), by the
// maximum m so far, and their sum into l.  o and vs are the sums of p d code and p mid,
// o times 2^(7 - ve): the products' operands p d 2^(7 - ve) have to stay below 2^16, and
// near there to keep their bits.  Maximum and power of two move only where a weight
// would pass 2^8 or an operand 2^15.  The power follows the largest p d, not the largest
// d: a token of large values and no weight takes no bits from the others (300 tokens,
// one with a step 2^20 times theirs and a weight of e^-60: fp32 calls were off by 1e-3).
// size(i): of a token's largest step, or more; exact(x): the largest x + size of a lane
// with no more.
// (Arrays by reference: as members of a struct the compiler copied all of o in every tile.)
template <int NG, class Size, class Exact>
__device__ __forceinline__ void ak_weigh(const float (&s)[8], float (&p)[8], float &m, float &l, int &ve, float (&vs)[NG],
                                         f32x4 (&o)[NG][4], Size size, Exact exact)
{
    // (from the differences: large scores have no room for a size)
    float x[8], top = -INFINITY, far = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        x[i] = s[i] - m;
        top = fmaxf(top, x[i]);
        far = fmaxf(far, x[i] + size(i));
    }
    if (__any(top > 8.0f || far > (float)ve + 22.5f)) {
        // (a row that need not move stays: what others see has no part in its rounding)
        float high = s[0];
#pragma unroll
        for (int i = 1; i < 8; i++) high = fmaxf(high, s[i]);
        high = row_max(high);
        const float was = m;
        m = row_max(top) > 8.0f ? high : m;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = s[i] - m;
        far = row_max(exact(x));
        // what is summed so far shrinks with the maximum's move, and its power of two with it
        const int sunk = ve - (int)fminf(m - was, 200.0f), here = (int)ceilf(fminf(fmaxf(far - 14.5f, -60.0f), 40.0f));
        const int e = far > (float)ve + 22.5f || m != was ? max(max(here, sunk), -60) : ve;
        const float f = __builtin_amdgcn_exp2f(was - m), fo = __builtin_amdgcn_exp2f(was - m + (float)(ve - e));
        ve = e;
        l *= f;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            vs[g] *= f;
#pragma unroll
            for (int i = 0; i < 4; i++) o[g][i] *= fo;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        p[i] = __builtin_amdgcn_exp2f(x[i]);
        l += p[i];
    }
}

// p[i] d[i] 2^(7 - ve) in fp16 parts, for group g
template <Code CODE, int NS, int NG>
__device__ __forceinline__ void ak_operand(const float (&p)[8], const uint32_t (&vdm)[8][NG], int ve, float (&vs)[NG], int g,
                                           half8 *ph, half8 *pl)
{
    const float up = exp2i(7 - ve);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        x[i] = p[i] * up * step_of(vdm[i][g]);
        vs[g] = fmaf(p[i], mid_of<CODE>(vdm[i][g]), vs[g]);
    }
    split8<NS>(x, ph, pl);
}

// Bytes of a wave's tile of 32 tokens in LDS: K codes, V codes, scales of both.
template <int D>
constexpr int ak_tile() { return 36 * D; }

// A group of 16 rows against a chunk of the cache: the NW waves take its tiles
// of 32 tokens in turn and join at the end.  Each wave keeps its next tile in
// flight from memory to its own part of LDS (two tiles, no registers, no
// barriers); a lane later reads back little more than what it asked for itself.
//
// A step of one sequence is bound by a chain of round trips: of 14 us for 32,768
// tokens (fp32, 16 heads of 256; 18.9 MB, 4 us at a large copy's rate) 0.8 are the
// plan, 1.2 the table and the first tiles' requests, 1.2 the queries, 3.3 the tiles,
// 2 the join of the waves; a launch alone takes 2.9, and what is left was not found.
// (A chunk of 128 tokens becomes 256, see ak_chunk: one workgroup to a CU there.)  A
// batch is bound by vector instructions, 12 of whose 16 rows are empty with four heads
// to a kv head: 32 sequences of up to 16,384 tokens (bf16, 32 heads of 128; 163 MB) 46
// us, 3.5 TB/s, 62,000 of a CU's 83,000 cycles.

// how many of its workgroups of 4 waves LDS and registers let a CU hold
template <class T, int D>
constexpr int few_resident() { return D == 256 ? 2 : D == 128 && sizeof(typename T::S) == 4 ? 3 : 4; }

template <class T, int D, int NW>
__global__ void __launch_bounds__(64 * NW, (few_resident<T, D>())) attn_kv4_kernel(AkArgs A)
{
    using S = typename T::S;
    constexpr int NS = sizeof(S) == 4 ? 2 : 1;
    constexpr Code CODE = std::is_same_v<T, TBF16> ? PLAIN : CENTRED;
    constexpr int NG = D / 64;
    constexpr int RG = 16, STEP = 32 * NW;
    constexpr int VD = (D + 127) / 128;            // dwords of a lane's V codes of a token
    constexpr int TILE = ak_tile<D>();
    constexpr int LROW = D + 4;                    // row of the join
    constexpr int LDS = NW * 2 * TILE > NW * 16 * LROW * 4 ? NW * 2 * TILE : NW * 16 * LROW * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
    __shared__ float join_m[NW][16], join_l[NW][16];

    int item, kvh;
    ak_item(A, &item, &kvh);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), n = lane & 15, h = lane >> 4;
    AkPlan P;
    if (!ak_find<RG, STEP>(A, item, false, &P)) return;
    const int local = item - P.item0, split = local % P.n_split, group = local / P.n_split;
    const int rows = P.nq * A.G, r0 = group * RG;

    // ---- the range of tokens
    const int row = r0 + n, j = min(row, rows - 1) / A.G, gh = min(row, rows - 1) - j * A.G;
    const bool live = row < rows;
    const int past = P.len - P.nq;                 // tokens before the first query's own
    const int lim = live ? past + j : INT32_MAX;   // the last token the row sees
    const int j_last = (min(r0 + 16, rows) - 1) / A.G, open = past + r0 / A.G;
    const int c0 = split * P.chunk + 32 * wave;
    const int c1 = min(min(P.len, split * P.chunk + P.chunk), past + j_last + 1);
    // (read as constants: no kernel writes the table while this one runs)
    const auto *table = (const __attribute__((address_space(4))) int *)(A.table + P.seq * (int64_t)A.max_blocks);
    const int64_t block_stride = 2 * A.half * A.n_kv;
    const uint8_t *head = A.data + kvh * 2 * A.half;
    const int64_t codes = (int64_t)(D / 2) << A.shift;
    uint8_t *ring = lds + wave * 2 * TILE;

    // ---- tiles from memory: where in a half (16 tokens, within a block) a lane's pieces lie
    int k_from, v_from, s_from;
    bool k_up = false, v_up = false, s_up;         // the lane's piece is of the upper half
    if constexpr (D == 256) {
        k_from = (lane & 15) * 128 + (lane >> 4) * 32;
        v_from = (4 * ((lane >> 3) & 3) + (lane >> 5)) * 128 + (lane & 7) * 16;
    } else if constexpr (D == 128) {
        k_from = (lane & 15) * 64 + (lane >> 4) * 16;
        v_from = (4 * ((lane >> 2) & 3) + (lane >> 4)) * 64 + (lane & 3) * 16;
    } else {
        k_from = (lane & 15) * 32 + ((lane >> 4) & 1) * 16;
        v_from = (4 * ((lane >> 1) & 3) + ((lane >> 3) & 3)) * 32 + (lane & 1) * 16;
        k_up = v_up = lane >= 32;
    }
    {
        const int w = lane / (8 * NG), c = lane % (8 * NG);
        s_up = c >= 4 * NG;
        s_from = (w ? (int)A.half : 0) + (int)codes + (c % (4 * NG)) * 16;
    }
    uint32_t gone = 0;                             // two bits a tile in flight: a half whose block is none
    auto dma = [&](const uint8_t *from, uint8_t *to) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                         (__attribute__((address_space(3))) void *)to, 16, 0, 0);
    };
    auto issue = [&](int t0, int slot) {
        const uint8_t *kb[2];
        int off[2];
        uint32_t bad = 0;
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const int t = t0 + 16 * a;
            const int id = table[min(t >> A.shift, A.max_blocks - 1)];
            const bool there = id >= 0 && id < A.n_block;
            bad |= there ? 0u : 1u << a;
            kb[a] = head + (there ? id : 0) * block_stride;
            off[a] = t & ((1 << A.shift) - 1);
        }
        gone = (gone >> 2) | (bad << 2);
        uint8_t *to = ring + slot * TILE;
        const uint8_t *k[2] = {kb[0] + off[0] * (D / 2), kb[1] + off[1] * (D / 2)};
        if constexpr (D == 64) {
            dma((k_up ? k[1] : k[0]) + (uint32_t)k_from, to);
            dma((v_up ? k[1] : k[0]) + A.half + (uint32_t)v_from, to + 1024);
        } else {
#pragma unroll
            for (int i = 0; i < D / 64; i++)       // D = 256: (half, piece), 128: half
                dma(k[D == 256 ? i >> 1 : i] + (D == 256 ? 16 * (i & 1) : 0) + (uint32_t)k_from, to + 1024 * i);
#pragma unroll
            for (int i = 0; i < D / 64; i++)
                dma(k[D == 256 ? i >> 1 : i] + A.half + (D == 256 ? 256 * (i & 1) : 0) + (uint32_t)v_from, to + 16 * D + 1024 * i);
        }
        if (lane < 16 * NG) dma((s_up ? kb[1] + off[1] * (NG * 4) : kb[0] + off[0] * (NG * 4)) + s_from, to + 32 * D);
    };
    float x[NG][2][8];                             // the row's queries, under way before the tiles
    {
        const S *qp = (const S *)A.q + (P.q0 + j) * A.qt + (kvh * A.G + gh) * A.qh;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int s = 0; s < 2; s++) load8<T>(qp + g * 64 + s * 32 + h * 8, A.q_vec, x[g][s]);
    }
    if (c0 < c1) issue(c0, 0);

    const Nibbles N;
    // ---- queries
    half8 qh[NG][2], ql[NS == 2 ? NG : 1][2];
    float qs[NG], rs;
    {
        float top = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[g][s][i]));
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

    f32x4 o[NG][4];
    float vs[NG], l = 0.0f, m = AK_NONE;
    int ve = -60;                                  // o carries 2^(7 - ve)
#pragma unroll
    for (int g = 0; g < NG; g++) {
        vs[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) o[g][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int slot = 0;
    for (int t0 = c0; t0 < c1; t0 += STEP) {
        // this tile's pieces are in; the next ones' go out
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (t0 + STEP < c1) issue(t0 + STEP, slot ^ 1);
        else gone >>= 2;
        const uint32_t bad = gone & 3;
        const uint8_t *tile = ring + slot * TILE;
        slot ^= 1;

        // ---- scores
        float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int a = 0; a < 2; a++) {
            uint32_t kc[D / 32], dm[4][NG];
            if constexpr (D == 64) load_dwords(tile + (a * 32 + (h >> 1) * 16 + n) * 16 + (h & 1) * 8, kc);
            else {
#pragma unroll
                for (int i = 0; i < D / 128; i++) {
                    const uint4 v = *(const uint4 *)(tile + ((a * (D / 128) + i) * 64 + lane) * 16);
                    kc[4 * i] = v.x, kc[4 * i + 1] = v.y, kc[4 * i + 2] = v.z, kc[4 * i + 3] = v.w;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) load_dwords(tile + 32 * D + (16 * a + 4 * h + r) * (NG * 4), dm[r]);
#pragma unroll
            for (int g = 0; g < NG; g++) {
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    const half8 kf = k_frag<CODE>(N, kc[2 * g + st]);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[g][st], acc, 0, 0, 0);
                    if constexpr (NS == 2) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[g][st], acc, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float d = step_of(dm[r][g]), mid = mid_of<CODE>(dm[r][g]);
                    s[4 * a + r] = fmaf(d, acc[r], fmaf(mid, qs[g], s[4 * a + r]));
                }
            }
        }
        uint32_t vdm[8][NG];
#pragma unroll
        for (int i = 0; i < 8; i++) load_dwords(tile + 32 * D + 128 * NG + (16 * (i >> 2) + 4 * h + (i & 3)) * (NG * 4), vdm[i]);
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] *= rs;
        if (bad || t0 + 31 > open) {
            // a token the row does not see has no weight, whatever the cache holds there
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int a = i >> 2, tk = t0 + 16 * a + 4 * h + (i & 3);
                const bool seen = tk <= lim && tk < c1 && !((bad >> a) & 1);
                s[i] = seen ? s[i] : -INFINITY;
#pragma unroll
                for (int g = 0; g < NG; g++) vdm[i][g] = seen ? vdm[i][g] : 0u;
            }
        }
        float p[8];
        ak_weigh<NG>(
            s, p, m, l, ve, vs, o,
            [&](int i) {
                typedef short s16x2 __attribute__((ext_vector_type(2)));
                s16x2 d = __builtin_bit_cast(s16x2, vdm[i][0]);
#pragma unroll
                for (int g = 1; g < NG; g++) d = __builtin_elementwise_max(d, __builtin_bit_cast(s16x2, vdm[i][g]));
                return ak_size(__builtin_bit_cast(uint32_t, d));
            },
            [&](const float (&x)[8]) {
                float far = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        const float e = ak_size(vdm[i][g]);
                        far = fmaxf(far, e < 31.0f ? x[i] + e : -INFINITY);        // (NaN has no part in it)
                    }
                return far;
            });

        // ---- output
        uint32_t vc[8][VD];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint8_t *v = tile + 16 * D + (i * 4 + h) * (D / 2) + n * (D / 32);
            if constexpr (D == 64) vc[i][0] = *(const uint16_t *)v;
            else load_dwords(v, vc[i]);
        }
#pragma unroll
        for (int g = 0; g < NG; g++) {
            half8 ph, pl;
            ak_operand<CODE, NS>(p, vdm, ve, vs, g, &ph, &pl);
#pragma unroll
            for (int b = 0; b < 2; b++) {
                // byte b of group g: channels 4 n + 2 b and the next of every token
                Frag even, odd;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int at = 2 * (g & 1) + b;
                    const uint32_t w = __builtin_amdgcn_perm(vc[2 * k + 1][g >> 1], vc[2 * k][g >> 1],
                                                             0x0C040C00u + 0x00010001u * (uint32_t)at);
                    even.u[k] = N.template even<CODE>(w);
                    odd.u[k] = N.template odd<CODE>(w);
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

    // ---- the waves' shares; a lane's row: channels 64 g + 4 (4 h + r) + i in o[g][i][r]
    l = row_sum(l);
    const float back = exp2i(ve - 7);
    if (h == 0) {
        join_m[wave][n] = m;
        join_l[wave][n] = l;
    }
    __syncthreads();                               // no wave reads its tiles any more either
    float all = AK_NONE;
#pragma unroll
    for (int w = 0; w < NW; w++) all = fmaxf(all, join_m[w][n]);
    const float share = __builtin_amdgcn_exp2f(m - all);      // (nothing seen: sums of zero; a NaN stays one)
    float *join = (float *)lds, *mine = join + (wave * 16 + n) * LROW;
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const float add = row_sum(vs[g]);
#pragma unroll
        for (int r = 0; r < 4; r++)
            *(float4 *)(mine + 64 * g + 4 * (4 * h + r)) =
                make_float4(fmaf(o[g][0][r], back, add) * share, fmaf(o[g][1][r], back, add) * share,
                            fmaf(o[g][2][r], back, add) * share, fmaf(o[g][3][r], back, add) * share);
    }
    __syncthreads();
    // 4 NW threads a row, four channels at a time
    constexpr int PER = 4 * NW, CP = D / (4 * PER) > 0 ? D / (4 * PER) : 1;
    const int rr = threadIdx.x / PER, cc = threadIdx.x % PER;
    if (r0 + rr >= rows) return;
    float M = AK_NONE, L = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) M = fmaxf(M, join_m[w][rr]);
#pragma unroll
    for (int w = 0; w < NW; w++) L += join_l[w][rr] * __builtin_amdgcn_exp2f(join_m[w][rr] - M);
    const int jj = (r0 + rr) / A.G, hh = r0 + rr - jj * A.G;
    S *op = (S *)A.out + (P.q0 + jj) * A.ot + (kvh * A.G + hh) * A.oh;
    const int64_t at = ak_part(A, P, kvh, group, RG, rr) + split;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int cb = 0; cb < CP; cb++) {
        const int c = 4 * (cb * PER + cc);
        if (c >= D) break;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float4 f = *(const float4 *)(join + (w * 16 + rr) * LROW + c);
            v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
        }
        if (P.n_split == 1) {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] *= inv;
            store4<T>(op + c, A.o_vec, v);
        } else {
            store4<TF32>(A.part + at * D + c, true, v);
        }
    }
    if (P.n_split > 1 && cc == 0) {
        A.ml[2 * at] = M;
        A.ml[2 * at + 1] = L;
    }
}

// Many rows to a sequence: NW waves of 16 rows each against a chunk of the cache.
// A tile of 32 tokens comes from memory to LDS as it lies there, is turned into
// fp16 codes once for all the waves (K and V row by row, in the order the
// products read them), and then serves as a tile of a prompt does; memory is two
// tiles ahead, the codes one, and a tile costs one barrier.
//
// Bound by what a tile costs a wave besides its 64 products (fp32, heads of 256:
// 1024 cycles): about 400 vector instructions, a quarter of them for steps and
// minima, and as many cycles of LDS reads, which 8 waves share.  512 rows of 8 heads
// each at 12,001 tokens: 303 us with the join, 325 TFLOP/s, or 650 of fp16 products.
// (With 4 waves of an earlier form 544 us against 349; 64 rows that formed their codes
// themselves 457.)

// how many of its workgroups of 8 waves the registers let a CU hold
template <class T, int D>
constexpr int rows_resident() { return D == 256 || (D == 128 && sizeof(typename T::S) == 4) ? 1 : 2; }

template <class T, int D, int NW>
__global__ void __launch_bounds__(64 * NW, (2 * rows_resident<T, D>())) attn_kv4_rows_kernel(AkArgs A)
{
    using S = typename T::S;
    constexpr int NS = sizeof(S) == 4 ? 2 : 1;
    constexpr Code CODE = std::is_same_v<T, TBF16> ? PLAIN : CENTRED;
    constexpr int NG = D / 64;
    constexpr int RG = 16 * NW, STEP = 32;
    constexpr int TILE = ak_tile<D>(), IMG = 32 * D, SC = 4 * D;   // bytes, values, bytes
    __shared__ __attribute__((aligned(16))) uint8_t raw[2][TILE];
    __shared__ __attribute__((aligned(16))) _Float16 ik[2][IMG], iv[2][IMG];
    __shared__ __attribute__((aligned(16))) uint8_t isc[2][SC];    // scales of K, then of V: [32][NG] each
    __shared__ __attribute__((aligned(16))) float isize[2][32];    // ak_size of a token's largest step of V

    int item, kvh;
    ak_item(A, &item, &kvh);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), n = lane & 15, h = lane >> 4;
    AkPlan P;
    if (!ak_find<RG, STEP>(A, item, false, &P)) return;
    const int local = item - P.item0, split = local % P.n_split, group = local / P.n_split;
    const int rows = P.nq * A.G, r0 = group * RG + wave * 16;

    // ---- the range of tokens
    const int row = r0 + n, j = min(row, rows - 1) / A.G, gh = min(row, rows - 1) - j * A.G;
    const bool live = row < rows;
    const int past = P.len - P.nq;                 // tokens before the first query's own
    const int lim = live ? past + j : INT32_MAX;   // the last token the row sees
    const int open = past + min(r0, rows - 1) / A.G;
    const int c0 = split * P.chunk, c1 = min(P.len, c0 + P.chunk);
    const int all = min(c1, past + (min(group * RG + RG, rows) - 1) / A.G + 1);        // what any row sees
    const int mine = r0 < rows ? min(c1, past + (min(r0 + 16, rows) - 1) / A.G + 1) : c0;   // what the wave's see
    const auto *table = (const __attribute__((address_space(4))) int *)(A.table + P.seq * (int64_t)A.max_blocks);
    const int64_t block_stride = 2 * A.half * A.n_kv;
    const uint8_t *head = A.data + kvh * 2 * A.half;
    const int codes = (D / 2) << A.shift;

    // ---- tiles from memory, 16-byte pieces in the order [K codes | V codes | K scales | V scales], halves in turn
    constexpr int PIECES = TILE / 16;
    uint32_t gone = 0;                             // two bits a tile: a half whose block is none
    auto issue = [&](int t0, int b) {
        const uint8_t *kb[2];
        int off[2];
        uint32_t bad = 0;
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const int t = t0 + 16 * a;
            const int id = table[min(t >> A.shift, A.max_blocks - 1)];
            const bool there = id >= 0 && id < A.n_block;
            bad |= there ? 0u : 1u << a;
            kb[a] = head + (there ? id : 0) * block_stride;
            off[a] = t & ((1 << A.shift) - 1);
        }
        gone = (gone >> 2) | (bad << 4);
#pragma unroll
        for (int w = 0; w < (PIECES + 64 * NW - 1) / (64 * NW); w++) {
            const int p0 = (w * NW + wave) * 64, p = p0 + lane;
            if (p >= PIECES) break;
            const bool sc = p >= 2 * D;
            const int q = sc ? p - 2 * D : p, per = sc ? D / 16 : D / 2;       // pieces of a half
            const int v = q >= 2 * per, a = (q / per) & 1, x = q % per;
            const uint8_t *from = (a ? kb[1] : kb[0]) + (v ? A.half : 0) + (sc ? codes + (a ? off[1] : off[0]) * (NG * 4) : (a ? off[1] : off[0]) * (D / 2)) + 16 * x;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                             (__attribute__((address_space(3))) void *)(raw[b] + 16 * p0), 16, 0, 0);
        }
    };
    const Nibbles N;
    auto unpack = [&](int b) {
#pragma unroll
        for (int w = 0; w < (PIECES + 64 * NW - 1) / (64 * NW); w++) {
            const int p = w * 64 * NW + (int)threadIdx.x;
            if (p >= PIECES) break;
            const uint4 x = *(const uint4 *)(raw[b] + 16 * p);
            const uint32_t u[4] = {x.x, x.y, x.z, x.w};
            if (p < D) {                           // K: dword h * D / 32 + 2 g + s of a row
                const int t = p / (D / 32), d0 = 4 * (p % (D / 32));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int hh = (d0 + i) / (D / 32), gs = (d0 + i) % (D / 32);
                    *(half8 *)(ik[b] + t * D + 8 * (D == 64 ? (4 * gs + hh) ^ ((t >> 1) & 7) : (4 * gs + hh) ^ (t & 15))) =
                        k_frag<CODE>(N, u[i]);
                }
            } else if (p < 2 * D) {                // V: 16-bit word i * NG + g of a row, four channels
                const int t = (p - D) / (D / 32), w0 = 8 * ((p - D) % (D / 32));
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t c = i & 1 ? u[i >> 1] >> 16 : u[i >> 1] & 0xFFFFu;
                    const int ii = (w0 + i) / NG, g = (w0 + i) % NG, ch = 8 * g + (ii >> 1);
                    union { uint32_t u[2]; s16x4 v; } y;
                    y.u[0] = N.template even<CODE>(c | (c << 12));
                    y.u[1] = N.template even<CODE>((c >> 8) | (c << 4));
                    *(s16x4 *)(iv[b] + t * D + 8 * (D == 64 ? ch ^ (t & 6) : ch ^ ((t & 7) << 1)) + 4 * (ii & 1)) = y.v;
                }
            } else {
                *(uint4 *)(isc[b] + 16 * (p - 2 * D)) = x;
                const int w0 = 4 * (p - 2 * D) - 32 * NG;          // V's, from this piece on
                if (w0 >= 0)
#pragma unroll
                    for (int i = 0; i < 4; i += NG) {
                        float e = 0.0f;            // (NaN has no part in it)
#pragma unroll
                        for (int g = 0; g < NG; g++) e = fmaxf(e, ak_size(u[i + g]) < 31.0f ? ak_size(u[i + g]) : 0.0f);
                        isize[b][w0 / NG + i / NG] = e;
                    }
            }
        }
    };
    auto arrived = [&]() {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
    };
    if (c0 < all) issue(c0, 0);

    // ---- queries
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

    f32x4 o[NG][4];                                // channels 64 g + 16 i + 4 h + r in o[g][i][r]
    float vs[NG], l = 0.0f, m = AK_NONE;
    int ve = -60;                                  // o carries 2^(7 - ve)
#pragma unroll
    for (int g = 0; g < NG; g++) {
        vs[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) o[g][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // a lane's places in an image: its chunk of K's row n, four of its tokens' 16 channels of V
    constexpr int KV = D == 64 ? 2 : 4, VV = D == 64 ? 4 : 8;        // places that differ by more than a constant
    int k_at[KV], v_at[VV];
#pragma unroll
    for (int i = 0; i < KV; i++) k_at[i] = n * D + 8 * (D == 64 ? (4 * i + h) ^ (n >> 1) : (4 * i + h) ^ n);
#pragma unroll
    for (int i = 0; i < VV; i++) {
        const int t = 4 * h + (n >> 2), ch = 2 * i + ((n & 3) >> 1);
        v_at[i] = t * D + 8 * (D == 64 ? ch ^ (t & 6) : ch ^ ((t & 7) << 1)) + 4 * (n & 1);
    }

    auto compute = [&](int t0, int b, uint32_t bad) {
        // ---- scores
        float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int a = 0; a < 2; a++) {
            uint32_t dm[4][NG];
#pragma unroll
            for (int r = 0; r < 4; r++) load_dwords(isc[b] + (16 * a + 4 * h + r) * (NG * 4), dm[r]);
#pragma unroll
            for (int g = 0; g < NG; g++) {
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    const int k = 2 * g + st;
                    const half8 kf = *(const half8 *)(ik[b] + k_at[k % KV] + 128 * (k / KV) + 16 * a * D);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[g][st], acc, 0, 0, 0);
                    if constexpr (NS == 2) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[g][st], acc, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float d = step_of(dm[r][g]), mid = mid_of<CODE>(dm[r][g]);
                    s[4 * a + r] = fmaf(d, acc[r], fmaf(mid, qs[g], s[4 * a + r]));
                }
            }
        }
        uint32_t vdm[8][NG];
#pragma unroll
        for (int i = 0; i < 8; i++) load_dwords(isc[b] + SC / 2 + (16 * (i >> 2) + 4 * h + (i & 3)) * (NG * 4), vdm[i]);
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] *= rs;
        if (bad || t0 + 31 > open) {
            // a token the row does not see has no weight, whatever the cache holds there
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int a = i >> 2, tk = t0 + 16 * a + 4 * h + (i & 3);
                const bool seen = tk <= lim && tk < mine && !((bad >> a) & 1);
                s[i] = seen ? s[i] : -INFINITY;
#pragma unroll
                for (int g = 0; g < NG; g++) vdm[i][g] = seen ? vdm[i][g] : 0u;
            }
        }
        float p[8];
        const f32x4 size[2] = {*(const f32x4 *)(isize[b] + 4 * h), *(const f32x4 *)(isize[b] + 16 + 4 * h)};
        ak_weigh<NG>(
            s, p, m, l, ve, vs, o, [&](int i) { return size[i >> 2][i & 3]; },
            [&](const float (&x)[8]) {
                float far = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++) far = fmaxf(far, x[i] + size[i >> 2][i & 3]);
                return far;
            });

        // the next tile's codes, between the two products: its LDS reads and vector work run while
        // the other waves multiply (fp32, heads of 256: ahead of the scores 321 us, behind the output
        // 333, here 305; bf16 of 128: 235, 238, 240)
        if (t0 + STEP < all) unpack(b ^ 1);

        // ---- output
#pragma unroll
        for (int g = 0; g < NG; g++) {
            half8 ph, pl;
            ak_operand<CODE, NS>(p, vdm, ve, vs, g, &ph, &pl);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                union { s16x4 r[2]; half8 v; } vf;
                const int part = 4 * g + i;        // of 16 channels
#pragma unroll
                for (int u = 0; u < 2; u++)
                    vf.r[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s16x4 *)(iv[b] + v_at[part % VV] + 128 * (part / VV) + 16 * u * D));
                o[g][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf.v, ph, o[g][i], 0, 0, 0);
                if constexpr (NS == 2) o[g][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf.v, pl, o[g][i], 0, 0, 0);
            }
        }
    };

    arrived();
    if (c0 + STEP < all) issue(c0 + STEP, 1);
    else gone >>= 2;
    if (c0 < all) unpack(0);
    for (int t0 = c0, b = 0; t0 < all; t0 += STEP, b ^= 1) {
        arrived();
        // two bits each: this tile, the next, the one after it
        const uint32_t bad = (gone >> 2) & 3;
        if (t0 + 2 * STEP < all) issue(t0 + 2 * STEP, b);
        else gone >>= 2;
        if (t0 < mine) compute(t0, b, bad);
        else if (t0 + STEP < all) unpack(b ^ 1);
    }

    if (!live) return;
    l = row_sum(l);
    const float back = exp2i(ve - 7);
    const float inv = P.n_split > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
    S *op = (S *)A.out + (P.q0 + j) * A.ot + (kvh * A.G + gh) * A.oh;
    const int64_t at = ak_part(A, P, kvh, group, RG, wave * 16 + n) + split;
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const float add = row_sum(vs[g]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = 64 * g + 16 * i + 4 * h;
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = fmaf(o[g][i][r], back, add) * inv;
            if (P.n_split == 1) store4<T>(op + c, A.o_vec, y);
            else store4<TF32>(A.part + at * D + c, true, y);
        }
    }
    if (P.n_split > 1 && h == 0) {
        A.ml[2 * at] = m;
        A.ml[2 * at + 1] = l;
    }
}

// Joins the partial results of the rows whose sequence was split: NW waves for CW
// channels of a row, the waves the parts in turn.  Decode of a few rows has many
// parts to a row (16 waves for 64 channels: a wave's parts are all requested at
// once), of more rows fewer (four waves a row), many rows to a sequence a handful
// (a wave for a row, four heads of a token to a workgroup).  4.9 us for 16 rows of 128
// parts, of which 2 are the launch; with 4 waves a row 7.2.  Of 16 parts 4 waves are
// 1.2 us faster than 16.
template <class T, int D, int RG, int STEP, int NW, int CW>
__global__ void __launch_bounds__(NW == 1 ? 256 : 64 * NW) attn_kv4_join_kernel(AkArgs A)
{
    using S = typename T::S;
    constexpr int C = CW / 64;                      // consecutive channels of a lane
    constexpr int U = NW == 1 ? 4 : 8;              // parts requested at once
    __shared__ float sum[NW][CW], sl[NW], sm[NW];
    const int wave = NW == 1 ? 0 : threadIdx.x >> 6, lane = lane_id();
    const int t = blockIdx.x, head = NW == 1 ? 4 * blockIdx.y + (threadIdx.x >> 6) : blockIdx.y;
    const int kvh = head / A.G, gh = head - kvh * A.G, c0 = CW * blockIdx.z + C * lane;
    AkPlan P;
    if (head >= A.n_kv * A.G || !ak_find<RG, STEP>(A, t, true, &P) || P.n_split == 1) return;
    const int row = (t - P.q0) * A.G + gh;
    const int64_t first = ak_part(A, P, kvh, row / RG, RG, row % RG);
    struct alignas(4 * C) Vec { float v[C]; };
    float acc[C], L = 0.0f, M = AK_NONE;
#pragma unroll
    for (int c = 0; c < C; c++) acc[c] = 0.0f;
    // (a part that saw no token has nothing but zeros)
    for (int i0 = wave; i0 < P.n_split; i0 += U * NW) {
        float2 ml[U];
        Vec v[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t at = first + min(i0 + u * NW, P.n_split - 1);
            ml[u] = *(const float2 *)(A.ml + 2 * at);
            v[u] = *(const Vec *)(A.part + at * D + c0);
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < U; u++) top = fmaxf(top, ml[u].x);
        const float old = __builtin_amdgcn_exp2f(M - top);
        M = top;
        L *= old;
#pragma unroll
        for (int c = 0; c < C; c++) acc[c] *= old;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float f = i0 + u * NW < P.n_split ? __builtin_amdgcn_exp2f(ml[u].x - M) : 0.0f;
            L = fmaf(f, ml[u].y, L);
#pragma unroll
            for (int c = 0; c < C; c++) acc[c] = fmaf(f, v[u].v[c], acc[c]);
        }
    }
    S *op = (S *)A.out + t * A.ot + head * A.oh + c0;
    if constexpr (NW > 1) {
#pragma unroll
        for (int c = 0; c < C; c++) sum[wave][C * lane + c] = acc[c];
        if (lane == 0) sl[wave] = L, sm[wave] = M;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, sm[w]);
        L = 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++) acc[c] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(sm[w] - M);
            L += f * sl[w];
#pragma unroll
            for (int c = 0; c < C; c++) acc[c] += f * sum[w][C * lane + c];
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int c = 0; c < C; c++) op[c] = T::down(acc[c] * inv);
}

template <class T, int D, bool ROWS>
static int ak_launch(AkArgs A, hipStream_t s)
{
    constexpr int NW = ROWS ? 8 : 4, RG = ROWS ? 16 * NW : 16, STEP = ROWS ? 32 : 32 * NW;
    // Row groups at most.  Chunks are cut for as many workgroups as the chip holds at
    // once: of more the last ones run alone, of fewer some CUs get two and others none.
    // (They are whole steps, so that between half and all of that many run.  Heads of 256
    // for 4 of a CU instead of the 2 that its LDS holds: 40.4 us against 36.0 for 131,072
    // tokens, 43.5 against 34.8 for 48 sequences; heads of 128 in 16 bits for 3 instead of 4:
    // 52.1 against 50.8 for 32 sequences, 38.0 against 36.8 for 8, 42.5 against 43.2 for one
    // of 131,072 tokens; of 64 for 3 instead of 4: 37.9 against 35.4, 25.7 against 24.7.)
    const int64_t groups = ak_most_groups(A.T, A.G, RG, A.n_seq);
    const int64_t goal = (ROWS ? rows_resident<T, D>() : few_resident<T, D>()) * (int64_t)ctx().n_cu;
    A.target = (int)((goal + A.n_kv - 1) / A.n_kv);
    // enough row groups to fill the chip twice over: nothing is split
    A.min_chunk = ((int64_t)A.T * A.G / RG) * A.n_kv >= 2 * goal ? 0 : 128;
    const int64_t parts = (((int64_t)A.max_blocks << A.shift) + 127) / 128;       // of a sequence at most
    const int64_t items = A.min_chunk ? ak_most_items(groups, A.target, parts) : groups;
    if (items * A.n_kv >= 1 << 23) return fail(QMAG_ERR_ARG, "attn_kv4: %lld groups of rows", (long long)items);
    A.max_items = (int)items;
    if (A.min_chunk) {
        int st;
        const size_t rows = (size_t)A.n_kv * A.max_items * RG;
        A.part = (float *)workspace(WS_ATTN, rows * (D + 2) * sizeof(float), &st);
        if (st) return st;
        A.ml = A.part + rows * D;
    }
    const dim3 grid((unsigned)(items * A.n_kv));
    if constexpr (ROWS) attn_kv4_rows_kernel<T, D, NW><<<grid, 64 * NW, 0, s>>>(A);
    else attn_kv4_kernel<T, D, NW><<<grid, 64 * NW, 0, s>>>(A);
    if (A.min_chunk) {
        const unsigned T_ = (unsigned)A.T, heads = (unsigned)(A.n_kv * A.G);
        if constexpr (ROWS)
            attn_kv4_join_kernel<T, D, RG, STEP, 1, D><<<dim3(T_, (heads + 3) / 4), 256, 0, s>>>(A);
        else if ((int64_t)A.T * heads * (D / 64) <= ctx().n_cu && (parts < A.target ? parts : A.target) > 48)
            attn_kv4_join_kernel<T, D, RG, STEP, 16, 64><<<dim3(T_, heads, D / 64), 1024, 0, s>>>(A);
        else
            attn_kv4_join_kernel<T, D, RG, STEP, 4, D><<<dim3(T_, heads), 256, 0, s>>>(A);
    }
    return QMAG_OK;
}

template <class T, int D>
static int ak_pick(const AkArgs &A, hipStream_t s)
{
    // Few rows to a sequence: the waves share them and split the tokens, and every 16
    // rows read the cache again; of more the codes are formed once for 128.  With / without
    // that, 256 rows: 25.1 / 22.3 us over 2000 tokens, 98 / 114 over 32,768 (bf16, 32 heads of
    // 128), 35 / 21 and 80 / 79 (fp32, 16 heads of 256); 512 rows: 35 / 31, 172 / 216, 38 / 25
    // and 125 / 136.  The host knows the mean of a call only: beside 40 decoding sequences a
    // chunk of 512 tokens is better a call of its own (bf16 161 us in one call, 141 in two), one
    // of 128 is not (63 and 75).
    if ((int64_t)A.T * A.G <= 256 * (int64_t)A.n_seq) return ak_launch<T, D, false>(A, s);
    return ak_launch<T, D, true>(A, s);
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
    if (T > 0 && t->n_seq > 0) {
        auto meets = [&](const void *p, size_t bytes) { return heads_meet(out, attn_type_size(type), c->head_dim, T, p, bytes); };
        if (meets(cu, sizeof(int) * (size_t)(t->n_seq + 1)) || meets(len, sizeof(int) * (size_t)t->n_seq) ||
            meets(t->table, sizeof(int) * (size_t)t->n_seq * (size_t)t->max_blocks) || meets(c->data, kv4_bytes(c)))
            return fail(QMAG_ERR_ARG, "attn_kv4: the output overlaps the lengths, the table or the cache");
    }
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
