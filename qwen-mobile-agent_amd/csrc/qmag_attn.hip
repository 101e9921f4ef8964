// qmag_attn.hip -- causal attention over whole prompts, packed one behind
// another, heads in groups that share K and V (the role of attn_worker on a
// prompt chunk, src/nn.c:1215-1453).
//
//   o_i = sum_{j <= i} p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max_i)
//
// Two launches.  The first lays K and V out in tiles of 32 keys of one sequence
// and kv head, in the order the second's LDS wants them, rows behind a
// sequence's end zero: split or converted once instead of by every head and
// group of queries that reads them.  In the second a workgroup takes 64 or 128
// queries of a head, 16 or 32 to a wave, and passes over the tiles once with a
// running maximum and sum.  Calls of few tokens are one launch (DIRECT).
//
// 16-bit calls multiply in their own type.  fp32 calls are carried by the fp16
// matrix cores, 16 times the fp32 ones' rate: every row of Q, K and V is scaled
// by a power of two (exact) and split into two fp16 parts, x = hi + lo to 22
// bits, and a product is hi hi + hi lo + lo hi.  16-bit calls round a weight to
// their type, for the second product and for the sum: as much again as the rounding
// of the result where many keys count (bf16 2.1e-3 of it in all, the result's rounding
// 1.6e-3), less where few do, nothing where one does.
//
// S^T = K Q^T by v_mfma_f32_32x32x16 leaves a lane with one query (n = lane % 32)
// and keys 8 (r / 4) + 4 (lane / 32) + r % 4 of a tile, by v_mfma_f32_16x16x32
// (n = lane % 16) with keys 4 (lane / 16) + r of each 16; O^T = V^T P^T takes the
// weights as they are when V's keys are read in that order, so they never leave
// their lane.  V^T comes from row-major LDS by transposing reads.
//
// Bound by the matrix and vector units in turn: a tile of 32 x 32 scores of heads
// of 128 is 512 cycles of products and about 500 of vector instructions, half of
// them exponentials (a quarter rate), on a SIMD that three waves share.  Measured,
// both launches: bf16, 8192 tokens in five prompts, 32 heads of 128 over 8: 370 us,
// 830 TFLOP/s (a large bf16 product in the library: 1223); fp32, 4096 tokens, 16
// heads of 256 over 2: 421 us, 326 TFLOP/s, or 979 of fp16 products (library: 1179;
// its fp32 ones 153).  The first launch is 16 and 12 us of these.
#include <type_traits>

#include "qmag_attn.h"

namespace qmag {

constexpr int AP_WG = 256;
constexpr int AP_KEYS = 32;               // keys of a tile

struct ApArgs {
    const void *q, *k, *v;
    void *out;
    int64_t qt, qh, kt, kh, vt, vh, ot, oh;
    const int *cu;
    uint8_t *img;                         // [n_kv][tiles][K image | V image]
    float *scale;                         // [n_kv][tiles][32 of K | 32 of V], fp32 calls
    int *flags;                           // [n_kv][tiles][2]: K (fp32 calls), V hold an infinity or a NaN
    int n_seq, T, tiles, n_kv, G;
    float sc;                             // scale * log2 e
    int q_vec, k_vec, v_vec, o_vec;
};

// Sequence i's rows, and its first tile: floor(cu / 32) + i leaves every
// sequence the tiles it needs, whatever the lengths.
__device__ __forceinline__ void ap_seq(const ApArgs &A, int i, int *a, int *n)
{
    *a = min(max(A.cu[i], 0), A.T);
    *n = max(min(max(A.cu[i + 1], 0), A.T) - *a, 0);
}

// The sequence and part of it that hold unit `want` of `per` rows each; last:
// counted from the end.  Found by the calling wave alone.  (At most 2^22 / 32
// units a sequence, whatever the lengths: the sums stay below 2^30.)
__device__ __forceinline__ bool ap_find(const ApArgs &A, int want, int per, bool last, int *seq, int *part, int *a, int *n)
{
    const int lane = lane_id();
    int x = 0, len = 0;
    if (lane < A.n_seq) ap_seq(A, lane, &x, &len);
    if (last) {
        int all = (len + per - 1) / per, y, m;
        for (int i = 64 + lane; i < A.n_seq; i += 64) {
            ap_seq(A, i, &y, &m);
            all += (m + per - 1) / per;
        }
        all = group_sum_i<64>(all);
        if (want >= all) return false;
        want = all - 1 - want;
    }
    int before = 0;
    for (int base = 0; base < A.n_seq; base += 64) {
        if (base) {
            x = len = 0;
            if (base + lane < A.n_seq) ap_seq(A, base + lane, &x, &len);
        }
        const int mine = (len + per - 1) / per, incl = wave_scan(mine);
        const unsigned long long hit = __ballot(want < before + incl);
        if (hit) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll(hit) - 1);
            *seq = base + at;
            *a = __builtin_amdgcn_readlane(x, at);
            *n = __builtin_amdgcn_readlane(len, at);
            *part = want - before - __builtin_amdgcn_readlane(incl - mine, at);
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// 16-byte chunks of an image row are exchanged by key so that the rows of a
// read keep apart in LDS's 64 banks (256 bytes): for K 16 keys' chunk; for V 64
// bytes of 4 keys, or 32 bytes of 8 with 16 queries.  (Where a row is 128 bytes,
// only keys of one parity share banks.)
template <int D>
__device__ __forceinline__ int k_chunk(int key, int c) { return c ^ (D == 64 ? (key >> 1) & 7 : key & 15); }
template <int D, int QW>
__device__ __forceinline__ int v_chunk(int key, int c)
{
    if (QW == 32) return c ^ (D == 64 ? (key & 2) << 1 : (key & 3) << 2);
    return c ^ (D == 64 ? (key & 6) : (key & 7) << 1);
}

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The exponent a row is scaled by: its largest finite value to 2^14 .. 2^15.
__device__ __forceinline__ int row_exp(float top) { return min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127); }

// over the lanes that hold a query: two of 32 queries, four of 16
template <int QW>
__device__ __forceinline__ float query_max(float v)
{
    if (QW == 16) {
        auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
template <int QW>
__device__ __forceinline__ float query_sum(float v)
{
    if (QW == 16) {
        auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
    auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// what a call of type T multiplies
template <class T> struct ApOperand { using E = _Float16; using V = half8; };
template <> struct ApOperand<TBF16> { using E = __bf16; using V = bf168; };

__device__ __forceinline__ f32x16 mfma(half8 a, half8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(bf168 a, bf168 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(bf168 a, bf168 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// a + b + c, rounded once (subnormal a and b count)
__device__ __forceinline__ float add_pair(_Float16 a, _Float16 b, float c)
{
    return __builtin_amdgcn_fdot2((half2v){a, b}, (half2v){1, 1}, c, false);
}
__device__ __forceinline__ float add_pair(__bf16 a, __bf16 b, float c)
{
    typedef __bf16 bf162v __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16((bf162v){a, b}, (bf162v){(__bf16)1.0f, (__bf16)1.0f}, c, false);
}

// ---------------------------------------------------------------- tiles ----
// A thread's part of a tile of K or V, NT threads: 8 channels of every ROWSth of
// its 32 rows.
template <class T, int D, int QW, int NT>
struct ApRows {
    using S = typename T::S;
    using E = typename ApOperand<T>::E;
    using V8 = typename ApOperand<T>::V;
    static constexpr int NS = sizeof(S) == 4 ? 2 : 1;
    static constexpr int CH = D / 8, ROWS = NT / CH, N = AP_KEYS / ROWS, PLANE = AP_KEYS * D;
    float x[N][8];

    // rows t0 .. t0 + 31 of a sequence of n, which begins at row a; zero behind its end
    template <bool ONCE>
    __device__ __forceinline__ void fetch(const ApArgs &A, bool v, int kvh, int a, int n, int t0)
    {
        const int c = threadIdx.x % CH;
        const S *base = (const S *)(v ? A.v : A.k) + kvh * (v ? A.vh : A.kh) + 8 * c;
        const int64_t stride = v ? A.vt : A.kt;
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int t = t0 + u * ROWS + (int)threadIdx.x / CH;
#pragma unroll
            for (int i = 0; i < 8; i++) x[u][i] = 0.0f;
            if (t < n) load8<T, ONCE>(base + (int64_t)(a + t) * stride, v ? A.v_vec : A.k_vec, x[u]);
        }
    }

    // into a tile's image and powers of two; odd: there was an infinity or a NaN, which
    // is left out and added where it is seen (V's, and those of K that have no two parts)
    __device__ __forceinline__ void lay(bool v, E *img, float *scale, int *odd)
    {
        const int c = threadIdx.x % CH;
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int key = u * ROWS + (int)threadIdx.x / CH;
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool fine = fabsf(x[u][i]) <= 3.402823466e38f;
                top = fmaxf(top, fine ? fabsf(x[u][i]) : 0.0f);
                if ((v || NS == 2) && !fine) *odd = 1, x[u][i] = 0.0f;
            }
            E *row = img + (v ? NS * PLANE : 0) + key * D + 8 * (v ? v_chunk<D, QW>(key, c) : k_chunk<D>(key, c));
            V8 hi, lo;
            if constexpr (NS == 2) {
                const int e = row_exp(group_max<CH>(top));
                const float up = pow2i(14 - e);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    half2v p, q;
                    split2(x[u][i] * up, x[u][i + 1] * up, &p, &q);
                    hi[i] = p[0], hi[i + 1] = p[1], lo[i] = q[0], lo[i + 1] = q[1];
                }
                *(V8 *)(row + PLANE) = lo;
                if (c == 0) scale[(v ? AP_KEYS : 0) + key] = pow2i(e - 14);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) hi[i] = (E)x[u][i];
            }
            *(V8 *)row = hi;
        }
    }
};

template <class T, int D, int QW>
__global__ void __launch_bounds__(AP_WG) prompt_tiles_kernel(ApArgs A)
{
    using R = ApRows<T, D, QW, AP_WG>;
    int seq, part, a, n;
    if (!ap_find(A, blockIdx.x, AP_KEYS, false, &seq, &part, &a, &n)) return;
    const int kvh = blockIdx.y;
    const int64_t tile = (int64_t)kvh * A.tiles + a / AP_KEYS + seq + part;
    const bool v = blockIdx.z;                     // K's image, or V's
    int odd = 0;
    R rows;
    rows.template fetch<true>(A, v, kvh, a, n, part * AP_KEYS);
    rows.lay(v, (typename R::E *)A.img + tile * 2 * R::NS * R::PLANE, A.scale + tile * 2 * AP_KEYS, &odd);
    if (v || R::NS == 2) {
        odd = __syncthreads_or(odd);
        if (threadIdx.x == 0) A.flags[2 * tile + v] = odd ? 1 : 0;
    }
}

// ------------------------------------------------------------- attention ----
// NW waves of QW queries; KT tiles of keys to a barrier; LDS read AHEAD steps
// ahead of the products; WE waves to a SIMD.  DIRECT: no tiles were laid out; the
// workgroup takes K and V as they are and lays each tile out in LDS itself.
template <class T, int D, int NW, int QW, int KT, int AHEAD, int WE, bool DIRECT>
__global__ void __launch_bounds__(64 * NW, WE) attn_prompt_kernel(ApArgs A)
{
    using S = typename T::S;
    using E = typename ApOperand<T>::E;
    using V8 = typename ApOperand<T>::V;
    constexpr int NS = sizeof(S) == 4 ? 2 : 1;
    constexpr int PLANE = AP_KEYS * D;
    constexpr int TILE = 2 * NS * PLANE;          // values of a tile, K and V
    // a product takes KW channels of 32 (QW = 16: twice 16) keys, or PK keys of QW channels
    using Acc = std::conditional_t<QW == 32, f32x16, f32x4>;
    constexpr int R = QW == 32 ? 16 : 4;          // values of it in a lane
    constexpr int NA = 32 / QW, NV = QW / 2;      // such scores of a tile, and a lane's scores
    constexpr int KW = QW == 32 ? 16 : 32, KS = D / KW;
    constexpr int DT = D / QW;                    // QW-channel parts of the output
    constexpr int PK = KW, PS = 32 / PK;
    constexpr int ROWS = QW * NW;
    static_assert(!DIRECT || KT == 1, "tiles are laid out one at a time");
    __shared__ __attribute__((aligned(16))) E lds[2][KT * TILE];
    __shared__ __attribute__((aligned(16))) float lsc[2][NS == 2 ? KT * 2 * AP_KEYS : 4];

    // Workgroups go to the 8 XCDs in turn.  An XCD takes consecutive eighths of
    // heads (a head's units counted from its longest rows, every eighth), so that
    // it finds the K and V its heads share in its L2, and goes through all of
    // them from the longest rows to the shortest.
    const unsigned heads = (unsigned)(A.n_kv * A.G), i8 = blockIdx.x >> 3, v8 = (blockIdx.x & 7) * heads + i8 % heads;
    const int head = (int)(v8 >> 3), unit = (int)(8 * (i8 / heads) + (v8 & 7)), kvh = head / A.G;
    int seq, part, a, len;
    if (!ap_find(A, unit, ROWS, true, &seq, &part, &a, &len)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), n = lane & (QW - 1), h = lane / QW;
    const int q0 = part * ROWS + wave * QW, qi = q0 + n;      // the wave's first query, the lane's

    const int64_t tile0 = (int64_t)kvh * A.tiles + a / AP_KEYS + seq;
    const int tiles = (min(part * ROWS + ROWS, len) + AP_KEYS - 1) / AP_KEYS;
    const uint4 *src = (const uint4 *)((const E *)A.img + tile0 * TILE);
    constexpr int PIECES = KT * TILE * (int)sizeof(E) / 16;
    auto load = [&](int step, int b) {
        // 1 KB of the image per wave and instruction, straight into LDS
#pragma unroll
        for (int i = 0; i < PIECES / (64 * NW); i++) {
            const int at = i * 64 * NW + wave * 64;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src + (int64_t)step * PIECES + at + lane),
                                             (__attribute__((address_space(3))) void *)((uint4 *)lds[b] + at), 16, 0, 0);
        }
        // their powers of two, a wave for a tile's 64, the same way (through a register the
        // wave waited here for the whole step)
        if constexpr (NS == 2)
            if (wave < KT)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void *)(A.scale + ((tile0 + (int64_t)step * KT + wave) * 64 + lane)),
                    (__attribute__((address_space(3))) void *)(lsc[b] + wave * 64), 4, 0, 0);
    };
    ApRows<T, D, QW, 64 * NW> kr, vr;
    if constexpr (DIRECT) {
        kr.template fetch<false>(A, false, kvh, a, len, 0);
        vr.template fetch<false>(A, true, kvh, a, len, 0);
    } else {
        load(0, 0);
    }
    // ---- queries; a negative scale turns their sign, none makes them zero (the
    // scores are multiplied behind the mask, whose -inf has to stay)
    V8 qh[KS], ql[NS == 2 ? KS : 1];
    float rs = A.sc == 0.0f ? 1.0f : fabsf(A.sc);
    {
        const S *qp = (const S *)A.q + (int64_t)(a + min(qi, len - 1)) * A.qt + head * A.qh;
        const float sign = A.sc == 0.0f ? 0.0f : A.sc < 0.0f ? -1.0f : 1.0f;
        if constexpr (NS == 2) {
            float x[KS][8], top = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                load8<T>(qp + KW * k + 8 * h, A.q_vec, x[k]);
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[k][i]));
            }
            const int e = row_exp(query_max<QW>(top));
            const float up = sign * pow2i(14 - e);
            rs *= pow2i(e - 14);
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    half2v a, b;
                    split2(x[k][i] * up, x[k][i + 1] * up, &a, &b);
                    qh[k][i] = a[0], qh[k][i + 1] = a[1], ql[k][i] = b[0], ql[k][i + 1] = b[1];
                }
        } else {
#pragma unroll
            for (int k = 0; k < KS; k++) {
                float x[8];
                load8<T>(qp + KW * k + 8 * h, A.q_vec, x);
#pragma unroll
                for (int i = 0; i < 8; i++) qh[k][i] = (E)(x[i] * sign);
            }
        }
    }

    Acc o[DT];
    // 16-bit calls: what is taken from the scores ahead of the scale.  Zero, unless scores are so large
    // that the maximum's own rounding (8 and more beyond 2^27) would be the weights' exponent.
    float ms = 0.0f;
    bool large = false;                            // a query of the wave has one
    float m = -3.402823466e38f, l = 0.0f;          // running maximum (of scaled scores), sum
    // fp32 calls: a weight's operand is p times V's power of two, 2^(7 - ve) of it: below 2^16, and near
    // there to keep its bits
    int ve = -110;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < R; i++) o[d][i] = 0.0f;

    // a lane's places in a tile: its chunk of K's row n, four keys of 16 channels
    // of V to every 16 lanes
    constexpr int KV = QW == 32 ? 8 : 4, VV = QW == 32 ? 4 : 8;      // places that differ by more than a constant
    int k_at[KV], v_at[VV];
#pragma unroll
    for (int i = 0; i < KV; i++) k_at[i] = n * D + 8 * k_chunk<D>(n, (KW / 8 * i + h) % (D / 8));
#pragma unroll
    for (int i = 0; i < VV; i++) {
        const int key = 4 * h + ((lane & 15) >> 2), c = QW * i + (QW == 32 ? ((lane >> 4) & 1) * 16 : 0) + (lane & 3) * 4;
        v_at[i] = NS * PLANE + key * D + 8 * v_chunk<D, QW>(key, c >> 3) + (c & 7);
    }

    // One tile of 32 keys from t0; EDGE: the one that holds the wave's own tokens; odd: fp32 calls, K
    // holds an infinity or a NaN.
    auto tile = [&](const E *K, const float *sc, int t0, bool odd, auto EDGE) {
        // ---- scores
        Acc sa[NA];
#pragma unroll
        for (int w = 0; w < NA; w++)
#pragma unroll
            for (int i = 0; i < R; i++) sa[w][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int w = 0; w < NA; w++) {
                const E *p = K + k_at[k % KV] + 128 * (k / KV) + w * 16 * D;
                const V8 kh = *(const V8 *)p;
                if constexpr (NS == 2) {
                    const V8 kl = *(const V8 *)(p + PLANE);
                    sa[w] = mfma(kh, ql[k], sa[w]);
                    sa[w] = mfma(kl, qh[k], sa[w]);
                }
                sa[w] = mfma(kh, qh[k], sa[w]);
            }
        // K is read AHEAD steps ahead of its products
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * NS, 0);
#pragma unroll
        for (int k = 0; k < KS * NA - AHEAD; k++) {
            __builtin_amdgcn_sched_group_barrier(0x008, NS == 2 ? 3 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, NS, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * (NS == 2 ? 3 : 1), 0);
        float s[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) s[i] = sa[i / R][i % R];
        constexpr int KG = QW == 32 ? 8 : 16;      // a lane's keys: KG g + 4 h + 0 .. 3
        if constexpr (NS == 2) {
#pragma unroll
            for (int g = 0; g < NV / 4; g++) {
                const float4 ks = *(const float4 *)(sc + KG * g + 4 * h);
                // (one after the other: together the two may leave the range, and 0 times that is no score)
                s[4 * g] = s[4 * g] * rs * ks.x, s[4 * g + 1] = s[4 * g + 1] * rs * ks.y;
                s[4 * g + 2] = s[4 * g + 2] * rs * ks.z, s[4 * g + 3] = s[4 * g + 3] * rs * ks.w;
            }
            if (odd) {
                // what was left out of the scores, by the definition
                int key = t0 + 4 * h, row = min(qi, len - 1);
                asm volatile("" : "+v"(key), "+v"(row));       // (formed here: the registers do not hold addresses across tiles)
                const float *qp = (const float *)A.q + (int64_t)(a + row) * A.qt + head * A.qh;
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const float *kp = (const float *)A.k + (int64_t)(a + min(key, len - 1)) * A.kt + kvh * A.kh;
                    float x = 0.0f;
#pragma unroll 1
                    for (int c = 0; c < D; c++)
                        if (!(fabsf(kp[c]) <= 3.402823466e38f)) x = fmaf(kp[c] * A.sc, qp[c], x);
                    s[i] += x;
                    key += (i & 3) == 3 ? KG - 3 : 1;
                    asm volatile("" : "+v"(key));
                }
            }
        }
        if constexpr (EDGE.value) {                // (keys behind the end are behind every query)
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const bool seen = KG * (i >> 2) + 4 * h + (i & 3) <= qi % AP_KEYS;
                s[i] = seen ? s[i] : -INFINITY;
            }
        }
        // ---- weights, by the maximum so far.  Whether it has to move is seen from
        // their sum, which is needed in any case: past 2^8 times the largest weight after a
        // move (an infinity included).  That is 2^LIFT: 2^7 in fp16, where 2^15 is still in
        // range, and weights down to 2^-32 of it are more than nothing (with 1 they ended at
        // 2^-25, which thousands of keys together can reach); 2^-32 in bf16, whose values
        // reach 2^128: their sums over 2^22 keys stay in fp32's range, those of 2^-94 and more
        // in its normal one.
        constexpr float LIFT = std::is_same_v<T, TF16> ? 7.0f : NS == 1 ? -32.0f : 0.0f;
        constexpr float FULL = std::is_same_v<T, TF16> ? 0x1p15f : NS == 1 ? 0x1p-24f : 0x1p8f;
        const float r = NS == 2 ? 1.0f : rs;
        float p[NV], w[NS == 2 ? NV : 1], sum = 0.0f, far = 0.0f;    // w: times V's powers of two
        if constexpr (NS == 1)
            if (large) {
#pragma unroll
                for (int i = 0; i < NV; i++) s[i] -= ms;
            }
        // (16-bit calls sum the weights as they are rounded for the second product: a row is a mean of
        // values, of one key that key's value, and none leaves the type's range)
        V8 ph[PS], pl[NS == 2 ? PS : 1];
        auto weigh = [&] {
            sum = far = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; i++) p[i] = __builtin_amdgcn_exp2f(NS == 2 ? s[i] - m : fmaf(s[i], r, -m));
#pragma unroll
            for (int i = 0; i < NV; i += NS == 2 ? 1 : 2) {
                if constexpr (NS == 2) {
                    sum += p[i];
                    w[i] = p[i] * sc[AP_KEYS + KG * (i >> 2) + 4 * h + (i & 3)];
                    far = fmaxf(far, w[i]);
                } else {
                    ph[i >> 3][i & 7] = (E)p[i], ph[i >> 3][(i & 7) + 1] = (E)p[i + 1];
                    sum = add_pair(ph[i >> 3][i & 7], ph[i >> 3][(i & 7) + 1], sum);
                }
            }
        };
        weigh();
        // fp32 calls: nor may an operand pass 2^15.  Its power of two follows the largest w, not V's
        // largest: a key of large values and no weight takes no bits from the others.
        if (__any(sum > FULL || (NS == 2 && far > pow2i(min(ve + 8, 127))))) {
            float top = s[0];
#pragma unroll
            for (int i = 1; i < NV; i++) top = fmaxf(top, s[i]);
            top = query_max<QW>(top);
            // (a query that need not move stays: what others see has no part in its rounding)
            const bool moves = query_max<QW>(sum) > FULL, wide = NS == 2 && query_max<QW>(far) > pow2i(min(ve + 8, 127));
            const float was = m;
            m = moves ? fmaxf(m, top * r - LIFT) : m;
            float f = __builtin_amdgcn_exp2f(was - m);
            l *= f;
            if constexpr (NS == 1)
                if (__any(moves && fabsf(m) > 0x1p24f)) {
                    const float by = moves && fabsf(m) > 0x1p24f ? top : 0.0f;
                    m = by != 0.0f ? -LIFT : m;
                    ms += by;
                    large = true;
#pragma unroll
                    for (int i = 0; i < NV; i++) s[i] -= by;
                }
            weigh();
            if constexpr (NS == 2) {
                // what is summed so far shrinks with the maximum's move, and its power of two with it
                const int sunk = ve - (int)fminf(m - was, 400.0f), here = (int)(__float_as_uint(query_max<QW>(far)) >> 23) - 126;
                const int e = moves || wide ? max(max(sunk, here), -110) : ve;
                f = __builtin_amdgcn_exp2f(was - m + (float)(ve - e));
                ve = e;
            }
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < R; i++) o[d][i] *= f;
        }
        l += sum;
        const float pv = NS == 2 ? pow2i(7 - ve) : 1.0f;
        if constexpr (NS == 2)
#pragma unroll
            for (int i = 0; i < NV; i += 2) {
                half2v a, b;
                split2(w[i] * pv, w[i + 1] * pv, &a, &b);
                ph[i >> 3][i & 7] = a[0], ph[i >> 3][(i & 7) + 1] = a[1];
                pl[i >> 3][i & 7] = b[0], pl[i >> 3][(i & 7) + 1] = b[1];
            }
        // ---- output
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int st = 0; st < PS; st++) {
                union { s16x4 r[2]; V8 v; } vh, vl;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const E *p = K + v_at[d % VV] + 128 * (d / VV) + (PK * st + KG * u) * D;
                    vh.r[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
                    if constexpr (NS == 2)
                        vl.r[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p + PLANE));
                }
                if constexpr (NS == 2) {
                    o[d] = mfma(vh.v, pl[st], o[d]);
                    o[d] = mfma(vl.v, ph[st], o[d]);
                }
                o[d] = mfma(vh.v, ph[st], o[d]);
            }
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * 2 * NS, 0);
#pragma unroll
        for (int k = 0; k < PS * DT - AHEAD; k++) {
            __builtin_amdgcn_sched_group_barrier(0x008, NS == 2 ? 3 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * NS, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * (NS == 2 ? 3 : 1), 0);
    };

    const int mine = q0 < len ? q0 / AP_KEYS : -1;           // the wave's last tile
    const int steps = (tiles + KT - 1) / KT;
    // (as constants: scalar loads, which wait for no step)
    const auto *flags = (const __attribute__((address_space(4))) int *)(uintptr_t)(A.flags + 2 * tile0);
    int flag[KT];
#pragma unroll
    for (int i = 0; i < KT; i++) flag[i] = NS == 2 && !DIRECT ? flags[2 * i] : 0;
    unsigned long long odd = 0;                    // DIRECT: tiles whose V holds an infinity or a NaN
    for (int step = 0; step < steps; step++) {
        const int b = step & 1;
        int next[KT] = {};
        if constexpr (DIRECT) {
            int here = 0;
            kr.lay(false, lds[b], lsc[b], &here);
            vr.lay(true, lds[b], lsc[b], &here);
            flag[0] = __syncthreads_or(here);      // K's or V's
            if (flag[0]) odd |= 1ull << step;
            if (step + 1 < steps) {
                kr.template fetch<false>(A, false, kvh, a, len, (step + 1) * AP_KEYS);
                vr.template fetch<false>(A, true, kvh, a, len, (step + 1) * AP_KEYS);
            }
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int i = 0; i < KT; i++) next[i] = NS == 2 ? flags[2 * ((step + 1) * KT + i)] : 0;
            if (step + 1 < steps) load(step + 1, b ^ 1);
        }
#pragma unroll
        for (int i = 0; i < KT; i++) {
            const int kt = step * KT + i;
            const float *sc = lsc[b] + (NS == 2 ? i * 2 * AP_KEYS : 0);
            if (kt < mine) tile(lds[b] + i * TILE, sc, kt * AP_KEYS, NS == 2 && flag[i], std::false_type{});
            else if (kt == mine) tile(lds[b] + i * TILE, sc, kt * AP_KEYS, NS == 2 && flag[i], std::true_type{});
        }
#pragma unroll
        for (int i = 0; i < KT; i++) flag[i] = next[i];
    }
    // ---- infinities and NaN of V, to the rows that see them: whatever else a
    // row sums, they decide its result, so they are added to it at the end
    const float inv = 1.0f / query_sum<QW>(l);          // every row sees itself
    constexpr int CG = QW == 32 ? 8 : 0;           // a lane's channels: QW d + CG g + 4 h + 0 .. 3
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < R; i++) o[d][i] *= inv;
    for (int t0 = 0; t0 <= mine; t0 += 64) {       // (64 flags to a load: one after the other they took longer than a tile)
        if constexpr (DIRECT) odd = mine < 0 ? 0 : odd & (~0ull >> (63 - mine));
        else odd = __ballot(t0 + lane <= mine && A.flags[2 * (tile0 + t0 + lane) + 1]);
        for (; odd; odd &= odd - 1) {
            const int k0 = (t0 + __ffsll(odd) - 1) * AP_KEYS, k1 = min(min(k0 + AP_KEYS, qi + 1), len);
            for (int k = k0; k < k1; k++) {
                const S *vr = (const S *)A.v + (int64_t)(a + k) * A.vt + kvh * A.vh;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int i = 0; i < R; i++) {
                        const float x = T::up(vr[QW * d + CG * (i >> 2) + 4 * h + (i & 3)]);
                        o[d][i] += fabsf(x) <= 3.402823466e38f ? 0.0f : x;
                    }
            }
        }
    }
    if (qi >= len) return;
    S *op = (S *)A.out + (int64_t)(a + qi) * A.ot + head * A.oh;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int g = 0; g < R / 4; g++) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = NS == 2 ? ldexpf(o[d][4 * g + i], ve - 7) : o[d][4 * g + i];
            store4<T>(op + QW * d + CG * g + 4 * h, A.o_vec, y);
        }
}

template <class T, int D, int NW, int QW, int KT, int AHEAD, int WE, bool DIRECT = false>
static int ap_run(ApArgs A, hipStream_t s)
{
    constexpr int NS = sizeof(typename T::S) == 4 ? 2 : 1;
    constexpr size_t TILE = 2 * NS * AP_KEYS * D * 2;
    A.tiles = A.T / AP_KEYS + A.n_seq;
    const int filled = A.T < A.n_seq ? A.T : A.n_seq;      // sequences that can hold a token
    const size_t n = (size_t)A.tiles * A.n_kv + 8;         // a barrier's tiles may reach past the last one
    const int64_t wgs = (((int64_t)A.T / (QW * NW) + filled + 7) / 8 * 8) * A.n_kv * A.G;
    if (wgs > UINT32_MAX / (64 * NW)) return fail(QMAG_ERR_ARG, "attn_prompt: %lld workgroups", (long long)wgs);
    if constexpr (DIRECT) {
        attn_prompt_kernel<T, D, NW, QW, KT, AHEAD, WE, true><<<dim3((unsigned)wgs), 64 * NW, 0, s>>>(A);
        return QMAG_OK;
    }
    int st;
    uint8_t *ws = (uint8_t *)workspace(WS_ATTN, n * (TILE + (NS == 2 ? 2 * AP_KEYS * sizeof(float) : 0) + 2 * sizeof(int)), &st);
    if (st) return st;
    A.img = ws;
    A.scale = (float *)(ws + n * TILE);
    A.flags = (int *)(A.scale + (NS == 2 ? n * 2 * AP_KEYS : 0));
    prompt_tiles_kernel<T, D, QW><<<dim3((unsigned)(A.T / AP_KEYS + filled), (unsigned)A.n_kv, 2), AP_WG, 0, s>>>(A);
    attn_prompt_kernel<T, D, NW, QW, KT, AHEAD, WE, false><<<dim3((unsigned)wgs), 64 * NW, 0, s>>>(A);
    return QMAG_OK;
}

template <class T, int D>
static int ap_launch(const ApArgs &A, hipStream_t s)
{
    constexpr bool F32 = sizeof(typename T::S) == 4;
    // Few tokens: one launch, every workgroup lays its tiles out itself.  With / without:
    // one token 8.7 / 10.9 us (fp32, 16 heads of 256) and 4.9 / 7.2 (bf16, 32 of 128), 64
    // tokens 15.3 / 16.7 and 8.9 / 10.2, 128 tokens 27.7 / 21.4 and 12.1 / 11.3.  (The lengths
    // are the device's: of several prompts none is taken to have all tokens.)
    if (A.T <= (D == 64 ? 128 : D == 128 ? 96 : 64) * (A.n_seq > 1 ? 3 : 2) / 2)
        return ap_run<T, D, D == 256 ? 8 : 4, 16, 1, 3, 2, true>(A, s);
    // Few workgroups of 128 queries: 64 to a workgroup, which leaves twice as many.  With /
    // without, at these counts of the large ones: fp32, heads of 256: 208 125 / 132 us, 256
    // 191 / 163; of 128: 416 88 / 93, 512 130 / 124; of 64: 800 129 / 134, 960 174 / 173; 16
    // bits, of 256: 384 118 / 129, 640 277 / 272; of 128: 640 86 / 91, 768 117 / 112; of 64:
    // 960 80 / 88, 1600 182 / 180.
    const int64_t wgs = ((int64_t)A.T / 128 + (A.T < A.n_seq ? A.T : A.n_seq)) * A.n_kv * A.G;
    if (wgs < (int64_t)ctx().n_cu * (F32 ? 1024 / D : D == 64 ? 16 : 11) / 4)
        return ap_run<T, D, 4, 16, 1, 3, F32 && D == 256 ? 1 : 2>(A, s);
    // Where 32 queries to a wave need more registers than three waves to a SIMD have: 16, and 8 waves
    if constexpr (F32 || D == 256) return ap_run<T, D, 8, 16, D == 64 ? 2 : 1, F32 && D == 128 ? 2 : 3, F32 && D == 128 ? 4 : 2>(A, s);
    else return ap_run<T, D, 4, 32, D == 64 ? 2 : 1, 3, D == 64 ? 4 : 3>(A, s);
}

}  // namespace qmag

using namespace qmag;

extern "C" int qmag_attn_prompt_dev(int type, int head_dim, const qmag_heads *q, const qmag_heads *k, const qmag_heads *v,
                                    const qmag_heads *out, const int *cu, int n_seq, int T, float scale)
{
    int st;
    if (!q || !k || !v || !out) return fail(QMAG_ERR_ARG, "attn_prompt: null pointer");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(QMAG_ERR_ARG, "attn_prompt: head_dim %d (64, 128 or 256)", head_dim);
    if (T < 0 || T > QMAG_ATTN_MAX_TOKENS || n_seq < 0 || n_seq > QMAG_KV_MAX_SEQ)
        return fail(QMAG_ERR_ARG, "attn_prompt: T=%d n_seq=%d", T, n_seq);
    if ((st = check_heads("attn_prompt q", q, type, head_dim, T, false))) return st;
    if ((st = check_heads("attn_prompt k", k, type, head_dim, T, false))) return st;
    if ((st = check_heads("attn_prompt v", v, type, head_dim, T, false))) return st;
    if ((st = check_heads("attn_prompt out", out, type, head_dim, T, true))) return st;
    if (k->n_head < 1 || k->n_head != v->n_head || q->n_head < 1 || q->n_head != out->n_head || q->n_head % k->n_head)
        return fail(QMAG_ERR_ARG, "attn_prompt: %d query, %d key, %d value and %d output heads", q->n_head, k->n_head,
                    v->n_head, out->n_head);
    if (T > 0 && n_seq > 0 && (!cu || (uintptr_t)cu % 4)) return fail(QMAG_ERR_ARG, "attn_prompt: cu is null or not aligned");
    const int size = attn_type_size(type);
    if (heads_overlap(q, out, size, head_dim, T) || heads_overlap(k, out, size, head_dim, T) ||
        heads_overlap(v, out, size, head_dim, T))
        return fail(QMAG_ERR_ARG, "attn_prompt: the output overlaps an input");
    if (T > 0 && n_seq > 0 && heads_meet(out, size, head_dim, T, cu, sizeof(int) * (size_t)(n_seq + 1)))
        return fail(QMAG_ERR_ARG, "attn_prompt: the output overlaps cu");
    if ((st = require_ready())) return st;
    if (T == 0 || n_seq == 0) return QMAG_OK;
    DeviceScope dev;
    if (dev.st) return dev.st;
    ApArgs A = {};
    A.q = q->ptr, A.k = k->ptr, A.v = v->ptr, A.out = out->ptr;
    A.qt = q->token_stride, A.qh = q->head_stride, A.kt = k->token_stride, A.kh = k->head_stride;
    A.vt = v->token_stride, A.vh = v->head_stride, A.ot = out->token_stride, A.oh = out->head_stride;
    A.cu = cu;
    A.n_seq = n_seq;
    A.T = T;
    A.n_kv = k->n_head;
    A.G = q->n_head / k->n_head;
    A.sc = scale * 1.44269504088896340736f;
    A.q_vec = heads_aligned(q, type), A.k_vec = heads_aligned(k, type), A.v_vec = heads_aligned(v, type);
    A.o_vec = heads_aligned(out, type);
    hipStream_t s = ctx().stream;
    prof_begin(PROF_ATTN, s);
    st = with_type(type, [&](auto t) {
        using TT = decltype(t);
        if (head_dim == 64) return ap_launch<TT, 64>(A, s);
        if (head_dim == 128) return ap_launch<TT, 128>(A, s);
        return ap_launch<TT, 256>(A, s);
    });
    prof_end(PROF_ATTN, s);
    if (st) return st;
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}
