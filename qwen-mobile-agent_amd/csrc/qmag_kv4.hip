// qmag_kv4.hip -- tokens' K and V into the 4-bit cache, and the values it holds.
//
// 64 consecutive values of a head share a minimum m and a step d, both fp16:
//   m = fp16(min), d = fp16((max - min) * (1 / 15)), code = clamp(rne((x - m) / d), 0, 15),
// every step in fp32 as written, 1 / 15 itself rounded to fp32, so that the codes
// do not depend on who forms them.  (The product, not the quotient, is what a
// tensor library on this device forms for a division by a constant: for 16-bit
// values the quotient is now and then half way between two fp16 steps, where the
// two part.)  m and d saturate at fp16's largest value; a group that holds an
// infinity or a NaN stands for NaN throughout (d NaN).
//
// Append: a thread takes 8 values of one head of one token; a group is 8 threads,
// its minimum and maximum three lane exchanges.  Read: a thread takes 4 values, so
// that a wave writes 1 KB in one piece.  A workgroup stays with one head of K or V
// (a division by the number of heads in every thread, and stores of every other 16
// bytes, had cost more than the memory).  Memory bound: 16,001 tokens of 8 heads of
// 128, bf16, in (84 MB) 24.5 us, and back as fp32 (150 MB) 30 us; 7 tokens a launch
// each, 2.8 us.
#include "qmag_attn.h"

namespace qmag {

constexpr int KV4_WG = 256;

// where the 8 codes from channel 8 * e of a token's row lie (K: one dword)
template <int D>
__device__ __forceinline__ int k_dword_at(int e)
{
    const int g = e >> 3, s = (e >> 2) & 1, h = e & 3;
    return h * (D / 8) + g * 8 + s * 4;
}
// V: four channels each in 16 bits, channels 4 * i of group g
template <int D>
__device__ __forceinline__ int v_short_at(int g, int i)
{
    return i * (D / 32) + g * 2;
}

struct Kv4Args {
    uint8_t *data;
    int n_slot, shift, n_kv;
    int64_t half;                 // bytes of K, or of V, of a head in a block
};

template <class T, int D>
__global__ void __launch_bounds__(KV4_WG) kv4_append_kernel(Kv4Args c, qmag_heads K, qmag_heads V, const int *slot, int n_tok,
                                                            bool vec)
{
    constexpr int PER = D / 8;                       // threads of a head
    constexpr int ROWS = KV4_WG / PER;
    const int e = threadIdx.x % PER, g = e >> 3;
    const int is_v = (int)blockIdx.y >= c.n_kv, head = is_v ? (int)blockIdx.y - c.n_kv : (int)blockIdx.y;
    for (int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / PER; t < n_tok; t += (int64_t)gridDim.x * ROWS) {
        const int sl = slot[t];                      // whole groups of lanes go on together
        if (sl < 0 || sl >= c.n_slot) continue;
        const qmag_heads &H = is_v ? V : K;
        float x[8];
        // past the caches, which the codes need more (16,001 bf16 tokens in and back: 11 us of 70)
        load8<T, true>((const typename T::S *)H.ptr + t * H.token_stride + head * H.head_stride + 8 * e, vec, x);
        float lo = x[0], hi = x[0];
        float none = 0.0f;                         // NaN with an infinity or a NaN in it
#pragma unroll
        for (int i = 0; i < 8; i++) {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
            none = fmaf(x[i], 0.0f, none);
        }
        lo = group_min<8>(lo);
        hi = group_max<8>(hi);
        const bool group_ok = group_sum<8>(none) == 0.0f;
        const _Float16 m = (_Float16)fminf(fmaxf(lo, -65504.0f), 65504.0f);
        const _Float16 d = (_Float16)fminf((hi - lo) * (1.0f / 15.0f), 65504.0f);
        const float mf = (float)m, df = (float)d;
        const bool step = group_ok && df > 0.0f;
        const float rd = step ? 1.0f / df : 0.0f, most = step ? 15.0f * df : 0.0f;      // no step: every code 0
        float code[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // the quotient t / d, rounded as a division rounds it: the residual of t (1 / d) is exact, and
            // with d of 11 bits t / d is never so near to half way that its correction's rounding
            // counts.  (Eight divisions had taken more time than the memory: 31 us against 24.)
            const float t = __builtin_amdgcn_fmed3f(x[i] - mf, 0.0f, most);
            const float q = t * rd;
            code[i] = rintf(fmaf(fmaf(-q, df, t), rd, q));
        }
        // four codes side by side are a whole number that fp32 holds
        uint32_t half[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
            half[i] = (uint32_t)fmaf(fmaf(fmaf(code[4 * i + 3], 16.0f, code[4 * i + 2]), 16.0f, code[4 * i + 1]), 16.0f, code[4 * i]);
        const uint32_t dword = half[0] | half[1] << 16;
        const int64_t blk = sl >> c.shift;
        const int off = sl & ((1 << c.shift) - 1);
        uint8_t *base = c.data + (blk * c.n_kv + head) * 2 * c.half + (is_v ? c.half : 0);
        uint8_t *codes = base + off * (D / 2);
        if (!is_v) {
            *(uint32_t *)(codes + k_dword_at<D>(e)) = dword;
        } else if constexpr (D == 64) {
            *(uint32_t *)(codes + v_short_at<D>(0, 2 * e)) = dword;
        } else {
            // two groups' words of a place lie side by side: one of the two from the thread 8 on
            const uint32_t o = (uint32_t)__shfl_xor((int)dword, 8);
            const uint32_t both = g & 1 ? (o >> 16) | (dword & 0xFFFF0000u) : (dword & 0xFFFFu) | (o << 16);
            *(uint32_t *)(codes + v_short_at<D>(g & ~1, 2 * (e & 7) + (g & 1))) = both;
        }
        if ((e & 7) == 0) {
            const uint32_t dm = group_ok ? (uint32_t)__builtin_bit_cast(uint16_t, d) |
                                               ((uint32_t)__builtin_bit_cast(uint16_t, m) << 16)
                                         : 0x7E00u;
            *(uint32_t *)(base + ((int64_t)(D / 2) << c.shift) + (off * (D / KV4_GROUP) + g) * 4) = dm;
        }
    }
}

template <int D>
__global__ void __launch_bounds__(KV4_WG) kv4_read_kernel(Kv4Args c, const int *slot, int n_tok, float *ko, float *vo, bool vec)
{
    constexpr int PER = D / 4;                       // threads of a head
    constexpr int ROWS = KV4_WG / PER;
    const int e = threadIdx.x % PER, g = e >> 4;
    const int is_v = (int)blockIdx.y >= c.n_kv, head = is_v ? (int)blockIdx.y - c.n_kv : (int)blockIdx.y;
    const int word_at = is_v ? v_short_at<D>(g, e & 15) : k_dword_at<D>(e >> 1) + 2 * (e & 1);
    float *out = (is_v ? vo : ko) + head * D + 4 * e;
    for (int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / PER; t < n_tok; t += (int64_t)gridDim.x * ROWS) {
        const int sl = slot[t];
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (sl >= 0 && sl < c.n_slot) {
            const int64_t blk = sl >> c.shift;
            const int off = sl & ((1 << c.shift) - 1);
            const uint8_t *base = c.data + (blk * c.n_kv + head) * 2 * c.half + (is_v ? c.half : 0);
            const uint32_t w = *(const uint16_t *)(base + off * (D / 2) + word_at);
            const uint32_t dm = *(const uint32_t *)(base + ((int64_t)(D / 2) << c.shift) + (off * (D / KV4_GROUP) + g) * 4);
            const float d = h2f(dm & 0xFFFFu), m = h2f(dm >> 16);
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = fmaf(d, (float)((w >> (4 * i)) & 15u), m);
        }
        // past the caches: nothing here is read again (46 us for 131 MB by way of them, 27 so)
        if (vec) __builtin_nontemporal_store((f32x4){y[0], y[1], y[2], y[3]}, (f32x4 *)(out + t * (c.n_kv * D)));
        else store4<TF32>(out + t * (c.n_kv * D), false, y);
    }
}

static Kv4Args kv4_args(const qmag_kv4 *c)
{
    int shift = 0;
    while ((1 << shift) < c->block_size) shift++;
    return {(uint8_t *)c->data, c->n_block * c->block_size, shift, c->n_kv, kv4_half_bytes(c->block_size, c->head_dim)};
}

template <class F>
static int with_dim(int dim, F f)
{
    if (dim == 64) return f(std::integral_constant<int, 64>{});
    if (dim == 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}

// workgroups for T tokens of every head of K and V, `per` tokens each at a time
static dim3 kv4_grid(int T, int n_kv, int per)
{
    const int64_t x = ((int64_t)T + per - 1) / per, most = 8192 / (2 * n_kv) + 1;
    return dim3((unsigned)(x < most ? x : most), (unsigned)(2 * n_kv));
}

}  // namespace qmag

using namespace qmag;

extern "C" int qmag_kv4_block_bytes(const qmag_kv4 *c, size_t *bytes)
{
    if (!c || !bytes) return fail(QMAG_ERR_ARG, "kv4_block_bytes: null pointer");
    qmag_kv4 shape = *c;
    shape.data = (void *)16;             // the shape alone is asked for
    if (shape.n_block < 1) shape.n_block = 1;
    int st = check_kv4(&shape);
    if (st) return st;
    *bytes = (size_t)(2 * kv4_half_bytes(c->block_size, c->head_dim)) * (size_t)c->n_kv;
    return QMAG_OK;
}

extern "C" int qmag_kv4_append_dev(const qmag_kv4 *c, int type, const qmag_heads *k, const qmag_heads *v, const int *slot,
                                   int T)
{
    int st = check_kv4(c);
    if (st) return st;
    if (!k || !v || T < 0 || (T > 0 && (!slot || (uintptr_t)slot % 4)))
        return fail(QMAG_ERR_ARG, "kv4_append: T=%d or a null or unaligned pointer", T);
    if ((st = check_heads("kv4_append k", k, type, c->head_dim, T, false))) return st;
    if ((st = check_heads("kv4_append v", v, type, c->head_dim, T, false))) return st;
    if (k->n_head != c->n_kv || v->n_head != c->n_kv)
        return fail(QMAG_ERR_ARG, "kv4_append: %d and %d heads for a cache of %d", k->n_head, v->n_head, c->n_kv);
    if ((st = require_ready())) return st;
    if (T == 0) return QMAG_OK;
    const bool vec = heads_aligned(k, type) && heads_aligned(v, type);
    DeviceScope dev;
    if (dev.st) return dev.st;
    hipStream_t s = ctx().stream;
    const dim3 grid = kv4_grid(T, c->n_kv, KV4_WG / (c->head_dim / 8));
    prof_begin(PROF_KV, s);
    with_type(type, [&](auto t) {
        return with_dim(c->head_dim, [&](auto d) {
            kv4_append_kernel<decltype(t), decltype(d)::value><<<grid, KV4_WG, 0, s>>>(kv4_args(c), *k, *v, slot, T, vec);
            return 0;
        });
    });
    prof_end(PROF_KV, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}

extern "C" int qmag_kv4_read_dev(const qmag_kv4 *c, const int *slot, int T, float *k, float *v)
{
    int st = check_kv4(c);
    if (st) return st;
    if (T < 0 || (T > 0 && (!slot || !k || !v || ((uintptr_t)slot | (uintptr_t)k | (uintptr_t)v) % 4)))
        return fail(QMAG_ERR_ARG, "kv4_read: T=%d or a null or unaligned pointer", T);
    const qmag_heads ko = {k, c->n_kv, (int64_t)c->n_kv * c->head_dim, c->head_dim}, vo = {v, ko.n_head, ko.token_stride, ko.head_stride};
    if (heads_overlap(&ko, &vo, 4, c->head_dim, T)) return fail(QMAG_ERR_ARG, "kv4_read: k and v overlap");
    for (const qmag_heads &o : {ko, vo})
        if (heads_meet(&o, 4, c->head_dim, T, slot, sizeof(int) * (size_t)T) ||
            heads_meet(&o, 4, c->head_dim, T, c->data, kv4_bytes(c)))
            return fail(QMAG_ERR_ARG, "kv4_read: k or v overlaps the slots or the cache");
    if ((st = require_ready())) return st;
    if (T == 0) return QMAG_OK;
    const bool vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
    DeviceScope dev;
    if (dev.st) return dev.st;
    hipStream_t s = ctx().stream;
    const dim3 grid = kv4_grid(T, c->n_kv, KV4_WG / (c->head_dim / 4));
    prof_begin(PROF_KV, s);
    with_dim(c->head_dim, [&](auto d) {
        kv4_read_kernel<decltype(d)::value><<<grid, KV4_WG, 0, s>>>(kv4_args(c), slot, T, k, v, vec);
        return 0;
    });
    prof_end(PROF_KV, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}
