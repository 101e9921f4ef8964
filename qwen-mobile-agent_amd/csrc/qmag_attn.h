// qmag_attn.h -- what the attention units share: the three activation types,
// heads in memory, the 4-bit cache's layout.
#pragma once

#include "qmag_internal.h"

namespace qmag {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf168 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct TF32 {
    using S = float;
    static constexpr int id = QMAG_TYPE_F32;
    __device__ static __forceinline__ float up(float v) { return v; }
    __device__ static __forceinline__ float down(float v) { return v; }
};
struct TF16 {
    using S = _Float16;
    static constexpr int id = QMAG_TYPE_F16;
    __device__ static __forceinline__ float up(_Float16 v) { return (float)v; }
    __device__ static __forceinline__ _Float16 down(float v) { return (_Float16)v; }     // to nearest even
};
struct TBF16 {
    using S = __bf16;
    static constexpr int id = QMAG_TYPE_BF16;
    __device__ static __forceinline__ float up(__bf16 v) { return (float)v; }
    __device__ static __forceinline__ __bf16 down(float v) { return (__bf16)v; }         // to nearest even
};

// bytes of a value of an activation type, 0 for any other type id
inline int attn_type_size(int type)
{
    return type == QMAG_TYPE_F32 ? 4 : type == QMAG_TYPE_F16 || type == QMAG_TYPE_BF16 ? 2 : 0;
}

// f(T{}) for the C++ type of a checked type id
template <class F>
int with_type(int type, F f)
{
    if (type == QMAG_TYPE_F32) return f(TF32{});
    if (type == QMAG_TYPE_F16) return f(TF16{});
    return f(TBF16{});
}

// a and b as fp16 (to nearest) in *hi, and what that leaves of them in *lo: two
// parts of 22 bits together.  *hi is held as the packed pair it is used as: left
// to itself the compiler converts a second time for the difference, and may then
// round the product behind a to fp16 at once on one side and by way of fp32 on
// the other, and where those fall to different sides of a step the parts no
// longer fit (2^-11 of a value, once in some thousand).
__device__ __forceinline__ void split2(float a, float b, half2v *hi, half2v *lo)
{
    uint32_t h = __builtin_bit_cast(uint32_t, (half2v){(_Float16)a, (_Float16)b});
    asm("" : "+v"(h));
    *hi = __builtin_bit_cast(half2v, h);
    *lo = (half2v){(_Float16)fmaf((float)(*hi)[0], -1.0f, a), (_Float16)fmaf((float)(*hi)[1], -1.0f, b)};
}

// Eight values from p; vec: p is 16-byte aligned; ONCE: they are not kept in the
// caches for others.
template <class T, bool ONCE = false>
__device__ __forceinline__ void load8(const typename T::S *p, bool vec, float (&o)[8])
{
    constexpr int N = 16 / (int)sizeof(typename T::S);
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    union Vec { u32x4 u; typename T::S v[N]; };
    if (vec) {
#pragma unroll
        for (int a = 0; a < 8; a += N) {
            Vec x;
            if constexpr (ONCE) x.u = __builtin_nontemporal_load((const u32x4 *)(p + a));
            else x.u = *(const u32x4 *)(p + a);
#pragma unroll
            for (int i = 0; i < N; i++) o[a + i] = T::up(x.v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = T::up(p[i]);
    }
}

// Four values to p; vec: p is aligned to four values.
template <class T>
__device__ __forceinline__ void store4(typename T::S *p, bool vec, const float (&v)[4])
{
    struct alignas(4 * sizeof(typename T::S)) Vec { typename T::S v[4]; };
    if (vec) {
        Vec x;
#pragma unroll
        for (int i = 0; i < 4; i++) x.v[i] = T::down(v[i]);
        *reinterpret_cast<Vec *>(p) = x;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = T::down(v[i]);
    }
}

// Inclusive sums over the wave, all lanes active: within rows of 16 lanes, then a
// row's last to the row behind it, then the lower half's to the upper.
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_move(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ long long scan_move(long long v)
{
    const uint32_t lo = (uint32_t)scan_move<CTRL, ROWS>((int)v);
    return (long long)((unsigned long long)(uint32_t)scan_move<CTRL, ROWS>((int)(v >> 32)) << 32 | lo);
}
template <class I>
__device__ __forceinline__ I wave_scan(I v)
{
    v += scan_move<0x111, 0xf>(v);
    v += scan_move<0x112, 0xf>(v);
    v += scan_move<0x114, 0xf>(v);
    v += scan_move<0x118, 0xf>(v);
    v += scan_move<0x142, 0xa>(v);
    v += scan_move<0x143, 0xc>(v);
    return v;
}

// ------------------------------------------------------------- host side --
// The device of the library current for the life of a call, whichever one the
// calling thread had.
struct DeviceScope {
    int was = -1;
    int st = QMAG_OK;
    DeviceScope();
    ~DeviceScope();
};

// QMAG_OK if h describes n_tok tokens of heads of `dim` values of the type,
// aligned to the values; written: no two of its values in one place (tokens
// of whole heads, or heads of whole tokens).
int check_heads(const char *what, const qmag_heads *h, int type, int dim, int64_t n_tok, bool written);
// whether the two may share a byte: false when their ranges are apart, or when
// they lie side by side within the tokens, or the heads, of one buffer; dim_b: the
// values of b's heads where they are others than a's
bool heads_overlap(const qmag_heads *a, const qmag_heads *b, int size, int dim, int64_t n_tok, int dim_b = 0);
// whether any of h's values lies in the `bytes` bytes from p
bool heads_meet(const qmag_heads *h, int size, int dim, int64_t n_tok, const void *p, size_t bytes);
// every head's first value 16-byte aligned
bool heads_aligned(const qmag_heads *h, int type);

// ------------------------------------------------------- the 4-bit cache --
// (the layout is described at qmag_kv4 in include/qma_gpu.h)
constexpr int KV4_GROUP = 64;
// bytes of one tensor (K or V) of one kv head in a block: codes, then scales
__host__ __device__ __forceinline__ constexpr int64_t kv4_half_bytes(int block, int dim)
{
    return (int64_t)block * (dim / 2 + dim / KV4_GROUP * 4);
}
inline size_t kv4_bytes(const qmag_kv4 *c)
{
    return (size_t)c->n_block * (size_t)c->n_kv * (size_t)(2 * kv4_half_bytes(c->block_size, c->head_dim));
}
int check_kv4(const qmag_kv4 *c);

}  // namespace qmag
