// qmag_rows.h -- what the units that take rows of activations share: loads and
// stores of whole 16 bytes wherever a row begins, ranges that must not meet.
#pragma once

#include "qmag_attn.h"

namespace qmag {

// N values of the type from p on, which is aligned to a value: global memory takes
// vectors at any such place.
template <class T, int N>
__device__ __forceinline__ void load_row(const typename T::S *p, float (&o)[N])
{
    constexpr int BYTES = N * (int)sizeof(typename T::S), STEP = BYTES < 16 ? BYTES : 16, PER = STEP / (int)sizeof(typename T::S);
    static_assert(BYTES % STEP == 0 && STEP % 4 == 0, "whole words");
    typedef uint32_t Words __attribute__((ext_vector_type(STEP / 4)));
    typedef uint32_t Loose __attribute__((ext_vector_type(STEP / 4), aligned(sizeof(typename T::S))));
    union Vec { Words u; typename T::S v[PER]; };
#pragma unroll
    for (int a = 0; a < N; a += PER) {
        Vec x;
        x.u = *(const QMAG_GLOBAL Loose *)(p + a);
#pragma unroll
        for (int i = 0; i < PER; i++) o[a + i] = T::up(x.v[i]);
    }
}
template <class T, int N>
__device__ __forceinline__ void store_row(typename T::S *p, const float (&v)[N])
{
    constexpr int BYTES = N * (int)sizeof(typename T::S), STEP = BYTES < 16 ? BYTES : 16, PER = STEP / (int)sizeof(typename T::S);
    static_assert(BYTES % STEP == 0 && STEP % 4 == 0, "whole words");
    typedef uint32_t Words __attribute__((ext_vector_type(STEP / 4)));
    typedef uint32_t Loose __attribute__((ext_vector_type(STEP / 4), aligned(sizeof(typename T::S))));
    union Vec { Words u; typename T::S v[PER]; };
#pragma unroll
    for (int a = 0; a < N; a += PER) {
        Vec x;
#pragma unroll
        for (int i = 0; i < PER; i++) x.v[i] = T::down(v[a + i]);
        *(QMAG_GLOBAL Loose *)(p + a) = x.u;
    }
}

// whether two ranges of bytes share one
inline bool ranges_meet(const void *a, size_t na, const void *b, size_t nb)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na && nb && x < y + nb && y < x + na;
}

}  // namespace qmag
