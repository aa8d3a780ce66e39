// Rows of logits on gfx950: values as ordered whole numbers, and pieces of eight of them.
#pragma once

#include "mx4_format.h"

namespace pimhip
{
// A value's place in the order of all values, as a whole number: -0 with 0, infinities at the ends.
__device__ __forceinline__ unsigned int ordered_bits(float v)
{
    const unsigned int b = __builtin_bit_cast(unsigned int, v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float from_ordered(unsigned int o) { return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// Eight values of a whole piece as fp32.
template <class T>
__device__ __forceinline__ void load_piece(const typename T::elem* row, int64_t piece, float (&v)[8])
{
    typename T::elem e[8];
    const uint4_any_t* p = reinterpret_cast<const uint4_any_t*>(row + piece * 8);
    if constexpr (sizeof(e[0]) == 2) {
        const uint4_t q = p[0];
        __builtin_memcpy(e, &q, 16);
    } else {
        const uint4_t q0 = p[0], q1 = p[1];
        __builtin_memcpy(e, &q0, 16);
        __builtin_memcpy(e + 4, &q1, 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)e[i];
}
}  // namespace pimhip
