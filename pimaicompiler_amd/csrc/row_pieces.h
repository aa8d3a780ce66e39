// Rows of logits on gfx950: values as ordered whole numbers, pieces of eight of them, and what wavefronts make of 64-bit numbers.
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

// The larger of two keys over the LANES (1, 4 or 16) lanes of a group; every lane returns it.
template <int LANES>
__device__ __forceinline__ unsigned long long group_max_u64(unsigned long long k)
{
    auto with = [&](unsigned int hi, unsigned int lo) {
        const unsigned long long o = (unsigned long long)hi << 32 | lo;
        k = o > k ? o : k;
    };
    static_assert(LANES == 1 || LANES == 4 || LANES == 16, "a group is part of a row of 16 lanes");
    if constexpr (LANES >= 4) {
        with(dpp_u32<kDppQuadXor1>((unsigned int)(k >> 32)), dpp_u32<kDppQuadXor1>((unsigned int)k));
        with(dpp_u32<kDppQuadXor2>((unsigned int)(k >> 32)), dpp_u32<kDppQuadXor2>((unsigned int)k));
    }
    if constexpr (LANES == 16) {
        with(dpp_u32<kDppRowHalfMirror>((unsigned int)(k >> 32)), dpp_u32<kDppRowHalfMirror>((unsigned int)k));
        with(dpp_u32<kDppRowMirror>((unsigned int)(k >> 32)), dpp_u32<kDppRowMirror>((unsigned int)k));
    }
    return k;
}

// ---- 64-bit numbers over the lanes of a wavefront, on DPP (a generic shuffle of 64 bits takes two trips through the LDS crossbar) ----
static constexpr int kDppRowShr1 = 0x111;       // row_shr:1 (and on: 2, 4, 8)
static constexpr int kDppRowBcast15 = 0x142;    // lane 15 of each row to the row behind it
static constexpr int kDppRowBcast31 = 0x143;    // lane 31 to the two rows behind it

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v)  // 0 in lanes without a source, and in rows that are left out
{
    const unsigned int lo = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)(unsigned int)v, CTRL, ROWS, 0xf, true);
    const unsigned int hi = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)(unsigned int)(v >> 32), CTRL, ROWS, 0xf, true);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t readlane_u64(uint64_t v, int lane)
{
    const unsigned int lo = (unsigned int)__builtin_amdgcn_readlane((int)(unsigned int)v, lane), hi = (unsigned int)__builtin_amdgcn_readlane((int)(unsigned int)(v >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}
// The sum over the lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v)
{
    v += dpp_u64<kDppRowShr1>(v);
    v += dpp_u64<kDppRowShr1 + 1>(v);
    v += dpp_u64<kDppRowShr1 + 3>(v);
    v += dpp_u64<kDppRowShr1 + 7>(v);
    v += dpp_u64<kDppRowBcast15, 0xa>(v);
    v += dpp_u64<kDppRowBcast31, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint64_t wave_total_u64(uint64_t v) { return readlane_u64(wave_scan_u64(v), 63); }
__device__ __forceinline__ unsigned int wave_total_u32(unsigned int v)
{
    v += dpp_u32<kDppRowShr1>(v);
    v += dpp_u32<kDppRowShr1 + 1>(v);
    v += dpp_u32<kDppRowShr1 + 3>(v);
    v += dpp_u32<kDppRowShr1 + 7>(v);
    v += (unsigned int)__builtin_amdgcn_update_dpp(0, (int)v, kDppRowBcast15, 0xa, 0xf, true);
    v += (unsigned int)__builtin_amdgcn_update_dpp(0, (int)v, kDppRowBcast31, 0xc, 0xf, true);
    return (unsigned int)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ double wave_total_f64(double d)
{
    auto with = [&](uint64_t o) { d += __builtin_bit_cast(double, o); };
    with(dpp_u64<kDppRowShr1>(__builtin_bit_cast(uint64_t, d)));
    with(dpp_u64<kDppRowShr1 + 1>(__builtin_bit_cast(uint64_t, d)));
    with(dpp_u64<kDppRowShr1 + 3>(__builtin_bit_cast(uint64_t, d)));
    with(dpp_u64<kDppRowShr1 + 7>(__builtin_bit_cast(uint64_t, d)));
    with(dpp_u64<kDppRowBcast15, 0xa>(__builtin_bit_cast(uint64_t, d)));
    with(dpp_u64<kDppRowBcast31, 0xc>(__builtin_bit_cast(uint64_t, d)));
    return __builtin_bit_cast(double, readlane_u64(__builtin_bit_cast(uint64_t, d), 63));
}
__device__ __forceinline__ unsigned long long wave_max_u64(unsigned long long v)
{
    v = group_max_u64<16>(v);
    unsigned long long best = readlane_u64(v, 0);
#pragma unroll
    for (int i = 16; i < 64; i += 16) {
        const unsigned long long o = readlane_u64(v, i);
        best = o > best ? o : best;
    }
    return best;
}
}  // namespace pimhip
