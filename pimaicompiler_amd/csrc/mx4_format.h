// Microscaled 4-bit floating point on gfx950: the format's constants, the 16-bit types its products run on, and conversions.
//
// A row of K values lies in blocks of 32.  A value is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} (sign, two exponent bits, one mantissa
// bit), two to a byte, the first in the low half; a block has one scale 2^(code - 127) in a byte, code 255 meaning "not a
// number".  The last block of a row is filled up with zeros.
#pragma once

#include "device_common.h"

namespace pimhip
{
typedef __bf16 bf16_t;
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned int uint4_t __attribute__((ext_vector_type(4)));
typedef unsigned int uint2_t __attribute__((ext_vector_type(2)));
typedef uint4_t uint4_any_t __attribute__((aligned(2)));  // sixteen bytes at any address a 16-bit value may have
typedef uint2_t uint2_any_t __attribute__((aligned(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef int int8v_t __attribute__((ext_vector_type(8)));

static constexpr int kMxBlock = 32;        // values that share a scale
static constexpr int kMxBlockBytes = 16;   // their packed bytes
static constexpr unsigned int kMxNan = 255u;

// 2^(code - 127) as a float: code 0 is the subnormal 2^-127, code 255 a NaN.
__device__ __forceinline__ float mx_scale_f32(unsigned int code)
{
    const unsigned int bits = code == kMxNan ? 0x7fc00000u : code << 23;
    return __builtin_bit_cast(float, bits > 0x00400000u ? bits : 0x00400000u);
}

// The 16-bit types of activations.  `scale` of a block in a row of 4-bit weights that meets them on the matrix cores:
//   bfloat16 has the range of every scale but the two largest, whose elements 4 and 6, or 2 to 6, are above it: elements are converted
//   with their block's own scale, exactly; in a row whose largest code is 253 or 254 with a half or a quarter of it, which the sum is
//   multiplied by at the end (such a row's blocks of codes 0 and 1, 2^-252 of its largest, come out larger by that).
//   fp16 has not.  Elements are converted relative to the row's largest scale code `top` (the largest element is below 2^15 then),
//   and the sum is multiplied by 2^(top - 127 - 12) at the end.  Exact for blocks down to 2^-35 of the row's largest scale; what is
//   further below loses bits that are under 2^-38 of the row's largest value.
struct F16 {
    typedef half_t elem;
    typedef half8_t frag;
    static constexpr int kLift = 12;
    static __device__ __forceinline__ float4_t mfma(const frag a, const frag b, const float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    // The power of two that a row's sums are multiplied by.
    static __device__ __forceinline__ int exponent(int top) { return top - 127 - kLift; }
    static __device__ __forceinline__ float scale(unsigned int code, int top)
    {
        // (no code is above its row's top, and 254 stands for one that was written there later: 255 is the exponent of infinities and NaN)
        const int e = (int)code - top + 127 + kLift;
        return __builtin_bit_cast(float, code == kMxNan ? 0x7fc00000u : (unsigned int)(e < 0 ? 0 : e > 254 ? 254 : e) << 23);
    }
    static __device__ __forceinline__ frag from_mx4(unsigned int d, float s)
    {
        const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, s, 1);
        const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, s, 3);
        return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
    }
    static __device__ __forceinline__ elem round(float v) { return round_f16(v); }
};

struct BF16 {
    typedef bf16_t elem;
    typedef bf16x8_t frag;
    static __device__ __forceinline__ float4_t mfma(const frag a, const frag b, const float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int exponent(int top) { return top > 252 ? top - 252 : 0; }
    static __device__ __forceinline__ float scale(unsigned int code, int top)
    {
        const int lower = (int)code - top + 252;
        const int bits = (lower < (int)code ? lower : (int)code) * (1 << 23);  // (below 2^-127: 2^-127)
        return __builtin_bit_cast(float, code == kMxNan ? 0x7fc00000 : bits > 0x00400000 ? bits : 0x00400000);
    }
    static __device__ __forceinline__ frag from_mx4(unsigned int d, float s)
    {
        const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 1);
        const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 3);
        return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
    }
    static __device__ __forceinline__ elem round(float v) { return (bf16_t)v; }
};

// fp32, as the type of what is quantised, read back, or written by a product; never an operand of the matrix cores here.
struct F32 {
    typedef float elem;
    static __device__ __forceinline__ elem round(float v) { return v; }
};

// A load by a pointer that was itself loaded, which the compiler would take for one that may point to LDS: such loads are counted with LDS
// accesses, and a wait for those would wait for them too.
template <class V>
__device__ __forceinline__ V load_global(const void* p)
{
    return *(const __attribute__((address_space(1))) V*)p;
}
template <class V>
__device__ __forceinline__ V load_global_once(const void* p)  // (and is not kept in the caches)
{
    return __builtin_nontemporal_load((const __attribute__((address_space(1))) V*)p);
}

// Eight 16-bit values at any address.
template <class T>
__device__ __forceinline__ typename T::frag load8_any(const typename T::elem* p)
{
    return __builtin_bit_cast(typename T::frag, (uint4_t)*reinterpret_cast<const uint4_any_t*>(p));
}

// Values k .. k + 7 of a row of K, zeros behind its end.
template <class T>
__device__ __forceinline__ typename T::frag load8_guarded(const typename T::elem* row, int64_t k, int64_t K)
{
    if (k + 8 <= K) return load8_any<T>(row + k);
    typename T::frag v = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k + i < K) v[i] = row[k + i];
    return v;
}

// Eight results of one row, next to each other from p on.
template <class O>
__device__ __forceinline__ void store8(typename O::elem* p, const float4_t v, const float4_t w)
{
    if constexpr (sizeof(typename O::elem) == 2) {
        const typename O::elem r[8] = {O::round(v[0]), O::round(v[1]), O::round(v[2]), O::round(v[3]), O::round(w[0]), O::round(w[1]), O::round(w[2]), O::round(w[3])};
        *reinterpret_cast<uint4_any_t*>(p) = __builtin_bit_cast(uint4_t, r);
    } else {
        reinterpret_cast<uint4_any_t*>(p)[0] = __builtin_bit_cast(uint4_t, v);
        reinterpret_cast<uint4_any_t*>(p)[1] = __builtin_bit_cast(uint4_t, w);
    }
}

// Four results of one row, next to each other from p on, of which `count` exist.
template <class O>
__device__ __forceinline__ void store4(typename O::elem* p, const float4_t v, int count)
{
    if constexpr (sizeof(typename O::elem) == 2) {
        const typename O::elem r[4] = {O::round(v[0]), O::round(v[1]), O::round(v[2]), O::round(v[3])};
        if (count >= 4) {
            *reinterpret_cast<uint2_any_t*>(p) = __builtin_bit_cast(uint2_t, r);
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) p[i] = r[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) p[i] = v[i];
    }
}
}  // namespace pimhip
