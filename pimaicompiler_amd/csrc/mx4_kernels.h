// Kernels on microscaled 4-bit values (mx4_format.h): quantisation, reading back, and the products with one or both operands in 4 bits.
#pragma once

#include "skinny.h"

namespace pimhip
{
// A quantised matrix as kernels see it: row r at packed + r * blocks * 16, its scale codes at scales + r * ld_scales (a multiple of
// 16; what lies behind the last block is any), its largest scale code at tops[r].
struct Mx4View {
    const uint8_t* packed;
    const uint8_t* scales;
    const uint8_t* tops;
    int64_t rows, cols, ld_scales;
};

// ---- quantisation ------------------------------------------------------------------------------------------------------------
// Eight values of one lane from k on, as bits of fp32 magnitudes' maximum and in the conversion's own type.
template <class T>
struct QuantLane {
    float v[8];
    __device__ __forceinline__ void load(const typename T::elem* row, int64_t k, int64_t K)
    {
        if (k + 8 <= K) {
            typename T::elem e[8];
            if constexpr (sizeof(typename T::elem) == 2) {
                const uint4_t q = *reinterpret_cast<const uint4_any_t*>(row + k);
                __builtin_memcpy(e, &q, 16);
            } else {
                const uint4_any_t* p = reinterpret_cast<const uint4_any_t*>(row + k);
                const uint4_t q0 = p[0], q1 = p[1];
                __builtin_memcpy(e, &q0, 16);
                __builtin_memcpy(e + 4, &q1, 16);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)e[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < K ? (float)row[k + i] : 0.0f;
        }
    }
};

// One row by WPR wavefronts, 256 / 64 / WPR rows a block.  Four lanes share a scale block, eight values each; the block's largest
// magnitude goes round them by DPP.  Its exponent less two (the exponent of 6, the largest element) is the scale; elements are
// rounded to the nearest, ties to even, and saturate at 6 (v_cvt_scalef32_pk_fp4_f32).  A block that holds an infinity or a NaN
// has the scale "not a number".  Bound by reading x: 16384 x 4096 in bf16 31 us, 5.5 TB/s with what is written.
template <class T, int WPR>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const typename T::elem* x, int64_t rows, int64_t cols, int64_t ld, uint8_t* packed, uint8_t* scales,
                                                           int64_t ld_scales, uint8_t* tops)
{
    constexpr int kRows = 4 / WPR;
    __shared__ unsigned int top_of[4];
    const int wave = wave_in_block();
    const int64_t row = (int64_t)blockIdx.x * kRows + wave / WPR;
    const int lane = threadIdx.x % (64 * WPR);
    const int64_t blocks = (cols + kMxBlock - 1) / kMxBlock;
    unsigned int top = 0;
    if (row < rows) {
        const typename T::elem* src = x + row * ld;
        for (int64_t k = lane * 8; k < blocks * kMxBlock; k += 64 * WPR * 8) {
            const int64_t block = k / kMxBlock;
            QuantLane<T> q;
            q.load(src, k, cols);
            unsigned int m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned int b = __builtin_bit_cast(unsigned int, q.v[i]) & 0x7fffffffu;
                m = m > b ? m : b;
            }
            unsigned int o = dpp_u32<kDppQuadXor1>(m);
            m = m > o ? m : o;
            o = dpp_u32<kDppQuadXor2>(m);
            m = m > o ? m : o;
            const unsigned int field = m >> 23;
            const unsigned int code = field == 255u ? kMxNan : field > 2u ? field - 2u : 0u;
            const float s = mx_scale_f32(code == kMxNan ? 0u : code);
            unsigned int d = 0;
            d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, q.v[0], q.v[1], s, 0);
            d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, q.v[2], q.v[3], s, 1);
            d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, q.v[4], q.v[5], s, 2);
            d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, q.v[6], q.v[7], s, 3);
            if (code == kMxNan) d = 0;
            reinterpret_cast<unsigned int*>(packed + row * blocks * kMxBlockBytes)[k / 8] = d;
            if (code != kMxNan && code > top) top = code;
            if ((lane & 3) == 0) scales[row * ld_scales + block] = (uint8_t)code;
        }
    }
    // The row's largest scale code.
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const unsigned int o = __shfl_xor(top, i);
        top = top > o ? top : o;
    }
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) top_of[wave] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
            const unsigned int o = top_of[wave / WPR * WPR + i];
            top = top > o ? top : o;
        }
    }
    if (row < rows && lane == 0) tops[row] = (uint8_t)top;
}

// The largest scale code of each row, codes 255 apart: what a matrix that was not quantised here lacks.  A wavefront a row.
__global__ __launch_bounds__(256) void mx4_tops_kernel(const uint8_t* scales, int64_t ld_scales, int64_t rows, int64_t blocks, uint8_t* tops)
{
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    unsigned int top = 0;
    for (int64_t b = threadIdx.x & 63; b < blocks; b += 64) {
        const unsigned int c = scales[row * ld_scales + b];
        if (c != kMxNan && c > top) top = c;
    }
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const unsigned int o = __shfl_xor(top, i);
        top = top > o ? top : o;
    }
    if ((threadIdx.x & 63) == 0) tops[row] = (uint8_t)top;
}

// The values of eight codes, rounded once to O.
template <class O>
__device__ __forceinline__ void mx4_values(unsigned int d, float s, typename O::elem (&e)[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2_t v = i == 0 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, s, 0) : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, s, 1)
                           : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, s, 2) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, s, 3);
        e[2 * i] = O::round(v[0]);
        e[2 * i + 1] = O::round(v[1]);
    }
}

// Reading back: eight values a lane, a row a block of the grid's y and 2048 values a block of its x.  Bound by writing: 16384 x 4096 in
// bf16 25 us, 6.7 TB/s.
template <class O>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t* packed, const uint8_t* scales, int64_t rows, int64_t cols, int64_t ld_scales,
                                                             typename O::elem* out, int64_t ld)
{
    const int64_t blocks = (cols + kMxBlock - 1) / kMxBlock;
    const int64_t k = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (k >= cols) return;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const unsigned int d = reinterpret_cast<const unsigned int*>(packed + row * blocks * kMxBlockBytes)[k / 8];
        typename O::elem e[8];
        mx4_values<O>(d, mx_scale_f32(scales[row * ld_scales + k / kMxBlock]), e);
        typename O::elem* to = out + row * ld + k;
        if (k + 8 <= cols) {
            uint4_t q[sizeof(e) / 16];
            __builtin_memcpy(q, e, sizeof(e));
#pragma unroll
            for (unsigned i = 0; i < sizeof(e) / 16; ++i) reinterpret_cast<uint4_any_t*>(to)[i] = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < cols) to[i] = e[i];
        }
    }
}

// ---- x in 16 bits, weights in 4: a few tokens --------------------------------------------------------------------------------
// y[m, n] = act(sum_k x[m, k] w[n, k] + b[n]).  WK wavefronts share k of 16 * RT rows and up to 16 * TT tokens (skinny.h).  SHARED: the
// tokens (at most 16) lie in LDS as a whole, in the launch's dynamic part of it.  Bound by the weights' bytes: 16384 x 4096 for one token
// 8.1 us, 4.4 TB/s; 31999 x 1024 for 16 tokens 7.0 us, 2.5 TB/s, a block's chain of loads being half of that.  What was measured to choose
// the tile and the wavefronts stands with the rule that chooses.
template <class T, bool SHARED, int RT, int TT, int WK>
__global__ __launch_bounds__(64 * WK) void mx4_linear_skinny_kernel(const typename T::elem* x, Mx4View w, const typename T::elem* bias, typename T::elem* out,
                                                                    int64_t ld_x, int64_t ld_out, int64_t M, int relu)
{
    typedef Mx4Weights<T, TT == 1 ? 2 : 1> W;
    typedef typename std::conditional<SHARED, SharedTokens<T>, TurnedTokens<T, false>>::type X;
    constexpr int kLds = kSkinnyLds<W, X>, kPart = RT * TT * 64;
    __shared__ uint4_t lds[WK * (kLds > kPart ? kLds : kPart)];
    __shared__ int tops[RT * 16];
    __shared__ float add[RT * 16];
    extern __shared__ uint4_t xs[];
    const int lane = threadIdx.x & 63, wave = wave_in_block(), group = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * (16 * RT), token0 = (int64_t)blockIdx.y * (16 * TT);
    typename W::Rows rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t at = row0 + i * 16;
        rows[i] = W::rows(w.packed, w.scales, w.tops, w.ld_scales, at < w.rows ? at : w.rows - 1, w.rows, w.cols);
    }
    auto token = [&](int64_t t) { return x + (t < M ? t : M - 1) * ld_x; };
    const int K = (int)w.cols, pitch = SharedTokens<T>::pitch(K, W::kUnit);
    typename X::Rows tokens[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        if constexpr (SHARED)
            tokens[j] = X::rows(xs, (lane & 15) < M ? lane & 15 : (int)M - 1, pitch);
        else
            tokens[j] = X::rows([&](int i) { return token(token0 + j * 16 + i); });
    }
    // What the results of a row need goes to LDS for the wavefronts that finish them.
    if (threadIdx.x < 16 * RT) {
        int64_t n = row0 + threadIdx.x;
        n = n < w.rows ? n : w.rows - 1;
        tops[threadIdx.x] = w.tops[n];
        add[threadIdx.x] = bias ? (float)bias[n] : 0.0f;
    }
    float4_t acc[RT][TT] = {};
    skinny_sum<T, W, X, RT, TT>(acc, rows, tokens, K, wave, WK, lds + wave * kLds, [&] {
        if constexpr (SHARED) SharedTokens<T>::stage(xs, token, (int)M, K, pitch);
        __syncthreads();
    });
    skinny_join<RT, TT, WK>(acc, reinterpret_cast<float4_t*>(lds));
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            if ((i * TT + j) % WK != wave) continue;
            const int64_t t = token0 + j * 16 + (lane & 15), n = row0 + i * 16 + group * 4;
            if (t >= M || n >= w.rows) continue;
            float4_t v = acc[i][j];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[c] = __builtin_amdgcn_ldexpf(v[c], T::exponent(tops[i * 16 + group * 4 + c]));
                if (bias) v[c] += add[i * 16 + group * 4 + c];  // (a zero that is no bias would turn -0 into 0)
                if (relu) v[c] = relu_f32(v[c]);
            }
            store4<T>(out + t * ld_out + n, v, w.rows - n < 4 ? (int)(w.rows - n) : 4);
        }
}

// ---- both operands in 4 bits: a few rows of a --------------------------------------------------------------------------------
// y[m, n] = sum_k a[m, k] b[n, k] on v_mfma_scale_f32_16x16x128_f8f6f4, which multiplies the scales in: 16 rows of b and 16 of a
// a product, one block and its scale code a lane.  Bound by latency or by b's bytes: 1024 x 1024 for one row 2.9 us, 16384 x 4096 for 16 rows
// 12.4 us, 2.9 TB/s (operands are read as the instruction wants them, 16 bytes of 16 rows
// a request each; loading runs of a row and turning them, as skinny.h does, has not been tried here).
template <class O, int RT, int TT, int WK>
__global__ __launch_bounds__(64 * WK) void mx4_matmul_skinny_kernel(Mx4View a, Mx4View b, typename O::elem* out, int64_t ld_out)
{
    __shared__ float4_t part[WK * RT * TT * 64];
    const int lane = threadIdx.x & 63, wave = wave_in_block(), group = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * (16 * RT), token0 = (int64_t)blockIdx.y * (16 * TT);
    const int blocks = (int)((b.cols + kMxBlock - 1) / kMxBlock);
    const uint8_t *bp[RT], *bs[RT], *ap[TT], *as[TT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        int64_t r = row0 + i * 16 + (lane & 15);
        r = r < b.rows ? r : b.rows - 1;
        bp[i] = b.packed + r * blocks * kMxBlockBytes;
        bs[i] = b.scales + r * b.ld_scales;
    }
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        int64_t t = token0 + j * 16 + (lane & 15);
        t = t < a.rows ? t : a.rows - 1;
        ap[j] = a.packed + t * blocks * kMxBlockBytes;
        as[j] = a.scales + t * a.ld_scales;
    }
    float4_t acc[RT][TT] = {};
    const int steps = (blocks + 3) / 4;
    for (int s = wave; s < steps; s += WK) {
        const int block = s * 4 + group;
        const bool in = block < blocks;
        int8v_t bv[RT] = {}, av[TT] = {};
        int bc[RT], ac[TT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            uint4_t q = {0, 0, 0, 0};
            bc[i] = 127;
            if (in) {
                q = *reinterpret_cast<const uint4_t*>(bp[i] + block * kMxBlockBytes);
                bc[i] = bs[i][block];
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) bv[i][c] = (int)q[c];
        }
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            uint4_t q = {0, 0, 0, 0};
            ac[j] = 127;
            if (in) {
                q = *reinterpret_cast<const uint4_t*>(ap[j] + block * kMxBlockBytes);
                ac[j] = as[j][block];
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) av[j][c] = (int)q[c];
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < TT; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bv[i], av[j], acc[i][j], 4, 4, 0, bc[i], 0, ac[j]);
    }
    skinny_join<RT, TT, WK>(acc, part);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            if ((i * TT + j) % WK != wave) continue;
            const int64_t t = token0 + j * 16 + (lane & 15), n = row0 + i * 16 + group * 4;
            if (t >= a.rows || n >= b.rows) continue;
            store4<O>(out + t * ld_out + n, acc[i][j], b.rows - n < 4 ? (int)(b.rows - n) : 4);
        }
}
}  // namespace pimhip
