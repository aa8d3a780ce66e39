// Sums of a few tokens against many rows of weights on the matrix cores: what the products with 4-bit weights and the experts of a
// mixture share.
//
//   acc[row, token] = sum_k w[row, k] * x[token, k]          v_mfma_f32_16x16x32: 16 rows x 16 tokens x 32 k
//
// The weights are read once and are what bounds such a product, so they go from memory into registers as the matrix cores
// want them, without a stop in LDS: lane l has row l % 16 and, of each step of 128 values, the 32 from 32 * (l / 16) on (one 16-byte
// load of 4-bit weights, which is one block with one scale; four of 16-bit weights).  The order of k inside a step is the same for both
// operands and otherwise free: product o of a step takes values 8 o .. 8 o + 7 of each lane's 32.  x is small and comes out of the
// caches.  Loads of weights run one unit of U steps ahead of the products; the unit's x is asked for before the next unit's
// weights, since a wavefront's loads come back in order.
#pragma once

#include "mx4_format.h"

namespace pimhip
{
static constexpr int kSkinnyStep = 128;  // values of k a wavefront takes at a time

// 16-bit weights.
template <class T>
struct DenseWeights {
    struct Row {
        const typename T::elem* p;  // the row, at this lane's 32 values of the first step
    };
    struct Raw {
        typename T::frag v[4];
    };
    static __device__ __forceinline__ Raw load(const Row& r, int step)
    {
        Raw w;
        const half8_any_t* q = reinterpret_cast<const half8_any_t*>(r.p + (int64_t)step * kSkinnyStep);
#pragma unroll
        for (int o = 0; o < 4; ++o) w.v[o] = __builtin_bit_cast(typename T::frag, (half8_t)__builtin_nontemporal_load(q + o));
        return w;
    }
    // The same where the row may end inside the step; rows are whole groups of eight values.
    static __device__ __forceinline__ Raw load_guarded(const Row& r, int step, int group, int K)
    {
        Raw w;
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            w.v[o] = typename T::frag{};
            if (step * kSkinnyStep + group * 32 + o * 8 < K) w.v[o] = load8_any<T>(r.p + (int64_t)step * kSkinnyStep + o * 8);
        }
        return w;
    }
    static __device__ __forceinline__ float scale(const Raw&, const Row&, int) { return 1.0f; }
    static __device__ __forceinline__ typename T::frag operand(const Raw& w, float, int o) { return w.v[o]; }
};

// 4-bit weights; T is the type of x.
template <class T>
struct Mx4Weights {
    struct Row {
        const uint8_t* packed;  // the row, at this lane's block of the first step
        const uint8_t* scales;  // the row's scale codes, 4-byte aligned
        int top;                // its largest scale code
    };
    struct Raw {
        uint4_t v;
        unsigned int codes;  // the scale codes of the step's four blocks
    };
    static __device__ __forceinline__ Raw load(const Row& r, int step)
    {
        return Raw{__builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(r.packed + (int64_t)step * (kSkinnyStep / 2))),
                   *reinterpret_cast<const unsigned int*>(r.scales + step * 4)};
    }
    // (the scale codes of a row fill whole groups of 16 bytes; those of no block are any)
    static __device__ __forceinline__ Raw load_guarded(const Row& r, int step, int group, int K)
    {
        if (step * kSkinnyStep + group * kMxBlock < K) return load(r, step);
        return Raw{uint4_t{0, 0, 0, 0}, 0x7f7f7f7fu};
    }
    static __device__ __forceinline__ float scale(const Raw& w, const Row& r, int group) { return T::scale((w.codes >> (8 * group)) & 255u, r.top); }
    static __device__ __forceinline__ typename T::frag operand(const Raw& w, float s, int o) { return T::from_mx4(w.v[o], s); }
};

// acc[i][j] += rows i of this lane x tokens j, over units of U steps first, first + stride, ... of K; x[j] is the token's row at this
// lane's 32 values of the first step.
template <class T, class W, int RT, int TT, int U>
__device__ __forceinline__ void skinny_sum(float4_t (&acc)[RT][TT], const typename W::Row (&w)[RT], const typename T::elem* const (&x)[TT], int K, int first,
                                           int stride)
{
    const int group = (threadIdx.x & 63) >> 4;
    const int units = K / (U * kSkinnyStep);
    typedef typename T::frag frag;
    typename W::Raw cur[U][RT], next[U][RT];
    frag xv[U][TT][4];
    auto load_w = [&](typename W::Raw(&to)[U][RT], int n) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RT; ++i) to[u][i] = W::load(w[i], n * U + u);
    };
    auto load_x = [&](int n) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < TT; ++j)
#pragma unroll
                for (int o = 0; o < 4; ++o) xv[u][j][o] = load8_any<T>(x[j] + (int64_t)(n * U + u) * kSkinnyStep + o * 8);
    };
    auto products = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const float s = W::scale(cur[u][i], w[i], group);
#pragma unroll
                for (int o = 0; o < 4; ++o) {
                    const frag a = W::operand(cur[u][i], s, o);
#pragma unroll
                    for (int j = 0; j < TT; ++j) acc[i][j] = T::mfma(a, xv[u][j][o], acc[i][j]);
                }
            }
    };
    if (first < units) {
        int n = first;
        load_w(cur, n);
        for (; n + stride < units; n += stride) {
            load_x(n);
            load_w(next, n + stride);
            products();
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < RT; ++i) cur[u][i] = next[u][i];
        }
        load_x(n);
        products();
    }
    // What is left of K, step by step, the last one guarded.
    const int steps = (K + kSkinnyStep - 1) / kSkinnyStep;
    for (int s = units * U + first; s < steps; s += stride) {
        typename W::Raw raw[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) raw[i] = W::load_guarded(w[i], s, group, K);
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            frag xt[TT];
#pragma unroll
            for (int j = 0; j < TT; ++j) xt[j] = load8_guarded<T>(x[j] - group * 32, (int64_t)s * kSkinnyStep + group * 32 + o * 8, K);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const frag a = W::operand(raw[i], W::scale(raw[i], w[i], group), o);
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[i][j] = T::mfma(a, xt[j], acc[i][j]);
            }
        }
    }
}

// Sums of the WK wavefronts of a block, which shared k: tile (i, j) ends up in wavefront (i * TT + j) % WK; returns whether this
// one has it.  `part` is WK * RT * TT * 64 vectors of LDS.  The order of the sum is the wavefronts'.
template <int RT, int TT, int WK>
__device__ __forceinline__ void skinny_join(float4_t (&acc)[RT][TT], float4_t* part)
{
    if constexpr (WK > 1) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < TT; ++j) part[((wave * RT + i) * TT + j) * 64 + lane] = acc[i][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                if ((i * TT + j) % WK != wave) continue;
                float4_t v = part[(i * TT + j) * 64 + lane];
#pragma unroll
                for (int k = 1; k < WK; ++k) v += part[((k * RT + i) * TT + j) * 64 + lane];
                acc[i][j] = v;
            }
    }
}
}  // namespace pimhip
