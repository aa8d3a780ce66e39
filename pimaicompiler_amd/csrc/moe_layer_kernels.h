// A mixture-of-experts layer for a few tokens: every token's top_k experts, their two products, and the weighted sum.
//
//   l = Wr x + br                      fp32;  S = the top_k largest, equal ones by their index
//   c_j = softmax(l)_j                 over all experts, or over S alone (renormalize)
//   y = sum_{j in S} c_j (W2_j act(W1_j x + b1_j) + b2_j)      gated: act(g) * u with [g; u] = W1_j x + b1_j
//
// Bound by the weights of the experts that some token chose, each read once: the router, then one launch per product in which a block
// has some rows of one expert and all tokens that chose it (skinny.h), then the sum.  A block finds its tokens in the router's
// table (at most kMoeLayerPairs entries) by itself; one whose expert nobody chose ends at once.
#pragma once

#include "skinny.h"

namespace pimhip
{
static constexpr int kMoeLayerTokens = 64;    // tokens of a launch
static constexpr int kMoeLayerTopK = 16;
static constexpr int kMoeLayerExperts = 256;
static constexpr int kMoeLayerPairs = kMoeLayerTokens * kMoeLayerTopK;

// One expert's weights, as device pointers.  4-bit ones: packed, scales and tops; 16-bit ones: the matrix in w1 / w2.
struct ExpertPointers {
    const void *w1, *s1, *t1, *b1;
    const void *w2, *s2, *t2, *b2;
};

struct MoeLayerArgs {
    const ExpertPointers* experts;  // device, [E]
    const void *x, *router_w, *router_b;
    void* y;
    int* chosen;      // [tokens][top_k]
    float* share;     // [tokens][top_k]
    void* h;          // [pairs][d_ff]: hidden values, rounded to x's type as operands of the matrix cores
    float* part;      // [pairs][d_model]
    int tokens, E, top_k, d_model, d_ff, ld_x;
    int ld_s1, ld_s2;  // pitches of 4-bit weights' scale codes
    int act, renormalize;
};

// ---- router ------------------------------------------------------------------------------------------------------------------
// One token a block: a wavefront an expert at a time, then the choice by the first wavefront.
template <class T>
__global__ __launch_bounds__(256) void moe_layer_router_kernel(MoeLayerArgs a)
{
    __shared__ float logits[kMoeLayerExperts];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, token = blockIdx.x;
    const typename T::elem* x = (const typename T::elem*)a.x + (int64_t)token * a.ld_x;
    for (int e = wave; e < a.E; e += 4) {
        const typename T::elem* w = (const typename T::elem*)a.router_w + (int64_t)e * a.d_model;
        float sum = 0.0f;
        for (int k = lane * 8; k < a.d_model; k += 512) {
            const typename T::frag p = load8_any<T>(w + k), q = load8_any<T>(x + k);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf((float)p[i], (float)q[i], sum);
        }
        sum = wave_sum(sum);
        if (lane == 0) logits[e] = sum + (a.router_b ? (float)((const typename T::elem*)a.router_b)[e] : 0.0f);
    }
    __syncthreads();
    if (wave != 0) return;
    // The choice: the largest of the keys (value, lowest index first) again and again.  A NaN counts as the largest value.
    unsigned long long key[kMoeLayerExperts / 64];
    float largest = -__builtin_inff(), v[kMoeLayerExperts / 64];
#pragma unroll
    for (int i = 0; i < kMoeLayerExperts / 64; ++i) {
        const int e = i * 64 + lane;
        key[i] = 0;
        v[i] = -__builtin_inff();
        if (e < a.E) {
            v[i] = logits[e];
            const unsigned int b = __builtin_bit_cast(unsigned int, v[i] != v[i] ? __builtin_nanf("") : v[i] + 0.0f);
            key[i] = ((unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (unsigned int)(kMoeLayerExperts - e);
        }
    }
    float mine = 0.0f;  // this lane's chosen logit (lane j: choice j)
    int expert = 0;
    for (int j = 0; j < a.top_k; ++j) {
        unsigned long long best = key[0];
#pragma unroll
        for (int i = 1; i < kMoeLayerExperts / 64; ++i) best = key[i] > best ? key[i] : best;
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) {
            const unsigned long long o = __shfl_xor(best, i);
            best = o > best ? o : best;
        }
#pragma unroll
        for (int i = 0; i < kMoeLayerExperts / 64; ++i)
            if (key[i] == best) key[i] = 0;
        const int e = kMoeLayerExperts - (int)(unsigned int)best;
        if (j == 0) largest = logits[e];
        if (lane == j) {
            expert = e;
            mine = logits[e];
        }
    }
    // Shares.  Where every logit is -inf no expert has any.
    float sum = 0.0f;
    if (a.renormalize) {
        sum = lane < a.top_k ? expf(mine - largest) : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < kMoeLayerExperts / 64; ++i) sum += i * 64 + lane < a.E ? expf(v[i] - largest) : 0.0f;
    }
    sum = wave_sum(sum);
    if (lane < a.top_k) {
        const int at = token * a.top_k + lane;
        a.chosen[at] = expert;
        a.share[at] = largest == -__builtin_inff() ? 0.0f : expf(mine - largest) / sum;
    }
}

// ---- the experts' products ---------------------------------------------------------------------------------------------------
// The pairs (token * top_k + choice) that chose expert e, in their order; every thread returns how many.
__device__ __forceinline__ int pairs_of(const int* chosen, int pairs, int e, short* list, int* count)
{
    if (threadIdx.x < 64) {
        int n = 0;
        for (int base = 0; base < pairs; base += 64) {
            const int p = base + (int)threadIdx.x;
            const bool is = p < pairs && chosen[p] == e;
            const unsigned long long all = __ballot(is);
            if (is) list[n + __popcll(all & ((1ull << threadIdx.x) - 1))] = (short)p;
            n += __popcll(all);
        }
        if (threadIdx.x == 0) *count = n;
    }
    __syncthreads();
    return *count;
}

template <class T, bool MX>
struct ExpertWeights;
template <class T>
struct ExpertWeights<T, false> {
    typedef DenseWeights<T> W;
    static __device__ __forceinline__ typename W::Rows rows(const void* w, const void*, const void*, int, int64_t first, int64_t count, int K)
    {
        return W::rows(w, first, count, K);
    }
    static __device__ __forceinline__ float unscale(float v, const void*, int64_t) { return v; }
};
template <class T>
struct ExpertWeights<T, true> {
    typedef Mx4Weights<T> W;
    static __device__ __forceinline__ typename W::Rows rows(const void* w, const void* s, const void* t, int ld, int64_t first, int64_t count, int K)
    {
        return W::rows((const uint8_t*)w, (const uint8_t*)s, (const uint8_t*)t, ld, first, count, K);
    }
    static __device__ __forceinline__ float unscale(float v, const void* t, int64_t r) { return T::unscale(v, ((const uint8_t*)t)[r]); }
};

// The first product of 16 * TT pairs: hidden values 16 * F a block, each with its gate where there is one.
template <class T, bool MX, bool GATED, int F, int TT, int U, int WK>
__device__ __forceinline__ void moe_first(const MoeLayerArgs& a, const ExpertPointers& p, const short* list, int n, float4_t* part)
{
    constexpr int RT = GATED ? 2 * F : F;
    typedef ExpertWeights<T, MX> EW;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4;
    const int f0 = blockIdx.x * (16 * F);
    typedef TurnedTokens<T> X;
    typename EW::W::Rows rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i)  // (value rows follow the gate rows; each kind ends at its own last row)
        rows[i] = EW::rows(p.w1, p.s1, p.t1, a.ld_s1, (i < F ? 0 : a.d_ff) + f0 + i % F * 16, i < F ? a.d_ff : 2 * a.d_ff, a.d_model);
    typename X::Rows tokens[TT];
    int pair[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        pair[j] = j * 16 + (lane & 15) < n ? list[j * 16 + (lane & 15)] : -1;
        tokens[j] = X::rows([&](int i) { return (const typename T::elem*)a.x + (int64_t)(list[j * 16 + i < n ? j * 16 + i : n - 1] / a.top_k) * a.ld_x; });
    }
    float4_t acc[RT][TT] = {};
    constexpr int kLds = kSkinnyLds<typename EW::W, X>;
    skinny_sum<T, typename EW::W, X, RT, TT, U>(acc, rows, tokens, a.d_model, wave, WK, reinterpret_cast<uint4_t*>(part) + wave * kLds, [] {});
    __syncthreads();
    // Gate and value of a hidden unit have to meet: the sums are joined in every wavefront that finishes a tile of them.
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) part[((wave * RT + i) * TT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            if ((i * TT + j) % WK != wave || pair[j] < 0) continue;
            const int f = f0 + i * 16 + group * 4;
            if (f >= a.d_ff) continue;
            float4_t g = {}, u = {};
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                g += part[((k * RT + i) * TT + j) * 64 + lane];
                if (GATED) u += part[((k * RT + F + i) * TT + j) * 64 + lane];
            }
            float4_t h;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float v = EW::unscale(g[c], p.t1, f + c);
                if (p.b1) v += (float)((const typename T::elem*)p.b1)[f + c];
                if (a.act == PIMHIP_EXPERT_RELU) v = relu_f32(v);
                if (a.act == PIMHIP_EXPERT_SILU) v = v / (1.0f + __expf(-v));
                if (GATED) {
                    float w = EW::unscale(u[c], p.t1, a.d_ff + f + c);
                    if (p.b1) w += (float)((const typename T::elem*)p.b1)[a.d_ff + f + c];
                    v *= w;
                }
                h[c] = v;
            }
            store4<T>((typename T::elem*)a.h + (int64_t)pair[j] * a.d_ff + f, h, 4);  // (d_ff is a multiple of 8)
        }
    __syncthreads();
}

// LDS of a product's block: what its wavefronts turn operands in, then their sums.
template <class T, bool MX, int RT, int WK>
constexpr int kExpertLds = WK * (kSkinnyLds<typename ExpertWeights<T, MX>::W, TurnedTokens<T>> > RT * 4 * 64 ? kSkinnyLds<typename ExpertWeights<T, MX>::W, TurnedTokens<T>> : RT * 4 * 64);

template <class T, bool MX, bool GATED, int F, int U, int WK>
__global__ __launch_bounds__(64 * WK) void moe_layer_first_kernel(MoeLayerArgs a)
{
    __shared__ float4_t part[kExpertLds<T, MX, GATED ? 2 * F : F, WK>];
    __shared__ short list[kMoeLayerPairs];
    __shared__ int count;
    const int e = blockIdx.y;
    const int n = pairs_of(a.chosen, a.tokens * a.top_k, e, list, &count);
    if (n == 0) return;
    const ExpertPointers p = a.experts[e];
    if (n <= 16)
        moe_first<T, MX, GATED, F, 1, U, WK>(a, p, list, n, part);
    else if (n <= 32)
        moe_first<T, MX, GATED, F, 2, 1, WK>(a, p, list, n, part);
    else
        moe_first<T, MX, GATED, F, 4, 1, WK>(a, p, list, n, part);
}

// The second product of 16 * TT pairs: rows of d_model, with the bias, not yet weighted.
template <class T, bool MX, int RT, int TT, int U, int WK>
__device__ __forceinline__ void moe_second(const MoeLayerArgs& a, const ExpertPointers& p, const short* list, int n, float4_t* part)
{
    typedef ExpertWeights<T, MX> EW;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4;
    const int d0 = blockIdx.x * (16 * RT);
    typedef TurnedTokens<T> X;
    typename EW::W::Rows rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) rows[i] = EW::rows(p.w2, p.s2, p.t2, a.ld_s2, d0 + i * 16, a.d_model, a.d_ff);
    typename X::Rows hidden[TT];
    int pair[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        pair[j] = j * 16 + (lane & 15) < n ? list[j * 16 + (lane & 15)] : -1;
        hidden[j] = X::rows([&](int i) { return (const typename T::elem*)a.h + (int64_t)list[j * 16 + i < n ? j * 16 + i : n - 1] * a.d_ff; });
    }
    float4_t acc[RT][TT] = {};
    constexpr int kLds = kSkinnyLds<typename EW::W, X>;
    skinny_sum<T, typename EW::W, X, RT, TT, U>(acc, rows, hidden, a.d_ff, wave, WK, reinterpret_cast<uint4_t*>(part) + wave * kLds, [] {});
    skinny_join<RT, TT, WK>(acc, part);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            const int d = d0 + i * 16 + group * 4;
            if ((i * TT + j) % WK != wave || pair[j] < 0 || d >= a.d_model) continue;
            float4_t v = acc[i][j];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[c] = EW::unscale(v[c], p.t2, d + c);
                if (p.b2) v[c] += (float)((const typename T::elem*)p.b2)[d + c];
            }
            *reinterpret_cast<float4_t*>(a.part + (int64_t)pair[j] * a.d_model + d) = v;
        }
}

template <class T, bool MX, int RT, int U, int WK>
__global__ __launch_bounds__(64 * WK) void moe_layer_second_kernel(MoeLayerArgs a)
{
    __shared__ float4_t part[kExpertLds<T, MX, RT, WK>];
    __shared__ short list[kMoeLayerPairs];
    __shared__ int count;
    const int e = blockIdx.y;
    const int n = pairs_of(a.chosen, a.tokens * a.top_k, e, list, &count);
    if (n == 0) return;
    const ExpertPointers p = a.experts[e];
    if (n <= 16)
        moe_second<T, MX, RT, 1, U, WK>(a, p, list, n, part);
    else if (n <= 32)
        moe_second<T, MX, RT, 2, 1, WK>(a, p, list, n, part);
    else
        moe_second<T, MX, RT, 4, 1, WK>(a, p, list, n, part);
}

// The weighted sum in the order of the choice.  An expert without a share adds nothing, whatever it computed.
template <class T>
__global__ __launch_bounds__(256) void moe_layer_sum_kernel(MoeLayerArgs a)
{
    const int d = (blockIdx.x * 256 + threadIdx.x) * 4, token = blockIdx.y;
    if (d >= a.d_model) return;
    float4_t y = {};
    for (int j = 0; j < a.top_k; ++j) {
        const float c = a.share[token * a.top_k + j];
        if (c == 0.0f) continue;
        y += c * *reinterpret_cast<const float4_t*>(a.part + (int64_t)(token * a.top_k + j) * a.d_model + d);
    }
    store4<T>((typename T::elem*)a.y + (int64_t)token * a.d_model + d, y, 4);
}
}  // namespace pimhip
