// A mixture-of-experts layer for a few tokens: every token's top_k experts, their two products, and the weighted sum.
//
//   l = Wr x + br                      fp32;  S = the top_k largest, equal ones by their index
//   c_j = softmax(l)_j                 over all experts, or over S alone (renormalize)
//   y = sum_{j in S} c_j (W2_j act(W1_j x + b1_j) + b2_j)      gated: act(g) * u with [g; u] = W1_j x + b1_j
//
// Bound by the weights of the experts that some token chose, each read once: the router, then one launch per product in which a block
// has some rows of one expert and all tokens that chose it (skinny.h).  A block finds its tokens in the router's table (at most
// kMoeLayerPairs entries) by itself; one whose expert nobody chose has nothing to read.
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
    void* h;          // [pairs][2][ld_h]: hidden values rounded to x's type, and what that left over, rounded too
    float* part;      // [pairs][d_model]
    unsigned int* counters;  // pairs whose second product is done, for each tile of rows
    int counters_used;
    int tokens, E, top_k, d_model, d_ff, ld_x;
    int ld_h;         // d_ff filled up to whole groups of eight, with zeros
    int ld_s1, ld_s2;  // pitches of 4-bit weights' scale codes
    int act, renormalize;
};

// ---- router ------------------------------------------------------------------------------------------------------------------
// One token a block.  A wavefront has four experts at a time and 1024 values of each, whose loads do not wait for one another; the first
// one chooses.  Bound by latency: 3.4 us for one token and 8 experts of 1024 values, 6.9 for 13 tokens and 64 of 2048.
static constexpr int kRouterThreads = 1024;

template <class T>
__global__ __launch_bounds__(kRouterThreads) void moe_layer_router_kernel(MoeLayerArgs a)
{
    __shared__ float logits[kMoeLayerExperts];
    const int lane = threadIdx.x & 63, wave = wave_in_block(), token = blockIdx.x;
    for (int i = token * kRouterThreads + threadIdx.x; i < a.counters_used; i += gridDim.x * kRouterThreads) a.counters[i] = 0u;
    const typename T::elem* x = (const typename T::elem*)a.x + (int64_t)token * a.ld_x;
    for (int e0 = wave * 4; e0 < a.E; e0 += kRouterThreads / 64 * 4) {
        const typename T::elem* w[4];
        float sum[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (const typename T::elem*)a.router_w + (int64_t)(e0 + i < a.E ? e0 + i : a.E - 1) * a.d_model;
        for (int k0 = lane * 8; k0 < a.d_model; k0 += 1024) {
            typename T::frag q[2], p[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = k0 + h * 512 < a.d_model ? k0 + h * 512 : k0;  // (what is loaded twice counts once)
                q[h] = k0 + h * 512 < a.d_model ? load8_any<T>(x + k) : typename T::frag{};
#pragma unroll
                for (int i = 0; i < 4; ++i) p[h][i] = load8_any<T>(w[i] + k);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (k0 + h * 512 >= a.d_model) continue;  // (a zero times an infinity is none)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < 8; ++c) sum[i] = fmaf((float)p[h][i][c], (float)q[h][c], sum[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum[i] = wave_sum(sum[i]);
            if (lane == 0 && e0 + i < a.E) logits[e0 + i] = sum[i] + (a.router_b ? (float)((const typename T::elem*)a.router_b)[e0 + i] : 0.0f);
        }
    }
    __syncthreads();
    if (wave != 0) return;
    // The choice: the largest value that is left, in its lowest place, again and again.  Lane l has experts l, l + 64, ...; places of no
    // expert and of chosen ones are 0, below every value.  A NaN counts as the largest value, -0 as 0.
    constexpr int kEach = kMoeLayerExperts / 64;
    const int each = (a.E + 63) / 64;
    unsigned int key[kEach];
    float v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        key[i] = 0;
        v[i] = -__builtin_inff();
        if (i < each && i * 64 + lane < a.E) {
            v[i] = logits[i * 64 + lane];
            const unsigned int b = __builtin_bit_cast(unsigned int, v[i] != v[i] ? __builtin_nanf("") : v[i] + 0.0f);
            key[i] = b & 0x80000000u ? ~b : b | 0x80000000u;
        }
    }
    int expert = 0, first = 0;  // this lane's choice (lane j: choice j), and the first one
    for (int j = 0; j < a.top_k; ++j) {
        unsigned int best = key[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i)
            if (i < each) best = key[i] > best ? key[i] : best;
        best = wave_max_u32(best);
        int e = -1;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i >= each || e >= 0) continue;
            const unsigned long long at = __ballot(key[i] == best);
            if (at == 0ull) continue;
            e = i * 64 + __builtin_ctzll(at);
            if (lane == (e & 63)) key[i] = 0;
        }
        if (j == 0) first = e;
        if (lane == j) expert = e;
    }
    // Shares.  Where every logit is -inf no expert has any.
    const float largest = logits[first], mine = logits[expert];
    float sum = 0.0f;
    if (a.renormalize) {
        sum = lane < a.top_k ? expf(mine - largest) : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i < each) sum += i * 64 + lane < a.E ? expf(v[i] - largest) : 0.0f;
    }
    sum = wave_sum(sum);
    if (lane < a.top_k) {
        const int at = token * a.top_k + lane;
        a.chosen[at] = expert;
        a.share[at] = largest == -__builtin_inff() ? 0.0f : expf(mine - largest) / sum;
    }
}

// ---- the experts' products ---------------------------------------------------------------------------------------------------
// The pairs (token * top_k + choice) that chose expert e, in their order; every thread returns how many.  The first wavefront looks, four
// loads at a time.
__device__ __forceinline__ int pairs_of(const int* chosen, int pairs, int e, short* list, int* count)
{
    if (threadIdx.x < 64) {
        int n = 0;
        for (int base = 0; base < pairs; base += 256) {
            int c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = base + i * 64 + (int)threadIdx.x;
                c[i] = chosen[p < pairs ? p : pairs - 1];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = base + i * 64 + (int)threadIdx.x;
                const bool is = p < pairs && c[i] == e;
                const unsigned long long all = __ballot(is);
                if (is) list[n + __popcll(all & ((1ull << threadIdx.x) - 1))] = (short)p;
                n += __popcll(all);
            }
        }
        if (threadIdx.x == 0) *count = n;
    }
    __syncthreads();
    return *count;
}

// (of 4-bit weights one step a unit leaves the registers that two columns a pair take)
template <class T, bool MX, int TT>
struct ExpertWeights;
template <class T, int TT>
struct ExpertWeights<T, false, TT> {
    typedef DenseWeights<T> W;
    static __device__ __forceinline__ typename W::Rows rows(const void* w, const void*, const void*, int, int64_t first, int64_t count, int K)
    {
        return W::rows(w, first, count, K);
    }
    static __device__ __forceinline__ float unscale(float v, const void*, int64_t) { return v; }
};
template <class T, int TT>
struct ExpertWeights<T, true, TT> {
    typedef Mx4Weights<T, TT == 1 ? 2 : 1> W;
    static __device__ __forceinline__ typename W::Rows rows(const void* w, const void* s, const void* t, int ld, int64_t first, int64_t count, int K)
    {
        return W::rows((const uint8_t*)w, (const uint8_t*)s, (const uint8_t*)t, ld, first, count, K);
    }
    static __device__ __forceinline__ float unscale(float v, const void* t, int64_t r) { return T::unscale(v, ((const uint8_t*)t)[r]); }
};

// What a block of the experts' products has in LDS: the tokens that chose its expert, what its wavefronts turn operands in (and then
// their sums), and, SHARED, in the launch's dynamic part the values of its columns.
template <class T, bool MX, bool SHARED, int RT, int WK, int TT, int PARTS>
struct ExpertLds {
    typedef typename ExpertWeights<T, MX, TT>::W W;
    typedef typename std::conditional<SHARED, SharedTokens<T>, TurnedTokens<T, true>>::type X;
    static constexpr int kTurn = kSkinnyLds<W, X>, kSum = RT * PARTS * 64;
    uint4_t turn[WK * (kTurn > kSum ? kTurn : kSum)];
    short list[kMoeLayerPairs];
    int count;
};

// Sums of 16 * RT rows for n columns, whose values are `columns(i)`.  TT 2, PARTS 1: of n (at most 16) sums of two, n apart.  Else n is at most 16 TT.
// Ends with every wavefront having the sums of its own k in `lds`, part[wave][i][j][lane].  SHARED: the values are staged in `xs`.
template <class T, bool MX, bool SHARED, int RT, int WK, int TT, int PARTS, class F>
__device__ __forceinline__ void expert_sums(const typename ExpertWeights<T, MX, TT>::W::Rows (&rows)[RT], int K, int n, uint4_t* xs, uint4_t* lds, F columns)
{
    typedef typename ExpertWeights<T, MX, TT>::W W;
    typedef typename std::conditional<SHARED, SharedTokens<T>, TurnedTokens<T, true>>::type X;
    const int lane = threadIdx.x & 63, wave = wave_in_block();
    const int pitch = SharedTokens<T>::pitch(K, W::kUnit);
    float4_t acc[RT][TT] = {};
    typename X::Rows x[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        // (columns behind the last one: that one again)
        auto at = [&](int i) { return PARTS == TT ? (j * 16 + i < n ? j * 16 + i : n - 1) : j * n + (i < n ? i : n - 1); };
        if constexpr (SHARED)
            x[j] = X::rows(xs, at(lane & 15), pitch);
        else
            x[j] = X::rows([&](int i) { return columns(at(i)); });
    }
    skinny_sum<T, W, X, RT, TT, 1>(acc, rows, x, K, wave, WK, lds + wave * kSkinnyLds<W, X>, [&] {
        if constexpr (SHARED) {
            X::stage(xs, columns, PARTS == TT ? n : TT * n, K, pitch);
            __syncthreads();
        }
    });
    __syncthreads();
    float4_t* part = reinterpret_cast<float4_t*>(lds);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < PARTS; ++j) part[((wave * RT + i) * PARTS + j) * 64 + lane] = PARTS == TT ? acc[i][j] : acc[i][0] + acc[i][TT - 1];
    __syncthreads();
}

// Tile i of the wavefronts' sums, in their order.
template <int RT, int WK>
__device__ __forceinline__ float4_t joined(const uint4_t* lds, int i)
{
    const float4_t* part = reinterpret_cast<const float4_t*>(lds) + i * 64 + (threadIdx.x & 63);
    float4_t v = part[0];
#pragma unroll
    for (int k = 1; k < WK; ++k) v += part[k * RT * 64];
    return v;
}

// The first product of up to 16 TT pairs: hidden values 16 * F a block, each with its gate where there is one.
template <class T, bool MX, bool SHARED, bool GATED, int F, int WK, int TT>
__device__ __forceinline__ void moe_first(const MoeLayerArgs& a, const ExpertPointers& p, const short* list, int n, uint4_t* xs, uint4_t* lds)
{
    constexpr int RT = GATED ? 2 * F : F;
    typedef ExpertWeights<T, MX, TT> EW;
    const int lane = threadIdx.x & 63, wave = wave_in_block(), group = lane >> 4;
    const int f0 = blockIdx.x * (16 * F);
    typename EW::W::Rows rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {  // (value rows follow the gate rows; each kind ends at its own last row)
        const int end = i < F ? a.d_ff : 2 * a.d_ff, at = (i < F ? 0 : a.d_ff) + f0 + i % F * 16;
        rows[i] = EW::rows(p.w1, p.s1, p.t1, a.ld_s1, at < end ? at : end - 1, end, a.d_model);
    }
    expert_sums<T, MX, SHARED, RT, WK, TT, TT>(rows, a.d_model, n, xs, lds,
                                   [&](int i) { return (const typename T::elem*)a.x + (int64_t)(list[i] / a.top_k) * a.ld_x; });
#pragma unroll
    for (int k = 0; k < F * TT; ++k) {
        const int i = k / TT, j = k % TT, f = f0 + i * 16 + group * 4, column = j * 16 + (lane & 15);
        if (k % WK != wave || column >= n || f >= a.ld_h) continue;
        const float4_t g = joined<RT * TT, WK>(lds, k);
        float4_t u = {}, h, left;
        if constexpr (GATED) u = joined<RT * TT, WK>(lds, (F + i) * TT + j);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            h[c] = left[c] = 0.0f;
            if (f + c >= a.d_ff) continue;
            float v = EW::unscale(g[c], p.t1, f + c);
            if (p.b1) v += (float)((const typename T::elem*)p.b1)[f + c];
            if (a.act == PIMHIP_EXPERT_RELU) v = relu_f32(v);
            if (a.act == PIMHIP_EXPERT_SILU) v = v / (1.0f + __expf(-v));
            if (GATED) {
                float w = EW::unscale(u[c], p.t1, a.d_ff + f + c);
                if (p.b1) w += (float)((const typename T::elem*)p.b1)[a.d_ff + f + c];
                v *= w;
            }
            // A hidden value is two operands of the next product: rounded to 16 bits alone it would be what limits y.
            h[c] = (float)T::round(v);
            left[c] = fabsf(h[c]) < __builtin_inff() ? v - h[c] : 0.0f;
        }
        typename T::elem* to = (typename T::elem*)a.h + (int64_t)list[column] * 2 * a.ld_h + f;
        store4<T>(to, h, 4);
        store4<T>(to + a.ld_h, left, 4);
    }
    __syncthreads();
}

// Block (x, y, z): rows x of expert y for 16 TT of its pairs, from 16 TT z on; those of more pairs read the weights again, out of the
// caches.  (A loop over pairs in one block instead costs so many registers that half the wavefronts fit: 39 us against 25 for 64 tokens
// through 8 gated 4-bit experts 1024 -> 4096, before blocks had twice the rows.)  That case takes 18 us now with TT 2, 35.7 MB; a block's chain of
// loads (its pairs, then weights and values, k being a unit or two a wavefront) is what it waits for.  13 tokens through 64 gated bf16 experts 2048 -> 1024, six
// chosen: 61 us, 6.3 TB/s.
template <class T, bool MX, bool SHARED, bool GATED, int F, int WK, int TT>
__global__ __launch_bounds__(64 * WK, TT > 1 ? 2 : F > 2 || (GATED && F > 1) ? 3 : 4) void moe_layer_first_kernel(MoeLayerArgs a)
{
    __shared__ ExpertLds<T, MX, SHARED, GATED ? 2 * F : F, WK, TT, TT> lds;
    extern __shared__ uint4_t xs[];
    const ExpertPointers p = a.experts[blockIdx.y];
    const int first = blockIdx.z * (16 * TT), n = pairs_of(a.chosen, a.tokens * a.top_k, blockIdx.y, lds.list, &lds.count) - first;
    if (n > 0) moe_first<T, MX, SHARED, GATED, F, WK, TT>(a, p, lds.list + first, n < 16 * TT ? n : 16 * TT, xs, lds.turn);
}

// The second product: rows of d_model, with the bias, not yet weighted.  TT 1: of up to 8 pairs, two columns each; TT 2: of up to 16.
template <class T, bool MX, bool SHARED, int RT, int WK, int TT>
__device__ __forceinline__ void moe_second(const MoeLayerArgs& a, const ExpertPointers& p, const short* list, int n, uint4_t* xs, uint4_t* lds)
{
    typedef ExpertWeights<T, MX, TT> EW;
    const int lane = threadIdx.x & 63, wave = wave_in_block(), group = lane >> 4;
    const int d0 = blockIdx.x * (16 * RT);
    typename EW::W::Rows rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) rows[i] = EW::rows(p.w2, p.s2, p.t2, a.ld_s2, d0 + i * 16 < a.d_model ? d0 + i * 16 : a.d_model - 1, a.d_model, a.d_ff);
    const typename T::elem* h = (const typename T::elem*)a.h;
    if constexpr (TT == 1)
        expert_sums<T, MX, SHARED, RT, WK, 1, 1>(rows, a.d_ff, 2 * n, xs, lds, [&](int i) { return h + ((int64_t)list[i / 2] * 2 + i % 2) * a.ld_h; });
    else
        expert_sums<T, MX, SHARED, RT, WK, 2, 1>(rows, a.d_ff, n, xs, lds, [&](int i) { return h + ((int64_t)list[i < n ? i : i - n] * 2 + (i < n ? 0 : 1)) * a.ld_h; });
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int d = d0 + i * 16 + group * 4, pair = TT == 1 ? (lane & 15) / 2 : lane & 15;
        if (i % WK != wave || pair >= n || d >= a.d_model) continue;  // (two lanes at a time)
        float4_t v = joined<RT, WK>(lds, i);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (TT == 1) v[c] += dpp_f32<kDppQuadXor1>(v[c]);  // (the pair's other column)
            v[c] = EW::unscale(v[c], p.t2, d + c);
            if (p.b2) v[c] += (float)((const typename T::elem*)p.b2)[d + c];
        }
        const uint4_t q = __builtin_bit_cast(uint4_t, v);
        if (TT == 2 || lane % 2 == 0) store16_device_scope(a.part + (int64_t)list[pair] * a.d_model + d, q[0] | (unsigned long long)q[1] << 32, q[2] | (unsigned long long)q[3] << 32);
    }
    __syncthreads();
}

// Blocks as above, with 8 TT pairs.  The one whose pairs are the last of a tile of rows makes the weighted sum there, in the order of the choice.
// An expert without a share adds nothing, whatever it computed.  Sums of other blocks come from other XCDs: they were stored past the L2s and
// are loaded past them, and each block waits for its stores before it counts its pairs.  One token through 2 of 8 fp16 experts 1024 -> 4096: 8.3 us
// (16.8 MB; dividing its k among two or four blocks is no faster); 13 tokens as above: 37 us, 5.2 TB/s; 64 as above: 18 us.
template <class T, bool MX, bool SHARED, int RT, int WK, int TT>
__global__ __launch_bounds__(64 * WK, TT == 2 ? 3 : 4) void moe_layer_second_kernel(MoeLayerArgs a)
{
    __shared__ ExpertLds<T, MX, SHARED, RT, WK, TT, 1> lds;
    __shared__ unsigned int before;
    extern __shared__ uint4_t xs[];
    const ExpertPointers p = a.experts[blockIdx.y];
    const int first = blockIdx.z * (8 * TT), left = pairs_of(a.chosen, a.tokens * a.top_k, blockIdx.y, lds.list, &lds.count) - first;
    if (left <= 0) return;
    const int n = left < 8 * TT ? left : 8 * TT;
    moe_second<T, MX, SHARED, RT, WK, TT>(a, p, lds.list + first, n, xs, lds.turn);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) before = __hip_atomic_fetch_add(&a.counters[blockIdx.x], (unsigned int)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (before + n != (unsigned int)(a.tokens * a.top_k)) return;
    // A thread has one choice of four rows of a token, so that what comes past the L2s comes at once; the first ones of each sum up.
    constexpr int kWords = 16 * RT / 4;
    float4_t* parts = reinterpret_cast<float4_t*>(lds.turn);
    const int at_once = 64 * WK / a.top_k, mine = threadIdx.x / a.top_k, choice = threadIdx.x % a.top_k;
    for (int i0 = 0; i0 < a.tokens * kWords; i0 += at_once) {
        const int i = i0 + mine, token = i / kWords, d = blockIdx.x * (16 * RT) + i % kWords * 4;
        const bool is = mine < at_once && i < a.tokens * kWords && d < a.d_model;
        if (is) {
            const int pair = token * a.top_k + choice;
            const float c = a.share[pair];
            unsigned long long lo, hi;
            load16_device_scope(a.part + (int64_t)pair * a.d_model + d, lo, hi);
            const uint4_t q = {(unsigned int)lo, (unsigned int)(lo >> 32), (unsigned int)hi, (unsigned int)(hi >> 32)};
            parts[threadIdx.x] = c == 0.0f ? float4_t{} : c * __builtin_bit_cast(float4_t, q);
        }
        __syncthreads();
        if (is && choice == 0) {
            float4_t y = parts[threadIdx.x];
            for (int j = 1; j < a.top_k; ++j) y += parts[threadIdx.x + j];
            store4<T>((typename T::elem*)a.y + (int64_t)token * a.d_model + d, y, 4);
        }
        __syncthreads();
    }
}
}  // namespace pimhip
