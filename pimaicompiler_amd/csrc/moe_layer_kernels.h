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
    float* h;         // [pairs][ld_h]: hidden values
    uint8_t* h_most;  // [pairs][ld_most]: the exponent field of the largest of each 16 of them, where the second product asks for it
    float* part;      // [pairs][d_model]
    unsigned int* counters;  // pairs whose second product is done, for each tile of rows
    int counters_used;
    int tokens, E, top_k, d_model, d_ff, ld_x;
    int ld_h;         // d_ff filled up to whole groups of eight, with zeros
    int ld_most;      // a multiple of 16
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
};
template <class T, int TT>
struct ExpertWeights<T, true, TT> {
    typedef Mx4Weights<T, TT == 1 ? 2 : 1> W;
    static __device__ __forceinline__ typename W::Rows rows(const void* w, const void* s, const void* t, int ld, int64_t first, int64_t count, int K)
    {
        return W::rows((const uint8_t*)w, (const uint8_t*)s, (const uint8_t*)t, ld, first, count, K);
    }
};

// ---- hidden values as operands -----------------------------------------------------------------------------------------------
// A hidden value is fp32; the second product takes it in pieces of the matrix cores' 16-bit type, each a column of its own, so that
// 16-bit hidden values are not what limits y.  Where a first piece's sum is not finite (an infinity among the hidden values or the
// weights) it is the result: the other pieces have a zero, or a NaN, in that place.
//   bfloat16 has fp32's range and 8 of its 24 bits: three pieces of eight bits are the value itself (from 2^-110 on:
//   below, the last bits are under its smallest subnormal).
//   fp16 has not the range.  A pair's hidden values are multiplied by the power of two that brings the largest one to 2^14 or above, and y
//   by its inverse; the second piece is what the first left over, 2^11 times: 22 bits of what is above 2^-29 of the pair's largest, and
//   2^-50 of that for the rest.
// They are taken apart by each block of the second product: stored in pieces by the first one they are more bytes, 64 tokens through 8 gated
// bfloat16 experts 1024 -> 4096 66.8 us a call, not 58.
template <class T>
struct Pieces;
template <>
struct Pieces<BF16> {
    static constexpr int kCount = 3;
    static constexpr bool kScaled = false;
    static __device__ __forceinline__ void prepare(float (&)[8], int) {}
    // The next piece of eight values, which keep what is left.
    static __device__ __forceinline__ uint4_t take(float (&v)[8])
    {
        uint4_t q;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned int a = __builtin_bit_cast(unsigned int, v[2 * i]), b = __builtin_bit_cast(unsigned int, v[2 * i + 1]);
            q[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            v[2 * i] -= __builtin_bit_cast(float, a & 0xffff0000u);
            v[2 * i + 1] -= __builtin_bit_cast(float, b & 0xffff0000u);
        }
        return q;
    }
    static __device__ __forceinline__ float rest(const float (&p)[3]) { return p[1] + p[2]; }
};
template <>
struct Pieces<F16> {
    static constexpr int kCount = 2;
    static constexpr bool kScaled = true;
    static __device__ __forceinline__ void prepare(float (&v)[8], int e)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_amdgcn_ldexpf(v[i], e);
    }
    static __device__ __forceinline__ uint4_t take(float (&v)[8])
    {
        half8_t h;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[i] = (half_t)v[i];
            v[i] = (v[i] - (float)h[i]) * 2048.0f;
        }
        return __builtin_bit_cast(uint4_t, h);
    }
    static __device__ __forceinline__ float rest(const float (&p)[2]) { return p[1] * 0x1p-11f; }
};

// The sum of a hidden row's pieces' products.
template <class T>
__device__ __forceinline__ float join_pieces(const float (&p)[Pieces<T>::kCount])
{
    return fabsf(p[0]) < __builtin_inff() ? p[0] + Pieces<T>::rest(p) : p[0];
}

// The exponents that the hidden values of a block's n pairs are lifted by: 14 less that of the largest one, found among those of the first
// product's tiles by 16 lanes a pair, 16 tiles a load.  (One atomic maximum a pair instead took 6 us longer for one token of 4096 hidden values, a
// tile a lane and a wavefront a pair 11 us for 64.)
template <class T, int WK, class F>
__device__ __forceinline__ void find_lifts(const MoeLayerArgs& a, int n, F pair, int* lift)
{
    if constexpr (Pieces<T>::kScaled) {
        const int tiles = (a.d_ff + 15) / 16;
        for (int i = threadIdx.x / 16; i < 16; i += 4 * WK) {
            const uint8_t* p = a.h_most + (int64_t)pair(i < n ? i : n - 1) * a.ld_most;
            unsigned int most = 0;
            for (int t = (threadIdx.x & 15) * 16; t < tiles; t += 256) {
                const uint4_t q = *reinterpret_cast<const uint4_t*>(p + t);
#pragma unroll
                for (int b = 0; b < 16; ++b) {
                    const unsigned int field = t + b < tiles ? q[b / 4] >> (b % 4 * 8) & 255u : 0u;
                    most = field > most ? field : most;
                }
            }
            auto larger = [&](unsigned int o) { most = o > most ? o : most; };
            larger(dpp_u32<kDppQuadXor1>(most));
            larger(dpp_u32<kDppQuadXor2>(most));
            larger(dpp_u32<kDppRowHalfMirror>(most));
            larger(dpp_u32<kDppRowMirror>(most));
            if ((threadIdx.x & 15) == 0) lift[i] = 14 + 127 - (int)most;
        }
        __syncthreads();
    }
}

// The hidden rows of up to 16 pairs, loaded, taken apart and turned by each wavefront (the other kinds of columns: skinny.h).  FEW: the pieces of
// n pairs are columns of one tile, piece p of pair i column p n + i; else each piece is a tile.
template <class T, bool FEW>
struct HiddenTokens {
    typedef DenseTile<T> Tile;
    typedef Pieces<T> P;
    static constexpr int kLds = Tile::kLds, kRows = FEW ? 2 : 4;
    static_assert(!FEW || 16 / P::kCount <= 4 * kRows, "a lane's rows cover the pairs");
    static constexpr int raws(int) { return 1; }
    struct Rows {
        const float* p[kRows];  // the lane's rows, at its chunk
        const int* lift;        // in LDS, of each pair
        int n;
    };
    struct Raw {
        float v[kRows][8];
    };
    // pair(i): the i-th pair
    template <class F>
    static __device__ __forceinline__ Rows rows(const MoeLayerArgs& a, int n, F pair, const int* lift)
    {
        Rows r;
        const int lane = threadIdx.x & 63;
        r.n = n;
        r.lift = lift;
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int i = pair(lane / 16 + 4 * j < n ? lane / 16 + 4 * j : n - 1);
            r.p[j] = a.h + (int64_t)i * a.ld_h + (lane & 15) * 8;
        }
        return r;
    }
    static __device__ __forceinline__ void load8(float (&v)[8], const float* p)
    {
        const float4_t lo = *reinterpret_cast<const float4_t*>(p), hi = *reinterpret_cast<const float4_t*>(p + 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            v[c] = lo[c];
            v[4 + c] = hi[c];
        }
    }
    static __device__ __forceinline__ void load(Raw& w, const Rows& r, int step)
    {
#pragma unroll
        for (int j = 0; j < kRows; ++j) load8(w.v[j], r.p[j] + (int64_t)step * kSkinnyStep);
    }
    static __device__ __forceinline__ void load_guarded(Raw& w, const Rows& r, int step, int K)
    {
        const bool in = step * kSkinnyStep + (int)(threadIdx.x & 15) * 8 < K;  // (rows are whole groups of eight)
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            if (in)
                load8(w.v[j], r.p[j] + (int64_t)step * kSkinnyStep);
            else
#pragma unroll
                for (int c = 0; c < 8; ++c) w.v[j][c] = 0.0f;
        }
    }
    static __device__ __forceinline__ void turn(typename T::frag (&f)[4], Raw& w, const Rows& r, int, int tile, uint4_t* lds)
    {
        const int lane = threadIdx.x & 63, chunk = lane & 15;
        if (tile == 0)
#pragma unroll
            for (int j = 0; j < kRows; ++j) P::prepare(w.v[j], P::kScaled ? r.lift[lane / 16 + 4 * j < r.n ? lane / 16 + 4 * j : r.n - 1] : 0);
#pragma unroll
        for (int p = 0; p < (FEW ? P::kCount : 1); ++p)
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                // (rows behind the last pair hold that one again, and go where it goes)
                const int row = lane / 16 + 4 * j, column = FEW ? p * r.n + (row < r.n ? row : r.n - 1) : row;
                lds[column * 16 + (chunk ^ (column & 7))] = P::take(w.v[j]);
            }
        wave_lds_order();
        Tile::from_lds(f, lds);
        wave_lds_order();
    }
    // Into the block's columns of SharedTokens, piece p of pair i column p n + i.
    template <class F>
    static __device__ __forceinline__ void stage(uint4_t* xs, const MoeLayerArgs& a, int n, F pair, const int* lift, int K, int pitch)
    {
        const int chunks = pitch - 1;
        for (int at = threadIdx.x; at < n * chunks; at += blockDim.x) {
            const int i = at / chunks, c = at % chunks;
            float v[8] = {};
            if (c * 8 < K) load8(v, a.h + (int64_t)pair(i) * a.ld_h + c * 8);
            P::prepare(v, P::kScaled ? lift[i] : 0);
#pragma unroll
            for (int p = 0; p < P::kCount; ++p) xs[(p * n + i) * pitch + c] = P::take(v);
        }
    }
};

// What a block of the experts' products has in LDS: the tokens that chose its expert, and what its wavefronts turn operands in (and then their
// sums, PARTS tiles of RT rows each).  Where columns are SharedTokens, their values lie in the launch's dynamic part.
template <class W, class X, int RT, int WK, int PARTS>
struct ExpertLds {
    static constexpr int kTurn = kSkinnyLds<W, X>, kSum = RT * PARTS * 64;
    uint4_t turn[WK * (kTurn > kSum ? kTurn : kSum)];
    uint8_t tops[16 * RT];  // the largest scale codes of a block's rows, where they are in 4 bits
    short list[kMoeLayerPairs];
    int count;
};

// Sums of 16 * RT rows for TT tiles of columns.  Ends with every wavefront having those of its own k in `lds`, part[wave][i][j][lane] being
// sums(acc[i], j) for PARTS tiles.
template <class T, class W, class X, int RT, int TT, int WK, int PARTS, class R, class F>
__device__ __forceinline__ void expert_sums(const typename W::Rows (&rows)[RT], const typename X::Rows (&x)[X::raws(TT)], int K, uint4_t* lds, R ready, F sums)
{
    const int lane = threadIdx.x & 63, wave = wave_in_block();
    float4_t acc[RT][TT] = {};
    skinny_sum<T, W, X, RT, TT>(acc, rows, x, K, wave, WK, lds + wave * kSkinnyLds<W, X>, ready);
    __syncthreads();
    float4_t* part = reinterpret_cast<float4_t*>(lds);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < PARTS; ++j) part[((wave * RT + i) * PARTS + j) * 64 + lane] = sums(acc[i], j);
    __syncthreads();
}

// What lane `lane` has of tile i of the wavefronts' sums, in their order.
template <int RT, int WK>
__device__ __forceinline__ float4_t joined(const uint4_t* lds, int i, int lane)
{
    const float4_t* part = reinterpret_cast<const float4_t*>(lds) + i * 64 + lane;
    float4_t v = part[0];
#pragma unroll
    for (int k = 1; k < WK; ++k) v += part[k * RT * 64];
    return v;
}

// The first product of up to 16 TT pairs: hidden values 16 * F a block, each with its gate where there is one.
template <class T, bool MX, bool SHARED, int TT>
struct FirstColumns {
    typedef typename ExpertWeights<T, MX, TT>::W W;
    typedef typename std::conditional<SHARED, SharedTokens<T>, TurnedTokens<T, true>>::type X;
};
template <class T, bool MX, bool SHARED, bool GATED, int F, int WK, int TT>
__device__ __forceinline__ void moe_first(const MoeLayerArgs& a, const ExpertPointers& p, const short* list, int n, uint8_t* tops, uint4_t* xs, uint4_t* lds)
{
    constexpr int RT = GATED ? 2 * F : F;
    static_assert(!SHARED || TT == 1, "tokens are staged as one tile");
    typedef ExpertWeights<T, MX, TT> EW;
    typedef typename FirstColumns<T, MX, SHARED, TT>::W W;
    typedef typename FirstColumns<T, MX, SHARED, TT>::X X;
    const int lane = threadIdx.x & 63, wave = wave_in_block(), group = lane >> 4;
    const int f0 = blockIdx.x * (16 * F), pitch = SharedTokens<T>::pitch(a.d_model, W::kUnit);
    // (value rows follow the gate rows; each kind ends at its own last row)
    auto end_of = [&](int i) { return i < F ? a.d_ff : 2 * a.d_ff; };
    auto row_at = [&](int i, int r) {
        const int at = (i < F ? 0 : a.d_ff) + f0 + i % F * 16 + r;
        return at < end_of(i) ? at : end_of(i) - 1;
    };
    uint8_t top = 0;
    if (MX && threadIdx.x < 16 * RT) top = ((const uint8_t*)p.t1)[row_at(threadIdx.x / 16, threadIdx.x % 16)];
    typename W::Rows rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) rows[i] = EW::rows(p.w1, p.s1, p.t1, a.ld_s1, row_at(i, 0), end_of(i), a.d_model);
    auto token = [&](int i) { return (const typename T::elem*)a.x + (int64_t)(list[i] / a.top_k) * a.ld_x; };
    typename X::Rows x[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        auto at = [&](int i) { return j * 16 + i < n ? j * 16 + i : n - 1; };  // (columns behind the last one: that one again)
        if constexpr (SHARED)
            x[j] = X::rows(xs, at(lane & 15), pitch);
        else
            x[j] = X::rows([&](int i) { return token(at(i)); });
    }
    expert_sums<T, W, X, RT, TT, WK, TT>(
        rows, x, a.d_model, lds,
        [&] {
            if (MX && threadIdx.x < 16 * RT) tops[threadIdx.x] = top;
            if constexpr (SHARED) {
                X::stage(xs, token, n, a.d_model, pitch);
                __syncthreads();
            }
        },
        [](const float4_t(&acc)[TT], int j) { return acc[j]; });
#pragma unroll
    for (int k = 0; k < F * TT; ++k) {
        const int i = k / TT, j = k % TT, f = f0 + i * 16 + group * 4, column = j * 16 + (lane & 15);
        if (k % WK != wave) continue;
        unsigned int most = 0;
        if (column < n && f < a.ld_h) {
            const float4_t g = joined<RT * TT, WK>(lds, k, lane);
            float4_t u = {}, h;
            if constexpr (GATED) u = joined<RT * TT, WK>(lds, (F + i) * TT + j, lane);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                h[c] = 0.0f;
                if (f + c >= a.d_ff) continue;
                float v = MX ? __builtin_amdgcn_ldexpf(g[c], T::exponent(tops[i * 16 + group * 4 + c])) : g[c];
                if (p.b1) v += (float)((const typename T::elem*)p.b1)[f + c];
                if (a.act == PIMHIP_EXPERT_RELU) v = relu_f32(v);
                if (a.act == PIMHIP_EXPERT_SILU) v = v / (1.0f + expf(-v));
                if (GATED) {
                    float w = MX ? __builtin_amdgcn_ldexpf(u[c], T::exponent(tops[(F + i) * 16 + group * 4 + c])) : u[c];
                    if (p.b1) w += (float)((const typename T::elem*)p.b1)[a.d_ff + f + c];
                    v *= w;
                }
                h[c] = v;
                const unsigned int bits = __builtin_bit_cast(unsigned int, v) & 0x7fffffffu;
                most = bits > most ? bits : most;
            }
            *reinterpret_cast<float4_t*>(a.h + (int64_t)list[column] * a.ld_h + f) = h;
        }
        if constexpr (Pieces<T>::kScaled) {
            const auto q = __builtin_amdgcn_permlane16_swap(most, most, false, false);
            most = q[0] > q[1] ? q[0] : q[1];
            const auto r = __builtin_amdgcn_permlane32_swap(most, most, false, false);
            most = r[0] > r[1] ? r[0] : r[1];
            if (group == 0 && column < n && f < a.ld_h) a.h_most[(int64_t)list[column] * a.ld_most + f / 16] = (uint8_t)(most >> 23);
        }
    }
}

// Block (x, y, z): rows x of expert y for 16 TT of its pairs, from 16 TT z on; those of more pairs read the weights again, out of the
// caches.  (A loop over pairs in one block instead costs so many registers that half the wavefronts fit: 39 us against 25 for 64 tokens
// through 8 gated 4-bit experts 1024 -> 4096, before blocks had twice the rows.)  That case takes 19.5 us now with TT 2, 35.7 MB; a block's chain of
// loads (its pairs, then weights and values, k being a unit or two a wavefront) is what it waits for.  13 tokens through 64 gated bf16 experts 2048 -> 1024, six
// chosen: 61 us, 5.5 TB/s.
template <class T, bool MX, bool SHARED, bool GATED, int F, int WK, int TT>
__global__ __launch_bounds__(64 * WK, TT > 1 ? 2 : F > 2 || (GATED && F > 1) ? 3 : 4) void moe_layer_first_kernel(MoeLayerArgs a)
{
    typedef FirstColumns<T, MX, SHARED, TT> C;
    __shared__ ExpertLds<typename C::W, typename C::X, GATED ? 2 * F : F, WK, TT> lds;
    extern __shared__ uint4_t xs[];
    const ExpertPointers p = a.experts[blockIdx.y];
    const int first = blockIdx.z * (16 * TT), n = pairs_of(a.chosen, a.tokens * a.top_k, blockIdx.y, lds.list, &lds.count) - first;
    if (n > 0) moe_first<T, MX, SHARED, GATED, F, WK, TT>(a, p, lds.list + first, n < 16 * TT ? n : 16 * TT, lds.tops, xs, lds.turn);
}

// The second product: rows of d_model, with the bias, not yet weighted.  FEW: of as many pairs as have their pieces in one tile; else of up to 16.
template <class T, bool MX, bool SHARED, bool FEW>
struct SecondColumns {
    typedef ExpertWeights<T, MX, FEW ? 1 : 2> EW;
    typedef typename EW::W W;
    typedef HiddenTokens<T, FEW> Turned;
    typedef typename std::conditional<SHARED, SharedTokens<T>, Turned>::type X;
    static constexpr int kPieces = Pieces<T>::kCount, kTiles = FEW ? 1 : kPieces, kPairs = FEW ? 16 / kPieces : 16;
};
template <class T, bool MX, bool SHARED, int RT, int WK, bool FEW>
__device__ __forceinline__ void moe_second(const MoeLayerArgs& a, const ExpertPointers& p, const short* list, int n, int* lift, uint8_t* tops, uint4_t* xs, uint4_t* lds)
{
    typedef SecondColumns<T, MX, SHARED, FEW> C;
    typedef typename C::EW EW;
    typedef typename C::W W;
    typedef typename C::X X;
    constexpr int P = C::kPieces, TT = C::kTiles;
    const int lane = threadIdx.x & 63, wave = wave_in_block(), group = lane >> 4;
    const int d0 = blockIdx.x * (16 * RT), pitch = SharedTokens<T>::pitch(a.d_ff, W::kUnit);
    auto row_at = [&](int r) { return d0 + r < a.d_model ? d0 + r : a.d_model - 1; };
    uint8_t top = 0;
    if (MX && threadIdx.x < 16 * RT) top = ((const uint8_t*)p.t2)[row_at(threadIdx.x)];
    typename W::Rows rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) rows[i] = EW::rows(p.w2, p.s2, p.t2, a.ld_s2, row_at(i * 16), a.d_model, a.d_ff);
    auto pair_at = [&](int i) { return (int)list[i]; };
    typename X::Rows x[X::raws(TT)];
    if constexpr (SHARED) {
#pragma unroll
        for (int j = 0; j < TT; ++j) {  // (columns behind the last one: that one again)
            const int i = lane & 15, last = FEW ? P * n - 1 : n - 1;
            x[j] = X::rows(xs, j * n + (i < last ? i : last), pitch);
        }
    } else {
        x[0] = X::rows(a, n, pair_at, lift);
    }
    expert_sums<T, W, X, RT, TT, WK, 1>(
        rows, x, a.d_ff, lds,
        [&] {
            if (MX && threadIdx.x < 16 * RT) tops[threadIdx.x] = top;
            find_lifts<T, WK>(a, n, pair_at, lift);
            if constexpr (SHARED) {
                C::Turned::stage(xs, a, n, pair_at, lift, a.d_ff, pitch);
                __syncthreads();
            }
        },
        [](const float4_t(&acc)[TT], int) {
            if constexpr (FEW) return acc[0];
            float4_t v;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float q[C::kPieces];
#pragma unroll
                for (int j = 0; j < C::kPieces; ++j) q[j] = acc[j % C::kTiles][c];
                v[c] = join_pieces<T>(q);
            }
            return v;
        });
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int d = d0 + i * 16 + group * 4, pair = lane & 15;
        if (i % WK != wave || pair >= n || d >= a.d_model) continue;
        float4_t v;
        if constexpr (FEW) {
            float4_t q[P];
#pragma unroll
            for (int j = 0; j < P; ++j) q[j] = joined<RT, WK>(lds, i, group * 16 + j * n + pair);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float s[P];
#pragma unroll
                for (int j = 0; j < P; ++j) s[j] = q[j][c];
                v[c] = join_pieces<T>(s);
            }
        } else {
            v = joined<RT, WK>(lds, i, lane);
        }
        const int at = list[pair];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int up = (MX ? T::exponent(tops[i * 16 + group * 4 + c]) : 0) - (Pieces<T>::kScaled ? lift[pair] : 0);
            if (MX || Pieces<T>::kScaled) v[c] = __builtin_amdgcn_ldexpf(v[c], up);
            if (p.b2) v[c] += (float)((const typename T::elem*)p.b2)[d + c];
        }
        const uint4_t q = __builtin_bit_cast(uint4_t, v);
        store16_device_scope(a.part + (int64_t)at * a.d_model + d, q[0] | (unsigned long long)q[1] << 32, q[2] | (unsigned long long)q[3] << 32);
    }
}

// Blocks as above, with kPairs pairs.  The one whose pairs are the last of a tile of rows makes the weighted sum there, in the order of the choice.
// An expert without a share adds nothing, whatever it computed.  Sums of other blocks come from other XCDs: they were stored past the L2s and
// are loaded past them, and each block waits for its stores before it counts its pairs.  One token through 2 of 8 fp16 experts 1024 -> 4096: 8.5 us
// (16.8 MB; dividing its k among two or four blocks is no faster); 13 tokens as above: 34 us, 5.0 TB/s; 64 as above: 22 us.
template <class T, bool MX, bool SHARED, int RT, int WK, bool FEW>
__global__ __launch_bounds__(64 * WK, FEW || WK == 8 ? 4 : 3) void moe_layer_second_kernel(MoeLayerArgs a)
{
    typedef SecondColumns<T, MX, SHARED, FEW> C;
    __shared__ ExpertLds<typename C::W, typename C::X, RT, WK, 1> lds;
    __shared__ unsigned int before;
    __shared__ int lift[16];
    extern __shared__ uint4_t xs[];
    const ExpertPointers p = a.experts[blockIdx.y];
    const int first = blockIdx.z * C::kPairs, left = pairs_of(a.chosen, a.tokens * a.top_k, blockIdx.y, lds.list, &lds.count) - first;
    if (left <= 0) return;
    const int n = left < C::kPairs ? left : C::kPairs;
    moe_second<T, MX, SHARED, RT, WK, FEW>(a, p, lds.list + first, n, lift, lds.tops, xs, lds.turn);
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
