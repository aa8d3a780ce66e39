// Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits.
//
//   m = max x,  s = sum exp(x - m),  t = sum exp(x - m) (x - m)
//   log p(token) = x[token] - m - log s          entropy = log s - t / s
//
// One pass over a row by one block: every thread keeps m, s and t of its own pieces (eight values each) in fp32 and, for the
// alternatives, its largest value and the piece that holds it.  Bound by reading the logits.
// Alternatives: the threads form 64 groups; the k-th largest of the groups' best (value, piece) is a bound that at least k values
// reach, so only threads whose own best reaches it look at their pieces again (out of the caches).  What reaches the bound goes to LDS,
// some more than k values as a rule, and is ranked there; ties go to the lowest index.
#pragma once

#include "mx4_format.h"

namespace pimhip
{
static constexpr int kTopMost = 32;            // alternatives a call can ask for
static constexpr int kTopCandidates = 4096;    // values that may reach the bound before a block goes over to one pass per alternative
static constexpr float kFarBelow = -10000.0f;  // exp of it is 0, and so is its product with it

// A value's place in the order of all values, as a whole number: -0 with 0, infinities at the ends.
__device__ __forceinline__ unsigned int ordered_bits(float v)
{
    const unsigned int b = __builtin_bit_cast(unsigned int, v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float from_ordered(unsigned int o) { return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// d, but nothing below kFarBelow; a NaN stays one.
__device__ __forceinline__ float not_far_below(float d) { return d < kFarBelow ? kFarBelow : d; }

// Eight values of a piece as fp32; those behind the row's end are -inf.
template <class T>
__device__ __forceinline__ void load_piece(const typename T::elem* row, int64_t piece, int64_t V, float (&v)[8])
{
    typename T::elem e[8];
    if (piece * 8 + 8 <= V) {
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
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = piece * 8 + i < V ? (float)row[piece * 8 + i] : -__builtin_inff();
    }
}

struct LogProbArgs {
    const void* logits;
    const void* tokens;  // [rows] int64 or int32, or null
    float* logp;         // [rows]
    float* entropy;      // [rows] or null
    float* top_logp;     // [rows, top]
    int* top_ids;        // [rows, top]
    int64_t V, ld;
    int top;
    int tokens64;
};

template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void token_log_probs_kernel(LogProbArgs a)
{
    constexpr int kWaves = THREADS / 64, kPerGroup = THREADS / 64;
    __shared__ float wave_f[3][kWaves];
    __shared__ unsigned long long group_best[64];
    __shared__ unsigned long long candidates[kTopCandidates];
    __shared__ unsigned long long bound, found;
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_in_block();
    const int64_t row = blockIdx.x, V = a.V;
    const typename T::elem* x = (const typename T::elem*)a.logits + row * a.ld;
    const int64_t pieces = (V + 7) / 8;

    // ---- the pass ----
    float m = -3.402823466e+38f, s = 0.0f, t = 0.0f;
    float best = -__builtin_inff();
    unsigned int best_piece = 0xffffffffu;
    for (int64_t p = tid; p < pieces; p += THREADS) {
        float v[8];
        load_piece<T>(x, p, V, v);
        float top = v[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, v[i]);
        if (top > best || best_piece == 0xffffffffu) {
            best = top;
            best_piece = (unsigned int)p;
        }
        const float mn = fmaxf(m, top);
        const float step = not_far_below(m - mn), f = __expf(step);
        t = f * (t + s * step);
        s *= f;
        m = mn;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = not_far_below(v[i] - m), e = __expf(d);
            s += e;
            t += e * d;
        }
    }

    // ---- the row's m, s, t ----
    float bm = m;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) bm = fmaxf(bm, __shfl_xor(bm, i));
    if (kWaves > 1) {
        if (lane == 0) wave_f[0][wave] = bm;
        __syncthreads();
        bm = wave_f[0][0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) bm = fmaxf(bm, wave_f[0][i]);
    }
    {
        const float step = not_far_below(m - bm), f = __expf(step);
        t = f * (t + s * step);
        s *= f;
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if (kWaves > 1) {
        if (lane == 0) {
            wave_f[1][wave] = s;
            wave_f[2][wave] = t;
        }
        __syncthreads();
        s = wave_f[1][0];
        t = wave_f[2][0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) {
            s += wave_f[1][i];
            t += wave_f[2][i];
        }
    }
    // A row with a NaN or +inf has no distribution (s is NaN); one of -inf alone leaves nothing (s is 0): every probability 0.
    const float log_s = s == 0.0f ? 0.0f : logf(s);
    const float none = s == 0.0f ? -__builtin_inff() : 0.0f;
    if (tid == 0) {
        if (a.logp) {
            const int64_t token = a.tokens64 ? ((const int64_t*)a.tokens)[row] : ((const int*)a.tokens)[row];
            float v = token < 0 ? 0.0f : __builtin_nanf("");
            if (token >= 0 && token < V) v = s == 0.0f ? none : (float)x[token] - bm - log_s;
            a.logp[row] = v;
        }
        if (a.entropy) a.entropy[row] = s == 0.0f ? 0.0f : log_s - t / s;
    }
    const int top = a.top;
    if (top == 0) return;
    if (s != s) {
        for (int i = tid; i < top; i += THREADS) {
            a.top_logp[row * top + i] = __builtin_nanf("");
            a.top_ids[row * top + i] = -1;
        }
        return;
    }

    // ---- the alternatives ----
    auto key_of = [](float v, unsigned int at) { return ((unsigned long long)ordered_bits(v) << 32) | (unsigned int)~at; };
    auto larger = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
    const unsigned long long mine = best_piece == 0xffffffffu ? 0ull : key_of(best, best_piece);
    unsigned long long g = mine;
#pragma unroll
    for (int i = 1; i < kPerGroup; i <<= 1) g = larger(g, __shfl_xor(g, i));
    if (tid % kPerGroup == 0) group_best[tid / kPerGroup] = g;
    if (tid == 0) count = 0;
    __syncthreads();
    if (wave == 0) {
        const unsigned long long k = group_best[lane];
        int rank = 0;  // (empty groups, all 0, go by their number)
        for (int i = 0; i < 64; ++i) {
            const unsigned long long o = group_best[i];
            rank += o > k || (o == k && i < lane) ? 1 : 0;
        }
        if (rank == top - 1) bound = k;
    }
    __syncthreads();
    const unsigned long long at_least = bound;
    if (mine != 0ull && mine >= at_least) {
        for (int64_t p = tid; p < pieces; p += THREADS) {
            float v[8];
            load_piece<T>(x, p, V, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (p * 8 + i >= V || key_of(v[i], (unsigned int)p) < at_least) continue;
                const int n = atomicAdd(&count, 1);
                if (n < kTopCandidates) candidates[n] = key_of(v[i], (unsigned int)(p * 8 + i));
            }
        }
    }
    __syncthreads();
    auto store = [&](int rank, unsigned long long key) {
        a.top_logp[row * top + rank] = s == 0.0f ? none : from_ordered((unsigned int)(key >> 32)) - bm - log_s;
        a.top_ids[row * top + rank] = (int)~(unsigned int)key;
    };
    const int n = count;
    if (n <= kTopCandidates) {
        for (int i = tid; i < n; i += THREADS) {
            const unsigned long long k = candidates[i];
            int rank = 0;
            for (int j = 0; j < n && rank < top; ++j) rank += candidates[j] > k ? 1 : 0;
            if (rank < top) store(rank, k);
        }
        return;
    }
    // More values reach the bound than LDS holds (large ones close together in a very long row): one pass for each alternative.
    unsigned long long below = ~0ull;
    for (int i = 0; i < top; ++i) {
        unsigned long long k = 0;
        for (int64_t p = tid; p < pieces; p += THREADS) {
            float v[8];
            load_piece<T>(x, p, V, v);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const unsigned long long q = key_of(v[c], (unsigned int)(p * 8 + c));
                if (p * 8 + c < V && q < below) k = larger(k, q);
            }
        }
        __syncthreads();
        if (tid == 0) found = 0ull;
        __syncthreads();
        atomicMax(&found, k);
        __syncthreads();
        below = found;
        if (tid == 0) store(i, below);
    }
}
}  // namespace pimhip
