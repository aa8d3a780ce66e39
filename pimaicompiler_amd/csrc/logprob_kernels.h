// Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits.
//
//   m = max x,  s = sum exp(x - m),  t = sum exp(x - m) (x - m)
//   log p(token) = x[token] - m - log s          entropy = log s - t / s
//
// One pass over a row by one block: every thread keeps m, s and t of its own pieces (eight values each) in fp32 and, for the
// alternatives, its largest value and the piece that holds it.  Bound by reading the logits.
// Alternatives: the threads form 64 groups; the k-th largest of the groups' best (value, piece) is a bound that at least k values
// reach, so only pieces of threads whose own best reaches it are looked at again (out of the caches).  What reaches the bound goes to
// LDS, some more than k values as a rule, and is ranked there; ties go to the lowest index.
// exp of a value's distance d to m by __expf, off by (1 + |d|) 2^-23 of itself: at most 2^-23 of the row's largest term, since (1 + |d|) e^d <= 1.
// 509 rows of 100003 bf16 logits: 23 us without alternatives (4.4 TB/s; the eight vector instructions and the exponential of a value take about
// 15 of it), 32 with 20 of them: all rows are at work at once, so that the few dependent steps at their ends are not hidden.  Asking for four
// pieces while the four before are looked at: 33.  One row of 32000: 8 us, the steps' latencies.
#pragma once

#include "row_pieces.h"

namespace pimhip
{
static constexpr int kTopMost = 32;            // alternatives a call can ask for
static constexpr float kFarBelow = -10000.0f;  // exp of it is 0, and so is its product with it

// The values of a row, eight at a time, those of thread tid being pieces tid, tid + THREADS, ...: f(piece, its values and those of the next
// three of the thread).  Four pieces are loaded together; behind the row's end, and where there is no piece, they are -inf.
template <class T, int THREADS, class F>
__device__ __forceinline__ void each_four_pieces(const typename T::elem* row, int64_t V, F f)
{
    const int64_t whole = V / 8;
    for (int64_t p = threadIdx.x; p < whole; p += 4 * THREADS) {
        float v[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) load_piece<T>(row, p + i * THREADS < whole ? p + i * THREADS : whole - 1, v[i]);
        if (p - threadIdx.x + 4 * THREADS > whole) {
#pragma unroll
            for (int i = 1; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 8; ++c) v[i][c] = p + i * THREADS < whole ? v[i][c] : -__builtin_inff();
        }
        f(p, v);
    }
    if (V % 8 != 0 && threadIdx.x == whole % THREADS) {
        float v[4][8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            v[0][c] = whole * 8 + c < V ? (float)row[whole * 8 + c] : -__builtin_inff();
            v[1][c] = v[2][c] = v[3][c] = -__builtin_inff();
        }
        f(whole, v);
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
    constexpr int kCandidates = THREADS == 64 ? 1024 : 4096;
    __shared__ unsigned long long candidates[kCandidates + 8];
    __shared__ unsigned short owners[THREADS];
    __shared__ unsigned long long bound, found;
    __shared__ int count, owner_count;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_in_block();
    const int64_t row = blockIdx.x, V = a.V;
    const typename T::elem* x = (const typename T::elem*)a.logits + row * a.ld;

    // ---- the pass ----
    // t only wants the product of a value that is far below with its exp to be 0; what is not finite shows in s.
    float m = -3.402823466e+38f, s = 0.0f, t = 0.0f;
    float best = -__builtin_inff();
    unsigned int best_piece = 0xffffffffu;
    each_four_pieces<T, THREADS>(x, V, [&](int64_t p, const float(&v)[4][8]) {
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            top[i] = v[i][0];
#pragma unroll
            for (int c = 1; c < 8; ++c) top[i] = fmaxf(top[i], v[i][c]);
        }
        const float mn = fmaxf(fmaxf(fmaxf(m, top[0]), fmaxf(top[1], top[2])), top[3]);
        if (mn > best || best_piece == 0xffffffffu) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (top[i] > best || best_piece == 0xffffffffu) {
                    best = top[i];
                    best_piece = (unsigned int)p + i * THREADS;
                }
        }
        const float step = fmaxf(m - mn, kFarBelow), f = __expf(step);
        t = f * (t + s * step);
        s *= f;
        m = mn;
        float ps[4], pt[4];  // (a row's sums grow by a piece's: fewer roundings of what they have)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ps[i] = pt[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float d = v[i][c] - m, e = __expf(d);
                ps[i] += e;
                pt[i] = fmaf(e, fmaxf(d, kFarBelow), pt[i]);
            }
        }
        s += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        t += (pt[0] + pt[1]) + (pt[2] + pt[3]);
    });

    // ---- the row's m, s, t ----
    float bm = wave_max_f32(m);
    if (kWaves > 1) {
        if (lane == 0) wave_f[0][wave] = bm;
        __syncthreads();
        bm = wave_f[0][0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) bm = fmaxf(bm, wave_f[0][i]);
    }
    {
        const float step = fmaxf(m - bm, kFarBelow), f = __expf(step);
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
    const unsigned long long g = group_max_u64<kPerGroup>(mine);
    if (tid % kPerGroup == 0) group_best[tid / kPerGroup] = g;
    if (tid == 0) count = owner_count = 0;
    __syncthreads();
    if (wave == 0) {
        const unsigned long long k = group_best[lane];
        int rank = 0;  // (empty groups, all 0, go by their number)
#pragma unroll
        for (int i = 0; i < 64; ++i) {
            const unsigned long long o = group_best[i];
            rank += o > k || (o == k && i < lane) ? 1 : 0;
        }
        if (rank == top - 1) bound = k;
    }
    __syncthreads();
    // The threads whose best reaches the bound name themselves, and the block looks at their pieces, a thread a piece.
    const unsigned long long at_least = bound;
    const float least = at_least == 0ull ? -__builtin_inff() : from_ordered((unsigned int)(at_least >> 32));
    if (mine != 0ull && mine >= at_least) owners[atomicAdd(&owner_count, 1)] = (unsigned short)tid;
    __syncthreads();
    const unsigned int named = (unsigned int)owner_count, pieces = (unsigned int)((V + 7) / 8), each = (pieces + THREADS - 1) / THREADS;
    for (unsigned int i = tid; i < named * each; i += THREADS) {
        const unsigned int p = owners[i % named] + i / named * THREADS;
        if (p >= pieces) continue;
        float v[8];
        if ((int64_t)p * 8 + 8 <= V) {
            load_piece<T>(x, p, v);
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = (int64_t)p * 8 + c < V ? (float)x[(int64_t)p * 8 + c] : __builtin_nanf("");
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (!(v[c] >= least) || key_of(v[c], p) < at_least) continue;
            const int n = atomicAdd(&count, 1);
            if (n < kCandidates) candidates[n] = key_of(v[c], p * 8 + c);
        }
    }
    __syncthreads();
    auto store = [&](int rank, unsigned long long key) {
        a.top_logp[row * top + rank] = s == 0.0f ? none : from_ordered((unsigned int)(key >> 32)) - bm - log_s;
        a.top_ids[row * top + rank] = (int)~(unsigned int)key;
    };
    const int n = count;
    if (n <= kCandidates) {
        if (tid < 8) candidates[n + tid] = 0ull;  // (a rank is counted eight at a time)
        __syncthreads();
        for (int i = tid; i < n; i += THREADS) {
            const unsigned long long k = candidates[i];
            int rank = 0;
            for (int j = 0; j < n && rank < top; j += 8)
#pragma unroll
                for (int c = 0; c < 8; ++c) rank += candidates[j + c] > k ? 1 : 0;
            if (rank < top) store(rank, k);
        }
        return;
    }
    // More values reach the bound than LDS holds (large ones close together in a very long row): one pass for each alternative.
    unsigned long long below = ~0ull;
    for (int i = 0; i < top; ++i) {
        unsigned long long k = 0;
        each_four_pieces<T, THREADS>(x, V, [&](int64_t first, const float(&v)[4][8]) {
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int64_t at = (first + h * THREADS) * 8 + c;
                    const unsigned long long q = key_of(v[h][c], (unsigned int)at);
                    if (at < V && q < below && (h == 0 || first + h * THREADS < V / 8)) k = larger(k, q);  // (the others are no pieces of the row)
                }
        });
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
