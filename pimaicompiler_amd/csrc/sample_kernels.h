// A token drawn from each row of logits.
//
//   w_i = exp((x_i - max x) / T);  of the tokens in falling order of x (equal ones by their index): the first top_k; of them those before which
//   less than top_p of their sum has been reached; of them those with w >= min_p.  The token is the first in the order of indices at which
//   the running sum over what stayed exceeds u times the whole.
//
// One block a row.  Nothing is sorted: top_k and top_p each come down to one value, the smallest that stays, and how many of those equal to
// it do.  It is found by histograms over the values' order (counts, or sums of w): the bucket in which the target is reached is cut into
// buckets again until it is one value.  Sums are whole numbers of 64 bits, w in units of 2^-shift of the largest: they are the same in
// any order.  w itself is worked out in 64 bits (the vector units take as long for an fma of 64 bits as for one of 32): with fp32's 2^-24 a
// number between two tokens of a large vocabulary would fall on the wrong one in some percent of the rows.
#pragma once

#include "row_pieces.h"

namespace pimhip
{
static constexpr int kSampleMost = 1 << 21;   // tokens of a vocabulary
static constexpr int kSegment = 512;          // tokens that a wavefront takes at a time, whose sum is kept
static constexpr int kSegments = kSampleMost / kSegment;

struct SampleArgs {
    const void* logits;
    const float* uniform;
    const float* temperatures;
    const int* top_ks;
    const float* top_ps;
    const float* min_ps;
    int64_t* tokens;
    float* logp;
    int64_t ld;
    int V, shift;  // shift: a weight of 1 is 2^shift, and V of them fit into 62 bits
    float temperature, top_p, min_p;
    int top_k;
};

// 2^f for f in [-1/2, 1/2]: 1 + f q(f), q through (2^f - 1) / f at the eight Chebyshev nodes; off by 2.2e-12 at most.
__device__ __forceinline__ double exp2_near_0(double f)
{
    double q = 1.3250805508543314e-06;
    q = fma(q, f, 1.5303700711228257e-05);
    q = fma(q, f, 0.00015403475186575116);
    q = fma(q, f, 0.0013333478473686068);
    q = fma(q, f, 0.009618129135236074);
    q = fma(q, f, 0.05550410906325866);
    q = fma(q, f, 0.24022650695888503);
    q = fma(q, f, 0.6931471805568324);
    return fma(q, f, 1.0);
}

struct SampleWeight {
    double top, rate, unit;  // largest value, log2(e) / T, 2^shift
    // exp((x - top) / T); what is below 2^-1000 counts as that.
    __device__ __forceinline__ double operator()(float x) const
    {
        const double d = fmax(((double)x - top) * rate, -1000.0), n = rint(d);
        return ldexp(exp2_near_0(d - n), (int)n);
    }
    // The same in whole units, rounded (2^52 added, a double's last bit is one).
    __device__ __forceinline__ uint64_t units(double w) const
    {
        return __builtin_bit_cast(uint64_t, fma(w, unit, 4503599627370496.0)) - 0x4330000000000000ull;
    }
};

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// What stays: x of a key above `key`, the ones equal to it up to index `last`, and none with a weight under `least`.
struct SampleKept {
    unsigned int key;
    int last;
    double least;
};

template <class T, int THREADS>
struct SampleRow {
    static constexpr int kWaves = THREADS / 64;
    static constexpr int kBins = 2 * THREADS;
    struct Shared {
        uint64_t bins[kBins > kSegments ? kBins : kSegments];
        uint64_t waves[kWaves];
        uint64_t found_before, found_amount;
        int found;
    };
    const typename T::elem* x;
    int V;
    Shared& sh;

    // f(index of the first, eight values) for the pieces of a row, thread by thread; behind the row's end values are -inf.
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
        const int pieces = (V + 7) / 8;
        for (int p = threadIdx.x; p < pieces; p += THREADS) {
            float v[8];
            piece(p, v);
            f(p * 8, v);
        }
    }
    __device__ __forceinline__ void piece(int p, float (&v)[8]) const
    {
        if (p * 8 + 8 <= V) {
            load_piece<T>(x, p, v);
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = p * 8 + c < V ? (float)x[p * 8 + c] : -__builtin_inff();
        }
    }

    __device__ __forceinline__ uint64_t block_sum(uint64_t v) const
    {
        v = wave_sum_u64(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.waves[threadIdx.x >> 6] = v;
        __syncthreads();
        uint64_t all = 0;
        for (int w = 0; w < kWaves; ++w) all += sh.waves[w];
        return all;
    }

    // The first of bins[0 .. n) at whose end base + the running sum reaches `target`; the sum before it in `before` (base included), its own in
    // `amount`.  n up to what THREADS take with `each_thread` bins each.  All of the block call it; the target is reached in some bin.
    __device__ __forceinline__ int find_bin(int n, uint64_t base, uint64_t target, uint64_t& before, uint64_t& amount) const
    {
        __syncthreads();
        const int per = (n + THREADS - 1) / THREADS, lo = threadIdx.x * per < n ? threadIdx.x * per : n, hi = lo + per < n ? lo + per : n;
        uint64_t mine = 0;
        for (int i = lo; i < hi; ++i) mine += sh.bins[i];
        uint64_t incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_up(incl, d);
            if ((int)(threadIdx.x & 63) >= d) incl += o;
        }
        if ((threadIdx.x & 63) == 63) sh.waves[threadIdx.x >> 6] = incl;
        __syncthreads();
        uint64_t at = base + incl - mine;
        for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) at += sh.waves[w];
        if (at < target && target <= at + mine) {
            int i = lo;
            while (i < hi - 1 && at + sh.bins[i] < target) at += sh.bins[i++];
            sh.found = i;
            sh.found_before = at;
            sh.found_amount = sh.bins[i];
        }
        __syncthreads();
        before = sh.found_before;
        amount = sh.found_amount;
        return sh.found;
    }

    __device__ __forceinline__ void clear_bins(int n) const
    {
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += THREADS) sh.bins[i] = 0;
        __syncthreads();
    }

    // The largest key such that the amounts of the keys from it on reach `target` (they do over keys lo .. hi), with the sum above it and its own.
    template <class F>
    __device__ __forceinline__ unsigned int select(unsigned int lo, unsigned int hi, uint64_t target, F amount_of, uint64_t& above, uint64_t& amount) const
    {
        above = 0;
        while (true) {
            int s = 0;
            while ((hi - lo) >> s >= (unsigned int)kBins) ++s;
            clear_bins(kBins);
            each([&](int at, const float(&v)[8]) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const unsigned int key = ordered_bits(v[c]);
                    if (key >= lo && key <= hi && at + c < V) atomicAdd((unsigned long long*)&sh.bins[(hi - key) >> s], (unsigned long long)amount_of(v[c]));
                }
            });
            uint64_t before;
            const int bin = find_bin(kBins, above, target, before, amount);
            above = before;
            hi -= (unsigned int)bin << s;
            if (s == 0) return hi;
            const unsigned int down = (1u << s) - 1u;
            lo = hi - lo > down ? hi - down : lo;
        }
    }
};

template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a)
{
    typedef SampleRow<T, THREADS> Row;
    __shared__ typename Row::Shared sh;
    __shared__ unsigned long long best_of[THREADS / 64];
    __shared__ int any_bad;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, V = a.V;
    const Row row{(const typename T::elem*)a.logits + r * a.ld, V, sh};
    const float temperature = a.temperatures ? a.temperatures[r] : a.temperature, top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float min_p = a.min_ps ? a.min_ps[r] : a.min_p, u = a.uniform[r];
    const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    auto answer = [&](int64_t token, float logp) {
        a.tokens[r] = token;
        a.logp[r] = logp;
    };

    // ---- the largest value, and the piece that has it first ----
    if (tid == 0) any_bad = 0;
    __syncthreads();
    unsigned long long best = 0;
    bool bad = false;
    row.each([&](int at, const float(&v)[8]) {
        float top = v[0];
#pragma unroll
        for (int c = 1; c < 8; ++c) top = fmaxf(top, v[c]);
#pragma unroll
        for (int c = 0; c < 8; ++c) bad |= !(v[c] < __builtin_inff());
        const unsigned long long key = (unsigned long long)ordered_bits(top) << 32 | (unsigned int)~(unsigned int)at;
        best = key > best ? key : best;
    });
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned long long o = __shfl_xor(best, d);
        best = o > best ? o : best;
    }
    if (lane == 0) best_of[tid >> 6] = best;
    if (bad) any_bad = 1;
    __syncthreads();
    for (int w = 0; w < THREADS / 64; ++w) best = best_of[w] > best ? best_of[w] : best;
    const unsigned int top_key = (unsigned int)(best >> 32);
    const float top = from_ordered(top_key);
    const bool unfit = !(temperature >= 0.0f && temperature < __builtin_inff()) || top_p != top_p || min_p != min_p || u != u;
    if (any_bad || unfit) {
        if (tid == 0) answer(-1, __builtin_nanf(""));
        return;
    }
    if (top == -__builtin_inff()) {
        if (tid == 0) answer(-1, -__builtin_inff());
        return;
    }
    if (temperature == 0.0f || top_k == 1 || top_p <= 0.0f) {  // the first of the largest is all that stays
        if (tid == 0) {
            const int at = (int)~(unsigned int)best;
            int c = 0;
            while (ordered_bits((float)row.x[at + c]) != top_key) ++c;
            answer(at + c, 0.0f);
        }
        return;
    }

    // ---- what stays ----
    const SampleWeight weight{(double)top, 1.4426950408889634 / (double)temperature, ldexp(1.0, a.shift)};
    SampleKept kept{0u, V, 0.0};
    uint64_t equal_kept = 0;   // how many of the smallest value that stays do, where not all do (0: all)
    const unsigned int bottom_key = ordered_bits(-__builtin_inff());
    if (top_k > 0 && top_k < V) {
        uint64_t above, amount;
        kept.key = row.select(bottom_key, top_key, (uint64_t)top_k, [](float) { return (uint64_t)1; }, above, amount);
        if (above + amount > (uint64_t)top_k) equal_kept = (uint64_t)top_k - above;
    }
    if (top_p < 1.0f) {
        uint64_t whole = 0;
        row.each([&](int, const float(&v)[8]) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const unsigned int key = ordered_bits(v[c]);
                if (equal_kept ? key > kept.key : key >= kept.key) whole += weight.units(weight(v[c]));
            }
        });
        whole = row.block_sum(whole);
        if (equal_kept) whole += equal_kept * weight.units(weight(from_ordered(kept.key)));
        // A token stays where what is before it is less than top_p of the whole, that is less than the whole number at or above that.
        const uint64_t target = (uint64_t)ceil((double)top_p * (double)whole);
        uint64_t above, amount;
        const unsigned int from = kept.key > bottom_key ? kept.key : bottom_key;
        const unsigned int key = row.select(from, top_key, target, [&](float v) { return weight.units(weight(v)); }, above, amount);
        const uint64_t one = weight.units(weight(from_ordered(key)));
        const uint64_t count = (target - above + one - 1) / one, all = amount / one;
        const uint64_t limit = key == kept.key && equal_kept ? equal_kept : all;
        kept.key = key;
        equal_kept = count < limit ? count : limit;
        if (equal_kept == all) equal_kept = 0;
    }
    if (min_p > 0.0f) {
        kept.least = fmin((double)min_p, 1.0);
        if (weight(from_ordered(kept.key)) < kept.least) equal_kept = 0;
    }

    // ---- the index of the last of the equal ones that stay ----
    const int segments = (V + kSegment - 1) / kSegment;
    if (equal_kept) {
        row.clear_bins(segments);
        row.each([&](int at, const float(&v)[8]) {
            int n = 0;
#pragma unroll
            for (int c = 0; c < 8; ++c) n += ordered_bits(v[c]) == kept.key && at + c < V ? 1 : 0;
            if (n) atomicAdd((unsigned long long*)&sh.bins[at / kSegment], (unsigned long long)n);
        });
        uint64_t before, amount;
        const int segment = row.find_bin(segments, 0, equal_kept, before, amount);
        if (tid < 64) {
            float v[8];
            row.piece(segment * 64 + lane < (V + 7) / 8 ? segment * 64 + lane : (V - 1) / 8, v);
            const bool mine = segment * 64 + lane < (V + 7) / 8;
            int n = 0;
            for (int c = 0; c < 8; ++c) n += mine && ordered_bits(v[c]) == kept.key && (segment * 64 + lane) * 8 + c < V ? 1 : 0;
            int incl = n;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int o = __shfl_up(incl, d);
                if (lane >= d) incl += o;
            }
            int at = (int)(before + incl - n);
            if (at < (int)equal_kept && (int)equal_kept <= at + n) {
                int c = 0;
                for (; c < 7; ++c) {
                    at += ordered_bits(v[c]) == kept.key ? 1 : 0;
                    if (at == (int)equal_kept) break;
                }
                sh.found = (segment * 64 + lane) * 8 + c;
            }
        }
        __syncthreads();
        kept.last = sh.found;
        __syncthreads();
    }

    // ---- the draw ----
    auto stays = [&](float v, int at, double w) {
        const unsigned int key = ordered_bits(v);
        return at < V && (key > kept.key || (key == kept.key && at <= kept.last)) && w >= kept.least;
    };
    row.clear_bins(segments);
    {
        const int pieces = (V + 7) / 8;
        for (int p0 = tid & ~63; p0 < pieces; p0 += THREADS) {
            uint64_t sum = 0;
            const int p = p0 + lane;
            if (p < pieces) {
                float v[8];
                row.piece(p, v);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const double w = weight(v[c]);
                    if (stays(v[c], p * 8 + c, w)) sum += weight.units(w);
                }
            }
            sum = wave_sum_u64(sum);
            if (lane == 0) sh.bins[p0 / 64] = sum;
        }
    }
    __syncthreads();
    uint64_t whole = 0;
    for (int i = tid; i < segments; i += THREADS) whole += sh.bins[i];
    whole = row.block_sum(whole);
    const float number = u < 0.0f ? 0.0f : u;
    uint64_t target = (uint64_t)((double)number * (double)whole);
    target = (target < whole ? target : whole - 1) + 1;  // (the running sum reaches it where it exceeds the number's share)
    uint64_t before, amount;
    const int segment = row.find_bin(segments, 0, target, before, amount);
    if (tid < 64) {
        const int p = segment * 64 + lane;
        float v[8];
        uint64_t w[8], sum = 0;
        row.piece(p * 8 < V ? p : (V - 1) / 8, v);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const double e = weight(v[c]);
            w[c] = p * 8 < V && stays(v[c], p * 8 + c, e) ? weight.units(e) : 0;
            sum += w[c];
        }
        uint64_t incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        uint64_t at = before + incl - sum;
        if (at < target && target <= at + sum) {
            bool found = false;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (!found && at + w[c] >= target) {
                    found = true;
                    answer(p * 8 + c, (float)(((double)v[c] - weight.top) / (double)temperature - log((double)whole / weight.unit)));
                }
                at += w[c];
            }
        }
    }
}
}  // namespace pimhip
