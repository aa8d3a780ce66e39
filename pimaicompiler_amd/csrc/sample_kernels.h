// A token drawn from each row of logits.
//
//   w_i = exp((x_i - max x) / T);  of the tokens in falling order of x (equal ones by their index): the first top_k; of them those before which
//   less than top_p of their sum has been reached; of them those with w >= min_p.  The token is the first in the order of indices at which
//   the running sum over what stayed exceeds u times the whole.
//
// One block a row.  The first pass finds the largest value and, where the sum over all tokens is asked for, that too.  What may stay is
// above a bound that this pass gives (top_k: the k-th largest of the threads' own largest values; top_p: tokens below (1 - top_p) / V of the sum
// cannot be among those that reach top_p of it, since all of them together do not have the rest; min_p: its own), and goes to a list
// in LDS in a second pass, out of the caches.  Up to 64 such tokens are put into order by one wavefront.
// Of more nothing is sorted: top_k and top_p each come down to one value, the smallest that stays, and how many of those equal to it do.  It
// is found by histograms over the values' order (counts, or sums of w): the bucket in which the target is reached is cut into buckets again
// until it is one value.  The same goes for the draw, over indices.  Rows whose list would not fit (flat distributions, a large top_k) are read
// again in place of it.
// Sums are whole numbers of 64 bits, w in units of 2^-shift of the largest: they are the same in any order.  w itself is worked out in 64 bits (the
// vector units take as long for an fma of 64 bits as for one of 32): with fp32's 2^-24 a number between two tokens of a large vocabulary would
// fall on the wrong one in some percent of the rows.
#pragma once

#include "row_pieces.h"

namespace pimhip
{
static constexpr int kSampleMost = 1 << 21;   // tokens of a vocabulary
static constexpr int kSegment = 512;          // tokens that a wavefront takes at a time, whose sum is kept
static constexpr int kSegments = kSampleMost / kSegment;
static constexpr int kListMost = 4096;        // tokens of a row's list
static constexpr double kExponents = 900.0;   // largest values up to 2^+-this are summed as they are, in the first pass

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

// 2^d, d from -1000 on (below: that) to 1000.  1.5 2^52 added leaves d's nearest whole number in the last bits, which go to the result's
// exponent as they are.
__device__ __forceinline__ double exp2_f64(double d)
{
    d = fmax(d, -1000.0);
    const double t = d + 6755399441055744.0, q = exp2_near_0(d - (t - 6755399441055744.0));
    const uint64_t n = (uint64_t)(unsigned int)__builtin_bit_cast(uint64_t, t) << 52;
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, q) + n);
}

struct SampleWeight {
    double top, rate, unit;  // largest value, log2(e) / T, 2^shift
    // exp((x - top) / T)
    __device__ __forceinline__ double operator()(float x) const { return exp2_f64(((double)x - top) * rate); }
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

// A share of the whole, as whole numbers.  The first pass's sums and those relative to the largest value differ by up to 4.3e-12 of themselves, so shares
// are moved by 2^-36 of theirs: one that meets a border exactly (equal weights) is on the border's right side whichever it is compared with.
// The draw falls on the token at which the running sum reaches sample_target(); what reaches nucleus_target() takes no more tokens.
static constexpr double kBorder = 0x1p-36;
__device__ __forceinline__ uint64_t sample_target(float u, uint64_t whole)
{
    const uint64_t t = (uint64_t)((double)(u < 0.0f ? 0.0f : u) * (1.0 + kBorder) * (double)whole);
    return (t < whole ? t : whole - 1) + 1;
}
__device__ __forceinline__ uint64_t nucleus_target(float top_p, uint64_t whole)
{
    const uint64_t t = (uint64_t)((double)top_p * (1.0 - kBorder) * (double)whole);
    return t < 1 ? 1 : t;
}

// What stays: values of a key above `key`, the ones equal to it up to index `last`, and none with a weight under `least`.
struct SampleKept {
    unsigned int key;
    int last;
    double least;
};

template <class T, int THREADS>
struct SampleRow {
    static constexpr int kWaves = THREADS / 64;
    static constexpr int kBins = 2048;
    // fp32 words of 16-bit values end in zeros (in their order, in zeros or ones): these bits tell no two of them apart.
    static constexpr int kDrop = __is_same(T, F16) ? 13 : __is_same(T, BF16) ? 16 : 0;
    struct Shared {
        union {
            uint64_t bins[kSegments];
            double segments[kSegments];
        };
        unsigned int list_key[kListMost];
        int list_at[kListMost];
        uint64_t waves[kWaves];
        double waves_f[kWaves];
        unsigned long long best[kWaves];
        uint64_t found_before, found_amount;
        int found, count, bad;
    };
    const typename T::elem* x;
    int V;
    Shared& sh;

    static __device__ __forceinline__ unsigned int key_of(float v) { return ordered_bits(v) >> kDrop; }
    static __device__ __forceinline__ float value_of(unsigned int key)
    {
        const unsigned int o = key << kDrop;  // (a negative value's dropped bits are ones)
        return from_ordered(o & 0x80000000u ? o : o | ((1u << kDrop) - 1u));
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
    // f(number of the segment, index of the first value, eight values) for the pieces of a row, a segment by each wavefront, four at a time;
    // behind the row's end values are -inf.
    template <class F>
    __device__ __forceinline__ void each_segment(F f) const
    {
        const int segments = (V + kSegment - 1) / kSegment, lane = threadIdx.x & 63, whole = V / 8;
        for (int first = wave_in_block(); first < segments; first += 4 * kWaves) {
            float v[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = (first + i * kWaves) * 64 + lane;
                if (p < whole) {
                    load_piece<T>(x, p, v[i]);
                } else {
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[i][c] = p * 8 + c < V ? (float)x[p * 8 + c] : -__builtin_inff();
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (first + i * kWaves < segments) f(first + i * kWaves, ((first + i * kWaves) * 64 + lane) * 8, v[i]);
        }
    }
    // f(value, index) for the values of the row, or of its list.
    template <bool LIST, class F>
    __device__ __forceinline__ void each(F f) const
    {
        if constexpr (LIST) {
            for (int i = threadIdx.x; i < sh.count; i += THREADS) f(value_of(sh.list_key[i]), sh.list_at[i]);
        } else {
            each_segment([&](int, int at, const float(&v)[8]) {
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (at + c < V) f(v[c], at + c);
            });
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

    // The first of bins[0 .. n) at whose end base + the running sum reaches `target` (that of all, where it is never reached); the sum before it
    // in `before` (base included), its own in `amount`.  All of the block call it; some bin is not 0.
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
        uint64_t at = base + incl - mine, all = base;
        for (int w = 0; w < kWaves; ++w) {
            if (w < (int)(threadIdx.x >> 6)) at += sh.waves[w];
            all += sh.waves[w];
        }
        if (target > all) target = all;
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
    __device__ __forceinline__ void add(int bin, uint64_t amount) const { atomicAdd((unsigned long long*)&sh.bins[bin], (unsigned long long)amount); }

    // The largest key such that the amounts of the keys from it on reach `target` (they do over keys lo .. hi), with the sum above it and its own.
    template <bool LIST, class F>
    __device__ __forceinline__ unsigned int select(unsigned int lo, unsigned int hi, uint64_t target, F amount_of, uint64_t& above, uint64_t& amount) const
    {
        above = 0;
        while (true) {
            int s = 0;
            while ((hi - lo) >> s >= (unsigned int)kBins) ++s;
            clear_bins(kBins);
            each<LIST>([&](float v, int) {
                const unsigned int key = key_of(v);
                if (key >= lo && key <= hi) add((hi - key) >> s, amount_of(v));
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

    // What of the row, or of its list, stays.  lo and hi: the smallest and the largest key.
    template <bool LIST>
    __device__ __forceinline__ SampleKept keep(const SampleWeight& weight, unsigned int lo, unsigned int hi, int top_k, float top_p, float min_p, bool has_whole,
                                               uint64_t whole) const
    {
        SampleKept kept{lo, V, 0.0};
        uint64_t equal_kept = 0;  // how many of the smallest value that stays do, where not all do (0: all)
        if (top_k > 0 && top_k < V) {
            uint64_t above, amount;
            kept.key = select<LIST>(lo, hi, (uint64_t)top_k, [](float) { return (uint64_t)1; }, above, amount);
            if (above + amount > (uint64_t)top_k) equal_kept = (uint64_t)top_k - above;
        }
        if (top_p < 1.0f) {
            if (!has_whole) {
                whole = 0;
                each<LIST>([&](float v, int) {
                    const unsigned int key = key_of(v);
                    if (equal_kept ? key > kept.key : key >= kept.key) whole += weight.units(weight(v));
                });
                whole = block_sum(whole);
                if (equal_kept) whole += equal_kept * weight.units(weight(value_of(kept.key)));
            }
            const uint64_t target = nucleus_target(top_p, whole);  // a token stays where what is before it is less
            uint64_t above, amount;
            const unsigned int key = select<LIST>(kept.key, hi, target, [&](float v) { return weight.units(weight(v)); }, above, amount);
            const uint64_t one = weight.units(weight(value_of(key)));
            const uint64_t all = amount / one, wanted = (target - above + one - 1) / one;
            const uint64_t limit = key == kept.key && equal_kept ? equal_kept : all;
            kept.key = key;
            equal_kept = wanted < limit ? wanted : limit;
            if (equal_kept == all) equal_kept = 0;
        }
        if (min_p > 0.0f) {
            kept.least = fmin((double)min_p, 1.0);
            if (weight(value_of(kept.key)) < kept.least) equal_kept = 0;
        }
        // ---- the index of the last of the equal ones that stay: the segment first, then its place there ----
        if (equal_kept) {
            uint64_t before, amount;
            clear_bins((V + kSegment - 1) / kSegment);
            each<LIST>([&](float v, int at) {
                if (key_of(v) == kept.key) add(at / kSegment, 1);
            });
            const int segment = find_bin((V + kSegment - 1) / kSegment, 0, equal_kept, before, amount);
            clear_bins(kSegment);
            if constexpr (LIST) {
                each<true>([&](float v, int at) {
                    if (key_of(v) == kept.key && at / kSegment == segment) add(at % kSegment, 1);
                });
            } else {
                for (int i = threadIdx.x; i < kSegment; i += THREADS)
                    if (segment * kSegment + i < V && key_of((float)x[segment * kSegment + i]) == kept.key) add(i, 1);
            }
            kept.last = segment * kSegment + find_bin(kSegment, before, equal_kept, before, amount);
        }
        return kept;
    }
    static __device__ __forceinline__ bool stays(const SampleKept& kept, float v, int at, double w)
    {
        const unsigned int key = key_of(v);
        return (key > kept.key || (key == kept.key && at <= kept.last)) && w >= kept.least;
    }
};

template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a)
{
    typedef SampleRow<T, THREADS> Row;
    constexpr int kWaves = THREADS / 64;
    __shared__ typename Row::Shared sh;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_in_block(), V = a.V;
    const Row row{(const typename T::elem*)a.logits + r * a.ld, V, sh};
    const float temperature = a.temperatures ? a.temperatures[r] : a.temperature, top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float min_p = a.min_ps ? a.min_ps[r] : a.min_p, u = a.uniform[r];
    const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    auto answer = [&](int64_t token, float logp) {
        a.tokens[r] = token;
        a.logp[r] = logp;
    };
    const bool unfit = !(temperature >= 0.0f && temperature < __builtin_inff()) || top_p != top_p || min_p != min_p || u != u;
    const bool greedy = unfit || temperature == 0.0f || top_k == 1 || top_p <= 0.0f;  // (the first of the largest is all that stays)
    const bool cut_k = top_k > 0 && top_k < V, cut_p = top_p < 1.0f, cut_m = min_p > 0.0f;
    const bool sums = !greedy && !cut_k && (cut_p || !cut_m);
    const double rate = 1.4426950408889634 / (double)temperature;
    const int segments = (V + kSegment - 1) / kSegment;

    // ---- the largest value, the piece that has it first, and the sum of 2^(x rate) ----
    unsigned long long best = 0;
    float my_top = -__builtin_inff();
    bool bad = false;
    double my_sum = 0.0;
    if (tid == 0) sh.bad = sh.count = 0;
    __syncthreads();
    row.each_segment([&](int segment, int at, const float(&v)[8]) {
        float top = v[0];
#pragma unroll
        for (int c = 1; c < 8; ++c) top = fmaxf(top, v[c]);
#pragma unroll
        for (int c = 0; c < 8; ++c) bad |= !(v[c] < __builtin_inff());
        if (top > my_top || best == 0) {
            my_top = top;
            best = (unsigned long long)ordered_bits(top) << 32 | (unsigned int)~(unsigned int)at;
        }
        if (sums) {
            double e[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) e[c] = exp2_f64((double)v[c] * rate);
            const double sum = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            my_sum += sum;
            if (!cut_p) {
                double all = sum;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
                if (lane == 0) sh.segments[segment] = all;
            }
        }
    });
    const unsigned int my_key = best ? Row::key_of(my_top) : 0u;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned long long o = __shfl_xor(best, d);
        best = o > best ? o : best;
        my_sum += __shfl_xor(my_sum, d);
    }
    if (lane == 0) {
        sh.best[wave] = best;
        sh.waves_f[wave] = my_sum;
    }
    if (bad) sh.bad = 1;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < kWaves; ++w) {
        best = sh.best[w] > best ? sh.best[w] : best;
        sum += sh.waves_f[w];
    }
    const float top = from_ordered((unsigned int)(best >> 32));
    const unsigned int top_key = Row::key_of(top), bottom_key = Row::key_of(-__builtin_inff());
    if (sh.bad || unfit) {
        if (tid == 0) answer(-1, __builtin_nanf(""));
        return;
    }
    if (top == -__builtin_inff()) {
        if (tid == 0) answer(-1, -__builtin_inff());
        return;
    }
    if (greedy) {
        if (tid == 0) {
            const int at = (int)~(unsigned int)best;
            int c = 0;
            while (at + c < V - 1 && (float)row.x[at + c] != top) ++c;
            answer(at + c, 0.0f);
        }
        return;
    }
    const SampleWeight weight{(double)top, rate, ldexp(1.0, a.shift)};
    const double exponent = (double)top * rate;
    const bool summed = sums && fabs(exponent) <= kExponents;
    const double to_units = summed ? exp2_f64(-exponent) * weight.unit : 0.0;
    auto log_share = [&](float v, uint64_t whole) { return (float)(((double)v - weight.top) / (double)temperature - log((double)whole / weight.unit)); };

    uint64_t before, amount, whole;
    SampleKept kept{bottom_key, V, 0.0};
    int segment;
    if (summed && !cut_p) {
        // ---- all tokens stay: the segments' sums are there ----
        for (int i = tid; i < segments; i += THREADS) sh.bins[i] = (uint64_t)(sh.segments[i] * to_units);
        __syncthreads();
        whole = 0;
        for (int i = tid; i < segments; i += THREADS) whole += sh.bins[i];
        whole = row.block_sum(whole);
        segment = row.find_bin(segments, 0, sample_target(u, whole), before, amount);
    } else {
        // ---- the list of what may stay ----
        // Bounds are a little too low: what does not stay of the list is found below.
        float least = __builtin_inff();
        if (cut_k) {
            if (top_k <= THREADS) {
                // (over the threads' largest values as an order of 2048 steps from the smallest of them)
                unsigned int low = my_key ? my_key : 0xffffffffu;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) {
                    const unsigned int o = __shfl_xor(low, d);
                    low = o < low ? o : low;
                }
                row.clear_bins(Row::kBins);
                if (lane == 0) sh.waves[wave] = low;
                __syncthreads();
                for (int w = 0; w < kWaves; ++w) low = (unsigned int)sh.waves[w] < low ? (unsigned int)sh.waves[w] : low;
                __syncthreads();
                int s = 0;
                while ((top_key - low) >> s >= (unsigned int)Row::kBins) ++s;
                if (my_key) row.add((top_key - my_key) >> s, 1);
                const int bin = row.find_bin(Row::kBins, 0, (uint64_t)top_k, before, amount);
                // (fewer threads than top_k have values, all of them: no bound then)
                const unsigned int edge = before + amount < (uint64_t)top_k ? bottom_key : top_key - ((unsigned int)bin << s) - ((1u << s) - 1u);
                least = Row::value_of(edge > bottom_key ? edge : bottom_key);
                if (edge > top_key) least = -__builtin_inff();
            }
        } else if (cut_p ? summed : true) {
            // w >= share, that is x >= top + T log share; an fp32's rounding and more below that.
            const double share = cut_p ? (1.0 - (double)top_p) * sum * (to_units / weight.unit) / (double)V : fmin((double)min_p, 1.0);
            const double at = (double)top + log(share) * (double)temperature;
            least = (float)(at - (fabs(at) + fabs((double)top)) * 0x1p-20 - 0x1p-100);
        }
        const bool bounded = least < __builtin_inff();
        if (bounded) {
            row.each_segment([&](int, int at, const float(&v)[8]) {
                float most = v[0];
#pragma unroll
                for (int c = 1; c < 8; ++c) most = fmaxf(most, v[c]);
                if (most >= least) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (v[c] >= least && at + c < V) {
                            const int i = atomicAdd(&sh.count, 1);
                            if (i < kListMost) {
                                sh.list_key[i] = Row::key_of(v[c]);
                                sh.list_at[i] = at + c;
                            }
                        }
                }
            });
            __syncthreads();
        }
        const int count = bounded ? sh.count : kListMost + 1;
        const uint64_t row_whole = summed ? (uint64_t)(sum * to_units) : 0;
        if (count <= 64) {
            // ---- one wavefront, a lane each token ----
            if (wave != 0) return;
            const unsigned int key = lane < count ? sh.list_key[lane] : 0u;
            const int at = lane < count ? sh.list_at[lane] : 0x7fffffff;
            const unsigned long long order = (unsigned long long)key << 32 | (unsigned int)~(unsigned int)at;
            const float v = Row::value_of(key);
            const double w = lane < count ? weight(v) : 0.0;
            const uint64_t mine = weight.units(w);
            int rank = 0;         // tokens in front of this one
            uint64_t ahead = 0;   // and their weights
            for (int i = 0; i < count; ++i) {
                const unsigned long long o = __shfl(order, i);
                const uint64_t wi = __shfl(mine, i);
                if (o > order) {
                    ++rank;
                    ahead += wi;
                }
            }
            bool in = lane < count && !(cut_k && rank >= top_k);
            if (cut_p) {
                const uint64_t all = cut_k ? wave_sum_u64(in ? mine : 0) : row_whole;
                const uint64_t target = nucleus_target(top_p, all);
                in = in && (ahead < target || rank == 0);
            }
            if (cut_m) in = in && w >= fmin((double)min_p, 1.0);
            const uint64_t share = in ? mine : 0;
            whole = wave_sum_u64(share);
            const uint64_t target = sample_target(u, whole);
            uint64_t front = 0;  // the weights of what stays at smaller indices
            for (int i = 0; i < count; ++i) {
                const int oi = __shfl(at, i);
                const uint64_t wi = __shfl(share, i);
                if (oi < at) front += wi;
            }
            if (in && front < target && target <= front + share) answer(at, log_share(v, whole));
            return;
        }
        if (count <= kListMost) {
            unsigned int low = 0xffffffffu;
            for (int i = tid; i < count; i += THREADS) low = sh.list_key[i] < low ? sh.list_key[i] : low;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const unsigned int o = __shfl_xor(low, d);
                low = o < low ? o : low;
            }
            __syncthreads();
            if (lane == 0) sh.waves[wave] = low;
            __syncthreads();
            for (int w = 0; w < kWaves; ++w) low = (unsigned int)sh.waves[w] < low ? (unsigned int)sh.waves[w] : low;
            __syncthreads();
            kept = row.template keep<true>(weight, low, top_key, top_k, top_p, min_p, !cut_k && cut_p, row_whole);
            // ---- the draw: the segment, then the place in it ----
            row.clear_bins(segments);
            uint64_t part = 0;
            row.template each<true>([&](float v, int at) {
                const double w = weight(v);
                if (!Row::stays(kept, v, at, w)) return;
                row.add(at / kSegment, weight.units(w));
                part += weight.units(w);
            });
            whole = row.block_sum(part);
            const uint64_t target = sample_target(u, whole);
            segment = row.find_bin(segments, 0, target, before, amount);
            row.clear_bins(kSegment);
            row.template each<true>([&](float v, int at) {
                if (at / kSegment != segment) return;
                const double w = weight(v);
                if (Row::stays(kept, v, at, w)) row.add(at % kSegment, weight.units(w));
            });
            const int place = row.find_bin(kSegment, before, target, before, amount);
            if (tid == 0) answer(segment * kSegment + place, log_share((float)row.x[segment * kSegment + place], whole));
            return;
        }
        // ---- the row in place of the list ----
        if (cut_k || cut_p || cut_m) kept = row.template keep<false>(weight, bottom_key, top_key, top_k, top_p, min_p, summed && cut_p, row_whole);
        __syncthreads();
        row.each_segment([&](int segment, int at, const float(&v)[8]) {
            uint64_t part = 0;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const double w = weight(v[c]);
                if (at + c < V && Row::stays(kept, v[c], at + c, w)) part += weight.units(w);
            }
            part = wave_sum_u64(part);
            if (lane == 0) sh.bins[segment] = part;
        });
        __syncthreads();
        whole = 0;
        for (int i = tid; i < segments; i += THREADS) whole += sh.bins[i];
        whole = row.block_sum(whole);
        segment = row.find_bin(segments, 0, sample_target(u, whole), before, amount);
    }
    // ---- the draw in its segment ----
    if (wave == 0) {
        const int at = (segment * 64 + lane) * 8;
        float v[8];
        uint64_t w[8], part = 0;
        row.piece(at < V ? at / 8 : (V - 1) / 8, v);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const double e = weight(v[c]);
            w[c] = at + c < V && Row::stays(kept, v[c], at + c, e) ? weight.units(e) : 0;
            part += w[c];
        }
        uint64_t incl = part;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        // (the first pass's sum of a segment may be some units more than its tokens': its last token is drawn then)
        const uint64_t all = __shfl(incl, 63), wanted = sample_target(u, whole) - before, target = wanted < all ? wanted : all;
        uint64_t front = incl - part;
        if (front < target && target <= incl) {
            bool found = false;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (!found && front + w[c] >= target) {
                    found = true;
                    answer(at + c, log_share(v[c], whole));
                }
                front += w[c];
            }
        }
    }
}
}  // namespace pimhip
