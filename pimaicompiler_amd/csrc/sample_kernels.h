// A token drawn from each row of logits.
//
//   w_i = exp((x_i - max x) / T);  of the tokens in falling order of x (equal ones by their index): the first top_k; of them those before which
//   less than top_p of their sum has been reached; of them those with w >= min_p.  The token is the first in the order of indices at which
//   the running sum over what stayed exceeds u times the whole.
//
// One block a row.  The first pass (few long rows: a launch of its own, by all CUs) finds the largest value and, where the sum over all tokens is asked
// for, that too.  What may stay is
// above a bound that this pass gives (top_k: the k-th largest of the threads' own largest values; top_p: tokens below (1 - top_p) / V of the sum
// cannot be among those that reach top_p of it, since all of them together do not have the rest; min_p: its own), and goes to a list
// in LDS, whose order is worked out there: up to 64 tokens by one wavefront, more of them by buckets.
// Where it does not fit (flat distributions, a large top_k), nothing is put into order: top_k and top_p each come down to one value, the smallest that
// stays, and how many of those equal to it do.  It is found by histograms over the values' order (counts, or sums of w): the bucket in which the
// target is reached is cut into buckets again until it is one value.  16-bit rows of a call that asks for top_p, or a large top_k, are counted value by value
// instead, all 65536 of them in LDS: the one pass that does so stands for the first, and w is worked out once for each value.
// Sums that are made in any order are whole numbers of 64 bits, w in units of 2^-shift of the largest.  w itself is worked out in 64 bits (an fma of
// 64 bits takes a wavefront 5.4 clocks, one of 32 bits 4.4): with fp32's 2^-24 a number between two tokens of a large vocabulary would fall
// on the wrong one in some percent of the rows.
// Bound by w: 25 vector instructions a token, 13 us for the 64000 tokens a CU has of 512 rows of 32000 (fp32, nothing cut off: 27 us in all; the
// bytes take 10).  256 rows of 131072 in bfloat16 whose nucleus holds half of them: 73 us, the counts 20 (LDS atomics), the last pass's w 33.  Reading
// w out of a table in LDS there takes as long as working it out (30 us for 131072 gathers a CU).  64 rows of 100003 with settings of their own: 29;
// one row of 32000 with top_k and top_p: 13.6, of 131072 with top_k 18.5, code that is run once and the dependent steps.
// Code is kept short, loops as loops: what one row takes is walked through once and comes cold out of the instruction cache.  (The same steps
// unrolled, 117 to 177 KB a kernel, took 17 us for one row of 32000 and 69 for 256 of 131072.)
#pragma once

#include <type_traits>

#include "row_pieces.h"

namespace pimhip
{
static constexpr int kSampleMost = 1 << 21;   // tokens of a vocabulary
static constexpr int kSegment = 2048;         // tokens that a wavefront takes at a time, whose sum is kept
static constexpr int kListMost = 1024;        // tokens of a row's list
static constexpr int kBins = 2048;            // buckets
static constexpr int kTopsMost = 1 << 17;     // tokens of a row whose pieces' largest values are kept in LDS
static constexpr int kCountWords = 32768;     // a count of 16 bits for each 16-bit value, two a word
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
    // What sample_parts_kernel leaves of each row, or null:
    unsigned long long* part_best;  // [rows, segments]: the largest value of each, and the complement of its piece's index; all ones: one that has no distribution
    double* part_sums;              // [rows, segments]: where the row's first pass has sums
    unsigned short* part_tops;      // [rows, ld_tops]: the upper half of each piece's largest value, in its order
    int64_t ld_tops;
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

// log2 of m >= 1: the hardware's in 32 bits, off by some 1e-7, and what is left of m there.
__device__ __forceinline__ double log2_f64(double m)
{
    const double y = (double)__builtin_amdgcn_logf((float)m);
    return y + (m * exp2_f64(-y) - 1.0) * 1.4426950408889634;
}

// What is asked of a row.
struct SampleAsked {
    float temperature, top_p, min_p, u;
    int top_k;
    bool unfit, greedy, cut_k, cut_p, cut_m, sums;  // greedy: the first of the largest is all that stays; sums: the first pass makes them
    double rate;                                    // log2(e) / T
    __device__ __forceinline__ SampleAsked(const SampleArgs& a, int64_t r)
    {
        temperature = a.temperatures ? a.temperatures[r] : a.temperature;
        top_p = a.top_ps ? a.top_ps[r] : a.top_p;
        min_p = a.min_ps ? a.min_ps[r] : a.min_p;
        u = a.uniform[r];
        top_k = a.top_ks ? a.top_ks[r] : a.top_k;
        unfit = !(temperature >= 0.0f && temperature < __builtin_inff()) || top_p != top_p || min_p != min_p || u != u;
        u = fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f);  // (the nearest in [0, 1))
        greedy = unfit || temperature == 0.0f || top_k == 1 || top_p <= 0.0f;
        cut_k = top_k > 0 && top_k < a.V;
        cut_p = top_p < 1.0f;
        cut_m = min_p > 0.0f;
        sums = !greedy && !cut_k && (cut_p || !cut_m);
        rate = 1.4426950408889634 / (double)temperature;
    }
};

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

// A share of the whole, as whole numbers.  The first pass's sums and those relative to the largest value differ by up to 4.3e-12 of themselves, so shares
// are moved by 2^-36 of theirs: one that meets a border exactly (equal weights) is on the border's right side whichever it is compared with.
// The draw falls on the token at which the running sum reaches sample_target(); what reaches nucleus_target() takes no more tokens.
static constexpr double kBorder = 0x1p-36;
__device__ __forceinline__ uint64_t sample_target(float u, uint64_t whole)
{
    const uint64_t t = (uint64_t)((double)u * (1.0 + kBorder) * (double)whole);
    return (t < whole ? t : whole - 1) + 1;
}
__device__ __forceinline__ uint64_t nucleus_target(float top_p, uint64_t whole)
{
    const uint64_t t = (uint64_t)((double)top_p * (1.0 - kBorder) * (double)whole);
    return t < 1 ? 1 : t;
}

// The thread's number, asked for anew: what is made of it is made where it is used, not at the kernel's start and kept in registers (24 to 53 of them spilled
// so, 25 to 87 MB written by a call; now 0 to 14, 10 MB for 512 rows of 32000, 30.4 us then and 27 now, and 19 for 2000 of 8000).
__device__ __forceinline__ int this_thread()
{
    int t = (int)threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// Eight values as they lie in memory.
template <class T>
struct Piece {
    static constexpr int kQuads = sizeof(typename T::elem) / 2;
    uint4_t q[kQuads];
    __device__ __forceinline__ void load(const typename T::elem* p)
    {
#pragma unroll
        for (int i = 0; i < kQuads; ++i) q[i] = reinterpret_cast<const uint4_any_t*>(p)[i];
    }
    __device__ __forceinline__ float value(int c) const
    {
        typename T::elem e[8];
        __builtin_memcpy(e, q, sizeof(e));
        return (float)e[c];
    }
    __device__ __forceinline__ void set(int c, float v)
    {
        typename T::elem e[8];
        __builtin_memcpy(e, q, sizeof(e));
        e[c] = (typename T::elem)v;
        __builtin_memcpy(q, e, sizeof(e));
    }
};

template <class T, int THREADS>
struct SampleTokens {
    typedef typename T::elem elem;
    static constexpr int kWaves = THREADS / 64, kAhead = sizeof(elem) == 2 ? 4 : 2;  // (pieces on their way)
    const elem* x;
    int V;

    // The piece of values 8 p .. 8 p + 7 and the index of its first; the row's last piece is the last eight values, those of the piece before it -inf.
    __device__ __forceinline__ int piece(int p, Piece<T>& v) const
    {
        const int at = p * 8 + 8 <= V || V < 8 ? p * 8 : V - 8;
        if (V >= 8) {
            v.load(x + at);
            if (at != p * 8)
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (at + c < p * 8) v.set(c, -__builtin_inff());
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) v.set(c, c < V ? (float)x[c] : -__builtin_inff());
        }
        return at;
    }
    // f(number of a piece, index of its first value, the piece) for the pieces of a lane, then after(segment) behind each segment of a wavefront (four
    // pieces of each lane), from the wavefront's first on, `step` from one to the next.
    template <class F, class G>
    __device__ __forceinline__ void each_segment(F f, G after, int from, int step) const
    {
        const int pieces = (V + 7) / 8, segments = (V + kSegment - 1) / kSegment, lane = this_thread() & 63;
#pragma unroll 1
        for (int segment = from; segment < segments; segment += step) {
            Piece<T> v[kAhead];
            const int p0 = segment * (kSegment / 8) + lane;
            auto load = [&](int i, int p) {
                if (p * 8 + 8 <= V) v[i].load(x + p * 8);
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) load(i, p0 + i * 64);
#pragma unroll 1
            for (int p = p0; p < p0 + 256; p += 64) {
                Piece<T> now = v[0];
#pragma unroll
                for (int i = 0; i < kAhead - 1; ++i) v[i] = v[i + 1];
                if (kAhead < 4 && p + kAhead * 64 < p0 + 256) load(kAhead - 1, p + kAhead * 64);
                if (p < pieces) {
                    int at = p * 8;
                    if (at + 8 > V) at = piece(p, now);
                    f(p, at, now);
                }
            }
            after(segment);
        }
    }
    template <class F, class G>
    __device__ __forceinline__ void each_segment(F f, G after) const
    {
        each_segment(f, after, wave_in_block(), kWaves);
    }
};

template <class T, int THREADS>
struct SampleRow : SampleTokens<T, THREADS> {
    typedef typename T::elem elem;
    typedef SampleTokens<T, THREADS> Tokens;
    using Tokens::kWaves;
    using Tokens::x;
    using Tokens::V;
    using Tokens::each_segment;
    static constexpr bool kUnitsKept = THREADS == 1024;
    // fp32 words of 16-bit values end in zeros (in their order, in zeros or ones): these bits tell no two of them apart.
    static constexpr int kDrop = __is_same(T, F16) ? 13 : __is_same(T, BF16) ? 16 : 0;
    struct Shared {
        unsigned long long list[kListMost];  // keys, and the complements of indices below them
        uint64_t waves[kWaves];
        unsigned long long best[kWaves];
        uint64_t chunk_sums[32], chunk_counts[32];
        uint64_t found_before, found_amount;
        int found, count, named, bad;
    };
    Shared& sh;
    uint64_t* bins;        // kBins of them, or one for each segment where those are more
    unsigned int* ties;    // one for each segment, or for each value of one; the counts, or the pieces' largest values, lie there too

    static __device__ __forceinline__ unsigned int key_of(float v) { return ordered_bits(v) >> kDrop; }
    static __device__ __forceinline__ float value_of(unsigned int key)
    {
        const unsigned int o = key << kDrop;  // (a negative value's dropped bits are ones)
        return from_ordered(o & 0x80000000u ? o : o | ((1u << kDrop) - 1u));
    }
    static __device__ __forceinline__ unsigned long long entry_of(unsigned int key, int at) { return (unsigned long long)key << 32 | (unsigned int)~(unsigned int)at; }
    static __device__ __forceinline__ float value_in(unsigned long long entry) { return value_of((unsigned int)(entry >> 32)); }
    static __device__ __forceinline__ int index_in(unsigned long long entry) { return (int)~(unsigned int)entry; }

    __device__ __forceinline__ SampleRow(const elem* row, int tokens, Shared& shared, uint64_t* bins_at, unsigned int* ties_at)
        : Tokens{row, tokens}, sh(shared), bins(bins_at), ties(ties_at)
    {
    }

    // The sum of the threads' numbers in front of this one's, and of all.
    struct Scan {
        uint64_t before, all;
    };
    __device__ __forceinline__ Scan scan(uint64_t mine) const
    {
        const uint64_t incl = wave_scan_u64(mine);
        const int lane = this_thread() & 63, wave = wave_in_block();
        __syncthreads();
        if (lane == 63) sh.waves[wave] = incl;
        __syncthreads();
        const uint64_t waves = wave_scan_u64(lane < kWaves ? sh.waves[lane] : 0);
        return Scan{incl - mine + (wave ? readlane_u64(waves, wave - 1) : 0), readlane_u64(waves, 63)};
    }
    // The largest of the threads' numbers.
    __device__ __forceinline__ unsigned long long largest(unsigned long long mine) const
    {
        const int lane = this_thread() & 63;
        mine = wave_max_u64(mine);
        __syncthreads();
        if (lane == 0) sh.best[wave_in_block()] = mine;
        __syncthreads();
        return wave_max_u64(lane < kWaves ? sh.best[lane] : 0ull);
    }

    // The first of a[0 .. n) at whose end base + the running sum reaches `target` (that of all, where it is never reached); the sum before it
    // in `before` (base included), its own in `amount`.  All of the block call it; where all numbers are 0 nothing is found,
    // and it returns what was found before.
    template <class A>
    __device__ __forceinline__ int find(const A* a, int n, uint64_t base, uint64_t target, uint64_t& before, uint64_t& amount) const
    {
        __syncthreads();
        const int tid = this_thread(), per = (n + THREADS - 1) / THREADS, lo = tid * per < n ? tid * per : n, hi = lo + per < n ? lo + per : n;
        uint64_t mine = 0;
#pragma unroll 1
        for (int i = lo; i < hi; ++i) mine += a[i];
        const Scan s = scan(mine);
        uint64_t at = base + s.before;
        if (target > base + s.all) target = base + s.all;
        if (at < target && target <= at + mine) {
            int i = lo;
#pragma unroll 1
            while (i < hi - 1 && at + a[i] < target) at += a[i++];
            sh.found = i;
            sh.found_before = at;
            sh.found_amount = a[i];
        }
        __syncthreads();
        before = sh.found_before;
        amount = sh.found_amount;
        return sh.found;
    }

    __device__ __forceinline__ void clear_bins() const
    {
        __syncthreads();
#pragma unroll 1
        for (int i = this_thread(); i < kBins; i += THREADS) bins[i] = 0;
        __syncthreads();
    }
    __device__ __forceinline__ void add(int bin, uint64_t amount) const { atomicAdd((unsigned long long*)&bins[bin], (unsigned long long)amount); }

    // The largest key such that the amounts (weights in units, or ones) of the keys from it on reach `target` (they do over keys lo .. hi), with the
    // sum above it and its own.
    __device__ __forceinline__ unsigned int select(unsigned int lo, unsigned int hi, uint64_t target, const SampleWeight& weight, bool by_weight, uint64_t& above,
                                                   uint64_t& amount) const
    {
        above = 0;
        const unsigned int top = hi;
        while (true) {
            int s = 0;
            while ((hi - lo) >> s >= (unsigned int)kBins) ++s;
            clear_bins();
            // (most values are in the first range, few in a bucket of it)
            const float from = value_of(lo), to = value_of(hi);
            each_segment([&](int, int at, const Piece<T>& v) {
                const int begin = at % 8 ? 8 - V % 8 : 0;  // (the last piece's first values are not its own)
                if (above == 0 && hi == top) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float one = v.value(c);
                        const uint64_t amount_of = by_weight ? weight.units(weight(one)) : 1;
                        if (one >= from && c >= begin) add((hi - key_of(one)) >> s, amount_of);
                    }
                    return;
                }
                unsigned int hits = 0;
#pragma unroll
                for (int c = 0; c < 8; ++c) hits |= v.value(c) >= from && v.value(c) <= to ? 1u << c : 0u;
                hits &= 0xffu << begin;
#pragma unroll 1
                while (hits) {
                    const float one = (float)x[at + __builtin_ctz(hits)];
                    hits &= hits - 1;
                    add((hi - key_of(one)) >> s, by_weight ? weight.units(weight(one)) : 1);
                }
            }, [](int) {});
            uint64_t before;
            const int bin = find(bins, kBins, above, target, before, amount);
            above = before;
            hi -= (unsigned int)bin << s;
            if (s == 0) return hi;
            const unsigned int down = (1u << s) - 1u;
            lo = hi - lo > down ? hi - down : lo;
        }
    }

    // ---- counts of 16-bit values ----
    // A value's place in the order of all, -0 with 0.
    static __device__ __forceinline__ unsigned int place_of(unsigned int u)
    {
        u = u == 0x8000u ? 0u : u;
        return u & 0x8000u ? ~u & 0xffffu : u | 0x8000u;
    }
    static __device__ __forceinline__ float value_at(unsigned int place)
    {
        const unsigned short u = (unsigned short)(place & 0x8000u ? place & 0x7fffu : ~place);
        elem e;
        __builtin_memcpy(&e, &u, 2);
        return (float)e;
    }
    __device__ __forceinline__ unsigned int count_at(unsigned int place) const { return ties[place >> 1] >> (place & 1u ? 16 : 0) & 0xffffu; }
    __device__ __forceinline__ void count_all() const
    {
        const uint4_t zero = {0, 0, 0, 0};
#pragma unroll 1
        for (int i = this_thread(); i < kCountWords / 4; i += THREADS) reinterpret_cast<uint4_t*>(ties)[i] = zero;
        __syncthreads();
        auto count = [&](unsigned int u) {
            const unsigned int place = place_of(u);
            atomicAdd(&ties[place >> 1], place & 1u ? 65536u : 1u);
        };
        each_segment([&](int, int at, const Piece<T>& v) {
            const int from = at % 8 ? 8 - V % 8 : 0;  // (the last piece's first values are not its own)
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c >= from) count(v.q[0][c / 2] >> c % 2 * 16 & 0xffffu);
        }, [](int) {});
        __syncthreads();
    }
    // The highest place such that the amounts (weights in units, or ones) of the places from it on reach `target`, with the sum above it and its
    // own; sums: those of chunks of 2048 places.
    __device__ __forceinline__ unsigned int select_counted(const uint64_t* sums, uint64_t target, const SampleWeight& weight, bool by_weight, uint64_t& above,
                                                           uint64_t& amount) const
    {
        const int lane = this_thread() & 63;
        const uint64_t mine = lane < 32 ? sums[31 - lane] : 0, incl = wave_scan_u64(mine), all = readlane_u64(incl, 63);
        if (target > all) target = all;
        const int at = __builtin_ctzll(__ballot(incl >= target)), chunk = 31 - at;  // (lane 31 has reached it)
        above = readlane_u64(incl - mine, at);
        __syncthreads();
#pragma unroll 1
        for (int i = this_thread(); i < kBins; i += THREADS) {
            const unsigned int place = (unsigned int)(chunk * 2048 + 2047 - i), n = count_at(place);
            bins[i] = n == 0 ? 0 : by_weight ? n * weight.units(weight(value_at(place))) : n;
        }
        const int bin = find(bins, kBins, above, target, above, amount);
        return (unsigned int)(chunk * 2048 + 2047 - bin);
    }
};

// The first pass over rows of which there are fewer than CUs, by all of them: a wavefront a segment.
template <class T>
__global__ __launch_bounds__(256) void sample_parts_kernel(SampleArgs a)
{
    const int64_t r = blockIdx.y;
    const int segments = (a.V + kSegment - 1) / kSegment, segment = (int)blockIdx.x * 4 + wave_in_block();
    const SampleTokens<T, 256> row{(const typename T::elem*)a.logits + r * a.ld, a.V};
    const SampleAsked asked(a, r);
    unsigned long long best = 0;
    bool bad = false;
    double sum = 0.0;
    row.each_segment(
        [&](int p, int at, const Piece<T>& v) {
            float top = v.value(0);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                top = fmaxf(top, v.value(c));
                bad |= !(v.value(c) < __builtin_inff());
            }
            const unsigned int o = ordered_bits(top);
            a.part_tops[r * a.ld_tops + p] = (unsigned short)(o >> 16);
            const unsigned long long entry = (unsigned long long)o << 32 | (unsigned int)~(unsigned int)at;
            best = entry > best ? entry : best;
            if (asked.sums) {
                double e[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) e[c] = exp2_f64((double)v.value(c) * asked.rate);
                sum += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            }
        },
        [&](int at) {
            best = __ballot(bad) ? ~0ull : wave_max_u64(best);
            if (asked.sums) sum = wave_total_f64(sum);
            if ((threadIdx.x & 63) != 0) return;
            a.part_best[r * segments + at] = best;
            if (asked.sums) a.part_sums[r * segments + at] = sum;
        },
        segment, segments);
}

// PARTS: sample_parts_kernel has made the first pass.
template <class T, int THREADS, bool COUNT, bool PARTS>
__global__ __launch_bounds__(THREADS, 4) void sample_kernel(SampleArgs a)
{
    typedef SampleRow<T, THREADS> Row;
    extern __shared__ __align__(16) char shared[];  // sample_shared_bytes()
    typename Row::Shared& sh = *reinterpret_cast<typename Row::Shared*>(shared);
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, V = a.V, segments = (V + kSegment - 1) / kSegment;
    uint64_t* const bins = reinterpret_cast<uint64_t*>(shared + sizeof(typename Row::Shared));
    const Row row((const typename T::elem*)a.logits + r * a.ld, V, sh, bins, reinterpret_cast<unsigned int*>(bins + (segments > kBins ? segments : kBins)));
    const SampleAsked asked(a, r);
    const float temperature = asked.temperature, top_p = asked.top_p, u = asked.u;
    const int top_k = asked.top_k;
    auto answer = [&](int64_t token, float logp) {
        a.tokens[r] = token;
        a.logp[r] = logp;
    };
    const bool unfit = asked.unfit, greedy = asked.greedy, cut_k = asked.cut_k, cut_p = asked.cut_p, cut_m = asked.cut_m, cut = cut_k || cut_p || cut_m;
    const double rate = asked.rate, unit = ldexp(1.0, a.shift), per_unit = ldexp(1.0, -a.shift), least_weight = cut_m ? fmin((double)asked.min_p, 1.0) : 0.0;
    const unsigned int bottom_key = Row::key_of(-__builtin_inff());
    SampleWeight weight{0.0, rate, unit};
    // What stays: values above `smallest`, and the first equal_kept of those equal to it (0: all), in the order of indices, up to `last`.
    float smallest = -__builtin_inff();
    uint64_t equal_kept = 0;
    int last = V;
    uint64_t row_whole = 0, whole = 0, before, amount;
    unsigned int top_key = 0;
    bool relative = false;           // a pass's weights are relative to the largest value
    double to_units = unit;          // and what they come to in units
    bool settled = false;            // what stays is known before any pass
    float least = __builtin_inff();  // what is to be listed: values from this on (inf: none)
    float bound = -__builtin_inff();  // nothing below this stays
    auto log_share = [&](float v) { return (float)((((double)v - weight.top) * rate - log2_f64((double)whole * per_unit)) * 0.6931471805599453); };

    // The pieces' largest values, as the upper halves of their keys, where they are looked at again.
    unsigned short* const tops = reinterpret_cast<unsigned short*>(row.ties);
    double* const sums_of = reinterpret_cast<double*>(bins);
    // f(piece, the upper half of its largest value) of what sample_parts_kernel has left, eight next to each other at a time.
    auto each_top = [&](auto f) {
        const int tid = this_thread(), pieces = (V + 7) / 8;
#pragma unroll 1
        for (int p = tid * 8; p < pieces; p += THREADS * 8) {
            const uint4_t q = *reinterpret_cast<const uint4_t*>(a.part_tops + r * a.ld_tops + p);
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (p + c < pieces) f(p + c, q[c / 2] >> c % 2 * 16 & 0xffffu);
        }
    };
    // Passes over the row: the first, one that sums what top_k leaves, the last one with the segments' sums of what stays.
    enum { kFirst, kSum, kLast };
    int phase = kFirst;
    // ---- 16-bit rows, value by value: what stays is settled, as long as no count passes its end.  Whether the row has an answer already (no distribution) ----
    bool counts = COUNT && !greedy && (cut_k ? top_k > kListMost / 2 : cut_p);
    auto count_row = [&]() -> bool {
        const int tid = this_thread();
        counts = false;
        static_assert(!COUNT || THREADS == 1024, "a chunk of places is a word for each thread");
        row.count_all();
        unsigned int high = 0, low = 0xffffu, n = 0;
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
            const unsigned int two = row.ties[i * 1024 + tid], place = (unsigned int)(i * 1024 + tid) * 2;
            n += (two & 0xffffu) + (two >> 16);
            if (two != 0) {
                high = place + (two >> 16 ? 1 : 0);
                low = low != 0xffffu ? low : place + (two & 0xffffu ? 0 : 1);
            }
        }
        const uint64_t counted = row.scan(n).all;
        high = (unsigned int)row.largest(high);
        low = 0xffffu - (unsigned int)row.largest(0xffffu - low);
        constexpr unsigned int kInf = __is_same(T, F16) ? 0x7c00u : 0x7f80u;
        if (counted == (uint64_t)V) {  // (else a count has passed 65535: the row is taken as others are)
            if (high >= (0x8000u | kInf) || low < (0x7fffu & ~kInf)) {
                if (tid == 0) answer(-1, __builtin_nanf(""));
                return true;
            }
            if (high == (0x7fffu & ~kInf)) {
                if (tid == 0) answer(-1, -__builtin_inff());
                return true;
            }
            weight.top = (double)Row::value_at(high);
            top_key = Row::key_of(Row::value_at(high));
            auto mass = [&](unsigned int place) { return weight.units(weight(Row::value_at(place))); };
            if (tid < 32) sh.chunk_sums[tid] = sh.chunk_counts[tid] = 0;
            __syncthreads();
#pragma unroll 1
            for (int i = (int)(high >> 11); i >= (int)(low >> 11); --i) {
                const unsigned int two = row.ties[i * 1024 + tid];
                if (!__ballot(two != 0)) continue;
                uint64_t part = 0;
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    const unsigned int count = h ? two >> 16 : two & 0xffffu;
                    if (count) part += count * mass((unsigned int)(i * 1024 + tid) * 2 + h);
                }
                part = wave_total_u64(part);
                const unsigned int some = wave_total_u32((two & 0xffffu) + (two >> 16));
                if (lane == 0) {
                    atomicAdd((unsigned long long*)&sh.chunk_sums[i], (unsigned long long)part);
                    atomicAdd((unsigned long long*)&sh.chunk_counts[i], (unsigned long long)some);
                }
            }
            __syncthreads();
            // First by counts (top_k), then by weights (top_p); behind each, what the places from the one found on have.
            unsigned int place = 0;
            uint64_t above, some = 0;
#pragma unroll 1
            for (int by_weight = 0; by_weight < 2; ++by_weight) {
                if (by_weight ? !cut_p : !cut_k) continue;
                if (by_weight && !cut_k) row_whole = wave_total_u64(lane < 32 ? sh.chunk_sums[lane] : 0);
                const uint64_t target = by_weight ? nucleus_target(top_p, row_whole) : (uint64_t)top_k;
                const unsigned int found = row.select_counted(by_weight ? sh.chunk_sums : sh.chunk_counts, target, weight, by_weight, above, amount);
                const uint64_t one = by_weight ? mass(found) : 1, all = amount / one, wanted = target > above ? (target - above + one - 1) / one : 1;
                const uint64_t limit = found == place && equal_kept ? equal_kept : all;
                equal_kept = wanted < limit ? wanted : limit;
                if (!by_weight) row_whole = equal_kept * mass(found);
                if (equal_kept == all) equal_kept = 0;
                place = found;
                uint64_t sum = tid < 32 && tid > (int)(place >> 11) ? sh.chunk_sums[tid] : 0;
                some = tid < 32 && tid > (int)(place >> 11) ? sh.chunk_counts[tid] : 0;
#pragma unroll 1
                for (unsigned int at = (place & ~2047u) + tid; at < (place | 2047u) + 1; at += THREADS) {
                    const unsigned int count = at >= place ? row.count_at(at) : 0;
                    some += count;
                    if (count && !by_weight && at > place) sum += count * mass(at);
                }
                some = row.scan(some).all;
                if (!by_weight) row_whole += row.scan(sum).all;
            }
            smallest = Row::value_at(place);
            const double exponent = weight.top * rate;
            relative = fabs(exponent) > kExponents;
            to_units = relative ? unit : exp2_f64(-exponent) * unit;
            settled = true;
            phase = kLast;
            if (some <= kListMost) least = smallest;
        }
        __syncthreads();
        return false;
    };
    if constexpr (COUNT && !PARTS) {
        if (counts && count_row()) return;
    }
    bool count_now = counts && cut_k;  // (PARTS: where the sum over all tokens is there already, a list is tried first)
    while (true) {
        if constexpr (COUNT && PARTS) {
            if (count_now && count_row()) return;
            count_now = false;
        }
        if (tid == 0) sh.bad = sh.count = sh.named = 0;
        __syncthreads();
        const bool first = phase == kFirst;
        if (!(settled && least < __builtin_inff())) {
            if (phase == kLast && weight(smallest) < least_weight) {
                // min_p comes down to a smallest value too: the lowest key of a weight that stays.
                unsigned int out = Row::key_of(smallest), in = top_key;
                while (in - out > 1) {
                    const unsigned int mid = out + (in - out) / 2;
                    (weight(Row::value_of(mid)) < least_weight ? out : in) = mid;
                }
                smallest = Row::value_of(in);
                equal_kept = 0;
            }
            // ---- a pass ----
            const int tid = this_thread(), lane = tid & 63;
            const bool sums = !first || asked.sums, given = PARTS && first, tops_kept = !greedy && cut && V <= kTopsMost;
            const bool strict = equal_kept != 0;
            // Values from `limit` on are summed: those above `smallest`, or from it on.  Exponents are those of x rate in the first pass and where that
            // keeps to 64 bits' range; else relative to the largest value, fp32's differences being exact for what is near it.
            const float limit = strict ? from_ordered(ordered_bits(smallest) + 1) : smallest, base = relative ? (float)weight.top : 0.0f;
            unsigned long long best = 0;
            float my_top = -__builtin_inff();
            bool bad = false;
            double sum = 0.0;
            unsigned int equal = 0, my_key = 0;
            if (given) {
                for (int i = tid; i < segments; i += THREADS) {
                    const unsigned long long one = a.part_best[r * segments + i];
                    bad |= one == ~0ull;
                    best = one > best ? one : best;
                    if (sums) sums_of[i] = a.part_sums[r * segments + i];
                }
                each_top([&](int, unsigned int top) { my_key = top > my_key ? top : my_key; });
                my_key = (unsigned int)((uint64_t)my_key << 16 >> Row::kDrop);  // (lower than its value's by what the upper half leaves out)
            } else row.each_segment(
                [&](int p, int at, const Piece<T>& v) {
                    if (first) {
                        float top = v.value(0);
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            top = fmaxf(top, v.value(c));
                            bad |= !(v.value(c) < __builtin_inff());
                        }
                        if (tops_kept) tops[p] = (unsigned short)(ordered_bits(top) >> 16);
                        if (top > my_top || best == 0) {
                            my_top = top;
                            best = (unsigned long long)ordered_bits(top) << 32 | (unsigned int)~(unsigned int)at;
                        }
                    }
                    if (sums) {
                        double e[8];
                        if (first) {
#pragma unroll
                            for (int c = 0; c < 8; ++c) e[c] = exp2_f64((double)v.value(c) * rate);
                        } else {
#pragma unroll
                            for (int c = 0; c < 8; ++c) e[c] = exp2_f64((double)(v.value(c) >= limit ? v.value(c) - base : -__builtin_inff()) * rate);
                        }
                        sum += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
                    }
                    if (strict)
#pragma unroll
                        for (int c = 0; c < 8; ++c) equal += v.value(c) == smallest ? 1 : 0;
                },
                [&](int segment) {
                    if (!sums) return;
                    sum = wave_total_f64(sum);
                    if (lane == 0) sums_of[segment] = sum;
                    if (strict) {
                        equal = wave_total_u32(equal);
                        if (lane == 0) row.ties[segment] = equal;
                    }
                    sum = 0.0;
                    equal = 0;
                });
            __syncthreads();
            if (first) {
                if (!given) my_key = best ? Row::key_of(my_top) : 0u;
                if (bad) sh.bad = 1;
                best = row.largest(best);
                const float top = from_ordered((unsigned int)(best >> 32));
                if (sh.bad || unfit || top == -__builtin_inff()) {
                    if (tid == 0) answer(-1, sh.bad || unfit ? __builtin_nanf("") : -__builtin_inff());
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
                top_key = Row::key_of(top);
                weight.top = (double)top;
                const double exponent = (double)top * rate;
                relative = fabs(exponent) > kExponents;
                const bool summed = sums && !relative;  // (else a pass relative to the largest value is next)
                to_units = relative ? unit : exp2_f64(-exponent) * unit;
                if (!cut) {
                    phase = kLast;
                    if (!summed) continue;
                } else if (sums && !summed) {
                    phase = kSum;
                }
                if (cut && phase == kFirst) {
                    // ---- the bound of what may stay: a little too low each, what does not stay of the list is found there ----
                    if (cut_k && top_k <= THREADS && top_k <= kListMost / 2) {
                        // (over the threads' largest values as an order of 2048 steps from the smallest of them)
                        const unsigned int low = ~(unsigned int)row.largest(my_key ? ~my_key : 0u);
                        row.clear_bins();
                        int s = 0;
                        while ((top_key - low) >> s >= (unsigned int)kBins) ++s;
                        if (my_key) row.add((top_key - my_key) >> s, 1);
                        const int bin = row.find(bins, kBins, 0, (uint64_t)top_k, before, amount);
                        // (fewer threads than top_k have values, all of them: no bound then)
                        const unsigned int edge = top_key - ((unsigned int)bin << s) - ((1u << s) - 1u);
                        least = before + amount < (uint64_t)top_k || edge > top_key || edge < bottom_key ? -__builtin_inff() : Row::value_of(edge);
                    } else if (cut_k && V <= kListMost) {
                        least = -__builtin_inff();
                    }
                }
            }
            if (sums) {
                // ---- the segments' sums as whole numbers, what is equal to the smallest value as far as it stays ----
                uint64_t part = 0;
                const uint64_t equal_units = strict ? weight.units(weight(smallest)) : 0;
                if (strict && phase == kLast) {
                    const int edge = row.find(row.ties, segments, 0, equal_kept, before, amount);
                    // (the index of the last that stays, a value each thread)
                    const uint64_t in_front = before;
                    for (int i = tid; i <= edge; i += THREADS) sums_of[i] += (double)((i < edge ? (uint64_t)row.ties[i] : equal_kept - in_front) * equal_units) / to_units;
                    __syncthreads();
                    for (int i = tid; i < kSegment; i += THREADS) row.ties[i] = edge * kSegment + i < V && (float)row.x[edge * kSegment + i] == smallest ? 1 : 0;
                    last = edge * kSegment + row.find(row.ties, kSegment, in_front, equal_kept, before, amount);
                }
                for (int i = tid; i < segments; i += THREADS) {
                    const uint64_t units = (uint64_t)(sums_of[i] * to_units + 0.5);
                    bins[i] = units;
                    part += units;
                }
                whole = row.scan(part).all;
                if (phase != kLast) row_whole = whole + (strict ? equal_kept * equal_units : 0);
            }
            if (phase == kLast) break;
            if (first && phase == kFirst && !cut_k && cut) {
                // w >= share, that is x >= top + T log share; an fp32's rounding and more below that.
                const double share = cut_p ? (1.0 - (double)top_p) * ((double)row_whole / unit) / (double)V : least_weight;
                const double at = weight.top + log(share) * (double)temperature;
                least = (float)(at - (fabs(at) + fabs(weight.top)) * 0x1p-20 - 0x1p-100);
            }
            if (first && phase == kSum) continue;
        }

        if (least < __builtin_inff()) {
            // ---- the list: from the pieces whose largest value reaches the bound, or from all ----
            const int tid = this_thread();
            auto take = [&](int at, const Piece<T>& v) {
                unsigned int hits = 0;
#pragma unroll
                for (int c = 0; c < 8; ++c) hits |= v.value(c) >= least ? 1u << c : 0u;
                if (V < 8) hits &= (1u << V) - 1u;
                if (at % 8) hits &= 0xffu << (8 - V % 8);  // (the last piece's first values are not its own)
#pragma unroll 1
                while (hits) {
                    const int at_hit = at + __builtin_ctz(hits), i = atomicAdd(&sh.count, 1);
                    hits &= hits - 1;
                    if (i < kListMost) sh.list[i] = Row::entry_of(Row::key_of((float)row.x[at_hit]), at_hit);
                }
            };
            if (first && (PARTS || V <= kTopsMost)) {
                unsigned int* names = reinterpret_cast<unsigned int*>(bins);
                const unsigned int from = ordered_bits(least) >> 16;
                const int pieces = (V + 7) / 8;
                auto name = [&](int p, unsigned int top) {
                    if (top < from) return;
                    const int i = atomicAdd(&sh.named, 1);
                    if (i < kListMost) names[i] = (unsigned int)p;
                };
                __syncthreads();
                if (PARTS)
                    each_top(name);
                else
#pragma unroll 1
                    for (int p = tid; p < pieces; p += THREADS) name(p, tops[p]);
                __syncthreads();
                // (of more pieces than the list is long none is looked at: it would not hold what they have)
                const int named = sh.named;
                if (named > kListMost && tid == 0) sh.count = named;
                if (named <= kListMost)
#pragma unroll 1
                    for (int i = tid; i < named; i += THREADS) {
                        Piece<T> v;
                        const int at = row.piece((int)names[i], v);
                        take(at, v);
                    }
            } else {
                row.each_segment([&](int, int at, const Piece<T>& v) { take(at, v); }, [](int) {});
            }
            __syncthreads();
            const int count = sh.count;
            bound = least;
            least = __builtin_inff();
            if (count <= 64) {
                // ---- one wavefront, a lane each token ----
                if (wave_in_block() != 0) return;
                const int lane = this_thread() & 63;
                const unsigned long long entry = lane < count ? sh.list[lane] : 0ull;
                const float v = Row::value_in(entry);
                const int at = Row::index_in(entry);
                const double w = lane < count ? weight(v) : 0.0;
                const uint64_t mine = weight.units(w);
                int rank = 0;         // tokens in front of this one
                uint64_t ahead = 0;   // and their weights
#pragma unroll 1
                for (int i = 0; i < count; ++i) {
                    const uint64_t wi = readlane_u64(mine, i);
                    if (readlane_u64(entry, i) > entry) {
                        ++rank;
                        ahead += wi;
                    }
                }
                bool in = lane < count && !(cut_k && rank >= top_k);
                const uint64_t all = !settled && cut_k ? wave_total_u64(in ? mine : 0) : row_whole;
                in = in && (!cut_p || ahead < nucleus_target(top_p, all) || rank == 0) && w >= least_weight;
                const uint64_t share = in ? mine : 0;
                whole = wave_total_u64(share);
                const uint64_t aim = sample_target(u, whole);
                ahead = 0;
#pragma unroll 1
                for (unsigned long long left = __ballot(in); left; left &= left - 1) {
                    const int i = __builtin_ctzll(left);
                    const uint64_t wi = readlane_u64(share, i);
                    if (__builtin_amdgcn_readlane(at, i) < at) ahead += wi;
                }
                if (in && ahead < aim && aim <= ahead + share) answer(at, log_share(v));
                return;
            }
            if (count <= kListMost) {
                // ---- buckets: by keys first, for the order; then by indices, for the draw ----
                constexpr int kEach = kListMost / THREADS, kPer = kBins / THREADS;
                unsigned int* const counts = row.ties;                               // [kBins + 1]
                unsigned short* const members = reinterpret_cast<unsigned short*>(counts + kBins + 2);  // [kListMost]: list entries, bucket by bucket
                // The tokens' weights: kept where a CU has one block, worked out again where LDS for them would cost blocks (4096 rows of 500: 87 us, with them 96.5; 2000 of 8000 34.5 and 43).
                uint64_t* const units = reinterpret_cast<uint64_t*>(members + kListMost);
                auto units_of = [&](int i) { return Row::kUnitsKept ? units[i] : weight.units(weight(Row::value_in(sh.list[i]))); };
                bool in[kEach];
                unsigned int low = 0xffffffffu;
                for (int i = tid; i < count; i += THREADS) low = (unsigned int)(sh.list[i] >> 32) < low ? (unsigned int)(sh.list[i] >> 32) : low;
                low = ~(unsigned int)row.largest(~low);
                uint64_t aim = 0;
#pragma unroll 1
                for (int by_index = 0; by_index < 2; ++by_index) {
                    const int tid = this_thread();
                    int s = 0;
                    const unsigned int range = by_index ? (unsigned int)V - 1 : top_key - low;
                    while (range >> s >= (unsigned int)kBins) ++s;
                    auto bucket = [&](unsigned long long entry) { return (by_index ? (unsigned int)Row::index_in(entry) : top_key - (unsigned int)(entry >> 32)) >> s; };
                    row.clear_bins();
                    for (int i = tid; i <= kBins; i += THREADS) counts[i] = 0;
                    __syncthreads();
                    unsigned int slot[kEach];
#pragma unroll
                    for (int q = 0; q < kEach; ++q) {
                        const int i = q * THREADS + tid;
                        if (!by_index) {
                            in[q] = i < count;
                            if (Row::kUnitsKept && in[q]) units[i] = weight.units(weight(Row::value_in(sh.list[i])));
                        }
                        if (in[q]) {
                            const unsigned int b = bucket(sh.list[i]);
                            slot[q] = atomicAdd(&counts[b], 1u);
                            row.add((int)b, units_of(i));
                        }
                    }
                    __syncthreads();
                    // Sums in front of each bucket.
                    uint64_t mine = 0, some = 0;
#pragma unroll
                    for (int q = 0; q < kPer; ++q) {
                        mine += bins[tid * kPer + q];
                        some += counts[tid * kPer + q];
                    }
                    const typename Row::Scan masses = row.scan(mine), numbers = row.scan(some);
                    mine = masses.before, some = numbers.before;
#pragma unroll
                    for (int q = 0; q < kPer; ++q) {
                        const uint64_t m = bins[tid * kPer + q];
                        const unsigned int c = counts[tid * kPer + q];
                        bins[tid * kPer + q] = mine;
                        counts[tid * kPer + q] = (unsigned int)some;
                        mine += m;
                        some += c;
                    }
                    if (tid == 0) counts[kBins] = (unsigned int)numbers.all;
                    __syncthreads();
#pragma unroll
                    for (int q = 0; q < kEach; ++q)
                        if (in[q]) members[counts[bucket(sh.list[q * THREADS + tid])] + slot[q]] = (unsigned short)(q * THREADS + tid);
                    __syncthreads();
                    // Each token's place in the order: what is in front of its bucket, and of its bucket what goes before it.
                    uint64_t kept_sum = 0, ahead[kEach];
                    int rank[kEach];
#pragma unroll
                    for (int q = 0; q < kEach; ++q) {
                        ahead[q] = 0, rank[q] = 0;
                        if (!in[q]) continue;
                        const unsigned long long entry = sh.list[q * THREADS + tid];
                        const unsigned int b = bucket(entry);
                        ahead[q] = bins[b];
                        rank[q] = (int)counts[b];
#pragma unroll 1
                        for (unsigned int i = counts[b]; i < counts[b + 1]; ++i) {
                            const int member = members[i];
                            const unsigned long long o = sh.list[member];
                            if (by_index ? (unsigned int)o > (unsigned int)entry : o > entry) {  // (lower halves are the indices' complements)
                                ++rank[q];
                                ahead[q] += units_of(member);
                            }
                        }
                        if (!by_index && !(cut_k && rank[q] >= top_k)) kept_sum += units_of(q * THREADS + tid);
                    }
                    if (by_index) {
#pragma unroll
                        for (int q = 0; q < kEach; ++q) {
                            if (!in[q]) continue;
                            const unsigned long long entry = sh.list[q * THREADS + tid];
                            const float v = Row::value_in(entry);
                            if (ahead[q] < aim && aim <= ahead[q] + units_of(q * THREADS + tid)) answer(Row::index_in(entry), log_share(v));
                        }
                        return;
                    }
                    if (!settled && cut_k) row_whole = row.scan(kept_sum).all;
                    const uint64_t target = nucleus_target(top_p, row_whole);
                    uint64_t share = 0;
#pragma unroll
                    for (int q = 0; q < kEach; ++q) {
                        if (!in[q]) continue;
                        in[q] = !(cut_k && rank[q] >= top_k) && (!cut_p || ahead[q] < target || rank[q] == 0);
                        if (cut_m) in[q] = in[q] && weight(Row::value_in(sh.list[q * THREADS + tid])) >= least_weight;
                        if (in[q]) share += units_of(q * THREADS + tid);
                    }
                    whole = row.scan(share).all;
                    aim = sample_target(u, whole);
                }
            }
            // The list has no room: all of the block have read how many there are before the next pass begins to count.
            __syncthreads();
        }

        // ---- the row in place of the list: the smallest value that stays ----
        if (PARTS && counts) {
            count_now = true;
            continue;
        }
        const bool by_weight = !(first && cut_k);
        if (by_weight ? cut_p : true) {
            const uint64_t target = by_weight ? nucleus_target(top_p, row_whole) : (uint64_t)top_k;
            const unsigned int from = Row::key_of(smallest), lowest = bound > smallest ? Row::key_of(bound) : from;
            uint64_t above;
            const unsigned int key = row.select(lowest, top_key, target, weight, by_weight, above, amount);
            const uint64_t one = by_weight ? weight.units(weight(Row::value_of(key))) : 1, all = amount / one, wanted = target > above ? (target - above + one - 1) / one : 1;
            const uint64_t limit = key == from && equal_kept ? equal_kept : all;
            equal_kept = wanted < limit ? wanted : limit;
            if (equal_kept == all) equal_kept = 0;
            smallest = Row::value_of(key);
        }
        phase = !by_weight && cut_p ? kSum : kLast;
    }

    // ---- the draw: the segment, then the value in it, one each thread ----
    const uint64_t aim = sample_target(u, whole);
    const int segment = row.find(bins, segments, 0, aim, before, amount);
    // A segment's sum is rounded as one, its values one by one.  Where they come to less the last of them that has a unit is drawn.  Where each is below half a unit none
    // has any, and they are looked at again in 2^-40 of a unit (they are below 2^39 of these then, and one of them above 2^27: 2048 come to half a unit at
    // least), of which the target's place in the segment is as many for each unit.
    uint64_t in_front = before, target = aim;
    int in = -1;
#pragma unroll 1
    for (int pass = 0; pass < 2 && in < 0; ++pass) {
        __syncthreads();
#pragma unroll 1
        for (int i = this_thread(); i < kSegment; i += THREADS) {
            const int at = segment * kSegment + i;
            uint64_t units = 0;
            if (at < V) {
                const float v = (float)row.x[at];
                const double w = weight(v);
                if (v > smallest || (v == smallest && at <= last)) units = weight.units(w);
            }
            bins[i] = units;
        }
        if (tid == 0) sh.found = -1;
        in = row.find(bins, kSegment, in_front, target, before, amount);
        target = ((aim - in_front - 1) << 40) + 1;
        in_front = 0;
        weight.unit *= 0x1p40;
    }
    const int at = segment * kSegment + in;
    if (tid == 0) answer(at, log_share((float)row.x[at]));
}

// What a block needs of LDS.
template <class T, int THREADS, bool COUNT>
inline unsigned int sample_shared_bytes(int V)
{
    const int segments = (V + kSegment - 1) / kSegment, bins = segments > kBins ? segments : kBins;
    const int own = V <= kTopsMost ? segments * (kSegment / 16) : segments > kSegment ? segments : kSegment, buckets = kBins + 2 + kListMost / 2 + (SampleRow<T, THREADS>::kUnitsKept ? kListMost * 2 : 0);
    const int words = COUNT ? kCountWords : own > buckets ? own : buckets;
    return (unsigned int)(sizeof(typename SampleRow<T, THREADS>::Shared) + bins * sizeof(uint64_t) + words * sizeof(unsigned int));
}
}  // namespace pimhip
