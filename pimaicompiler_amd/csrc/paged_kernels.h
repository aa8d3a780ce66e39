// A cache of keys and values in pages on gfx950: appending to it with the position rotation on the way, and attention of each
// sequence's new token over it.
//
//   append    a pair (a, b) of a key's or query's first `rotary` values becomes (a c - b w, a w + b c), c and w the cosine and sine of
//             its token's position; the token at position p lies in place p % page_size of page table[sequence, p / page_size]
//   attend    o = sum_j e_j v_j / sum_j e_j,  e_j = exp(scale q . k_j - m),  j over the sequence's last `window` tokens
#pragma once

#include <type_traits>

#include "mx4_format.h"

namespace pimhip
{
struct PagedView {
    char* k;
    char* v;
    const float* k_scale;  // [kv_heads] or null: an 8-bit value times its head's scale is what it stands for
    const float* v_scale;
    int64_t k_page, k_head, v_page, v_head;  // bytes from one to the next
    int k_tok, v_tok;
    int pages, page_size, kv_heads, dim;
    const int* table;
    const int* lengths;
    int64_t ld_table;
    int sequences;
    int most;  // tokens a row of the table has room for
    unsigned int magic;  // ceil(2^shift / page_size), shift = 31 + ceil(log2 page_size): n / page_size is n magic / 2^shift for n < 2^31
    int shift;
    __device__ __forceinline__ int page_of(int token) const { return (int)(((uint64_t)(unsigned int)token * magic) >> shift); }
};

__device__ __forceinline__ int paged_length(const PagedView& a, int s)
{
    const int n = a.lengths[s];
    return n < 0 ? 0 : n < a.most ? n : a.most;
}

// ---- append ---------------------------------------------------------------------------------------

// Two fp32 values to 8 bits (E4M3), the nearest, ties to even, saturating at +-448; a NaN stays one.
__device__ __forceinline__ unsigned int to_e4m3x2(float a, float b)
{
    constexpr float most = 448.0f;
    a = a > most ? most : a < -most ? -most : a;
    b = b > most ? most : b < -most ? -most : b;
    return (unsigned int)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

struct AppendArgs {
    PagedView c;
    const int* starts;  // [sequences + 1] or null: token t is sequence t's
    const void* k;
    const void* v;
    const void* q;  // null: none
    void* q_out;    // [tokens, q_heads, dim]
    const float* angles;
    int64_t k_token, k_head, v_token, v_head, q_token, q_head;  // elements from one to the next
    int64_t ld_angles;
    int q_heads, half;  // half: pairs of a head that are turned
    int items;                  // groups of eight of a token
};

// A head of a token: those of keys come first, then those of values and of queries.
template <class E>
__device__ __forceinline__ const E* row_of(const AppendArgs& a, int t, int head)
{
    const int kv = a.c.kv_heads;
    return head < kv ? (const E*)a.k + t * a.k_token + head * a.k_head
           : head < 2 * kv ? (const E*)a.v + t * a.v_token + (head - kv) * a.v_head
                           : (const E*)a.q + t * a.q_token + (head - 2 * kv) * a.q_head;
}

// A block is heads of one token, a thread ITEMS groups of eight values of it, all asked for at once: of a key (query) the eight that a rotation turns
// them with beside them, out of the caches as a rule.  Values are asked for before the token's place is known, which takes three dependent loads: the
// sequence, its length, the page.  Bound by the bytes where tokens are many (8001 of 32 query and 8 key heads of 128 in bfloat16, neighbouring pairs of half of a
// head, 199 MB: 48 us, 4.1 TB/s where a copy has 4.8; into 8 bits 45), but by the angles and partners
// read beside them where more is turned (neighbouring pairs of all of a head 56 us; halves of half a head 66, of all of it 90, into 8 bits 89), else by those loads
// (one token: 4.2 us, a launch).
template <class T, bool FP8, bool INTERLEAVED, int ITEMS>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a)
{
    typedef typename T::elem elem;
    typedef typename T::frag frag;
    const int t = blockIdx.x, groups = a.c.dim / 8;
    const bool halves = !INTERLEAVED && a.half % 8 == 0;  // a group's partner is another group
    // ---- the values ----
    int head[ITEMS], d[ITEMS];  // heads of keys, then of values, then of queries; -1: none
    frag mine[ITEMS], other[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int item = ((int)blockIdx.y * ITEMS + i) * 256 + (int)threadIdx.x;
        head[i] = item < a.items ? item / groups : -1;
        d[i] = (item - head[i] * groups) * 8;
        if (head[i] < 0) continue;
        const elem* x = row_of<elem>(a, t, head[i]);
        mine[i] = load8_any<T>(x + d[i]);
        other[i] = frag{};
        if (halves && d[i] < 2 * a.half) other[i] = load8_any<T>(x + (d[i] < a.half ? d[i] + a.half : d[i] - a.half));
    }
    // ---- the token's place ----
    int s = t, end = t + 1;
    if (a.starts) {
        // The last of starts[0 .. sequences] that is not behind t, 64 candidates at a time.
        int lo = 0, span = a.c.sequences + 1;
        const int lane = threadIdx.x & 63;
        while (true) {
            const int step = (span + 63) / 64, i = lo + lane * step;
            const int n = __builtin_popcountll(__ballot(lane * step < span && a.starts[i < a.c.sequences ? i : a.c.sequences] <= t));
            if (n == 0) break;
            lo += (n - 1) * step;
            span = step < span - (n - 1) * step ? step : span - (n - 1) * step;
            if (step == 1) break;
        }
        s = lo;
        end = s < a.c.sequences ? a.starts[s + 1] : t;
        if (a.starts[s] > t || end <= t) s = a.c.sequences;
    }
    int64_t where = -1;
    if (s < a.c.sequences) where = (int64_t)a.c.lengths[s] - ((int64_t)end - t);
    const int pos = where >= 0 && where < a.c.most ? (int)where : -1;
    const int page = pos >= 0 ? a.c.table[s * a.c.ld_table + a.c.page_of(pos)] : -1, at = pos - a.c.page_of(pos) * a.c.page_size;
    const bool stored = page >= 0 && page < a.c.pages;
    const float* row = a.angles + pos * a.ld_angles;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const bool is_k = head[i] >= 0 && head[i] < a.c.kv_heads, is_q = head[i] >= 2 * a.c.kv_heads;
        if (head[i] < 0 || (!is_q && !stored)) continue;
        float y[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) y[c] = (float)mine[i][c];
        if ((is_k || is_q) && d[i] < 2 * a.half && pos >= 0) {
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int p = d[i] / 2 + c;
                    if (p < a.half) {
                        const float cosine = row[p], sine = row[a.half + p], u = y[2 * c], v = y[2 * c + 1];
                        y[2 * c] = u * cosine - v * sine;
                        y[2 * c + 1] = u * sine + v * cosine;
                    }
                }
            } else {
                // (a group may hold values of both halves, and values behind them, where a half is no multiple of eight)
                const elem* x = row_of<elem>(a, t, head[i]);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int e = d[i] + c;
                    if (halves || e < 2 * a.half) {
                        const bool first = e < a.half;
                        const int p = first ? e : e - a.half;
                        const float o = halves ? (float)other[i][c] : (float)x[first ? e + a.half : e - a.half];
                        const float cosine = row[p], sine = row[a.half + p];
                        y[c] = first ? y[c] * cosine - o * sine : o * sine + y[c] * cosine;
                    }
                }
            }
        }
        if (is_q) {
            if (pos < 0)  // a query of no sequence
#pragma unroll
                for (int c = 0; c < 8; ++c) y[c] = 0.0f;
            store8<T>((elem*)a.q_out + ((int64_t)t * a.q_heads + head[i] - 2 * a.c.kv_heads) * a.c.dim + d[i], float4_t{y[0], y[1], y[2], y[3]}, float4_t{y[4], y[5], y[6], y[7]});
            continue;
        }
        const int h = is_k ? head[i] : head[i] - a.c.kv_heads;
        char* out = is_k ? a.c.k + page * a.c.k_page + h * a.c.k_head + (int64_t)at * a.c.k_tok : a.c.v + page * a.c.v_page + h * a.c.v_head + (int64_t)at * a.c.v_tok;
        if constexpr (FP8) {
            const float scale = (is_k ? a.c.k_scale : a.c.v_scale)[h];
            unsigned int r[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) r[c] = to_e4m3x2(y[4 * c] / scale, y[4 * c + 1] / scale) | to_e4m3x2(y[4 * c + 2] / scale, y[4 * c + 3] / scale) << 16;
            typedef uint2_t bytes8_t __attribute__((aligned(1)));
            *reinterpret_cast<bytes8_t*>(out + d[i]) = uint2_t{r[0], r[1]};
        } else {
            store8<T>((elem*)out + d[i], float4_t{y[0], y[1], y[2], y[3]}, float4_t{y[4], y[5], y[6], y[7]});
        }
    }
}

// ---- attend ---------------------------------------------------------------------------------------
//
// The tokens of all sequences and key heads lie in a row of units of 64; each block takes an equal stretch of them, so that lengths may differ
// as they like (short sequences: a block takes a key head of one from end to end).  A piece of a (sequence, key head) that does not fill it goes to the workspace with its own maximum and sum, and a second
// kernel joins such pieces.  A wavefront takes 16 tokens of a unit at a time:
//   scores    K [16 tokens x dim] . Q^T [dim x 16 heads] on the 16-bit matrix instruction (8-bit keys become Q's type, exactly): a lane has
//             the scores of head l % 16 and tokens 4 (l / 16) + r
//   values    P [16 heads x 16 tokens] . V [16 tokens x 16 columns]: a lane's four e_j are its operand as they are, and V's is four tokens of a column that
//             16 lanes read as rows: nothing is exchanged.  Values of bfloat16 and of 8 bits, which bfloat16 has exactly, go through its matrix
//             instruction, with e_j in three pieces of it, which are all of its 24 bits; fp16 ones through the 32-bit one, four tokens at a time, e_j
//             as it is.  (The 32-bit one takes 2.7 times as long: 8-bit caches with 8 query heads a key head 159 us, in pieces 143; with 32, 16-bit
//             ones 319 and 299.)
// More than 16 query heads of up to 128 values go 32 at a time, so that keys and values are read once (24 heads: 278 us, 16 at a time some 530).  Fewer
// leave rows of the instructions empty (a form with the instruction of 16 blocks of 4 rows for up to 4 heads took 0 to 3 % longer).
// Values lie in registers from memory on, in loads that pass the caches (1.07 GB: 182 us, through them 208); a tile's are issued while the one
// before is worked on.  Registers are bounded for three wavefronts a SIMD (two with two tiles each on their way, or four: 1 to 3 % slower).
// Bound by the bytes: 537 MB of one sequence of 131071 tokens 93 us (5.8 TB/s), 1.07 GB of 64 sequences 177 (6.1), 1.64 GB in 8 bits 270 (6.1), where a kernel that
// only reads has 6.9.  From 16 query heads a key head on, products are as long as the loads (8-bit caches: 149 us with 16, 140 with 8, 136 with 4).
// Short calls take two launches and the dependent loads length, page, keys: 1000 tokens of one sequence 8 us.
static constexpr int kUnit = 64;           // tokens that the four wavefronts of a block take together
static constexpr float kLazy = 10.0f;      // a running maximum moves on when a score is above it by so many powers of two

struct AttendArgs {
    PagedView c;
    const void* q;
    void* out;
    float* lse;   // [sequences, heads] or null
    float* work;  // [blocks][2][heads at a time][dim + 4]: sums, then their maximum and weight
    int2* pieces; // [sequences * kv_heads * tiles_of_heads]: the first and the last block that worked on each
    int64_t q_seq, q_head;  // elements
    int group, tiles_of_heads, window;
    int whole;  // a block takes one (sequence, key head) from end to end, and nothing is joined
    float scale_log2;
};

// Four results of a head, and its sum's logarithm beside the first.
template <class T>
__device__ __forceinline__ void store_attended(const AttendArgs& a, int64_t head, int d, const float4_t sum, float weight, float top, float scale)
{
    const float f = weight == 0.0f ? 0.0f : scale / weight;
    store4<T>((typename T::elem*)a.out + head * a.c.dim + d, sum * f, 4);
    if (a.lse && d == 0) a.lse[head] = (top + __builtin_amdgcn_logf(weight)) * 0.6931471805599453f;
}

struct PagedSpan {
    int first, base, end, units;  // tokens first .. end - 1 are seen; tiles begin at base
};
__device__ __forceinline__ PagedSpan paged_span(int length, int window)
{
    PagedSpan p;
    p.end = length;
    p.first = window > 0 && p.end > window ? p.end - window : 0;
    p.base = p.first & ~15;
    const int n = (p.end - p.base + kUnit - 1) / kUnit;
    p.units = n < 1 ? 1 : n;  // (a sequence of no tokens has a result too)
    return p;
}

// Units up to which sequences are not cut, with `heads` (sequence, key head)s: each of these is then a block's from end to end.  Where the room that sequences
// have, or the window, says so (first), nothing is joined either; where lengths do, the launch that joins finds nothing.  In us, cut, whole and whole by
// lengths (8 key heads of 128, bfloat16): 1 sequence of 200 tokens 8.6, 5.7 and -, of 2000 10.1 and 14.9; 16 of 500 15.6, 13.3 and 16.3; 64 of 300 22.4, 15.2 and 18.5, of
// 1000 44.0, 38.1 and 41.4, of 4000 132 and 137; 256 of 500 83.8, 72.7 and 77.7, of 1 to 1000 114, 99 and 112.
__host__ __device__ constexpr int paged_whole_units(int64_t heads, bool first) { return first ? (heads >= 256 ? 16 : heads >= 64 ? 8 : 4) : heads >= 512 ? 16 : heads >= 256 ? 8 : 0; }

// The stretch of a block in the row of units (`times` units for each of a sequence's, less than 2^31 in all): units first .. end - 1 of `per` a
// block, and the sequence it begins in, which begins at unit `before` and is `length` tokens long.
struct PagedStretch {
    int first, end, per, s, before, length;
    bool whole;  // this and every grid's size-th (sequence, key head) behind it instead, as long as there are any
};
// The block's first (sequence, key head), as a stretch of its own.
__device__ __forceinline__ void paged_whole(const PagedView& c, int window, int times, int at, PagedStretch& f)
{
    f.whole = true;
    f.s = at / times;
    f.before = 0;
    f.first = f.end = 0;
    if (f.s >= c.sequences) return;
    f.length = paged_length(c, f.s);
    f.per = paged_span(f.length, window).units;
    f.first = (at - f.s * times) * f.per;
    f.end = f.first + f.per;
}
__device__ __forceinline__ PagedStretch paged_stretch(const PagedView& c, int window, int times, bool whole)
{
    PagedStretch f;
    if (whole) {
        paged_whole(c, window, times, (int)blockIdx.x, f);
        return f;
    }
    f.whole = false;
    const int most = paged_whole_units((int64_t)c.sequences * times, false);
    if (c.sequences == 1) {
        f.s = f.before = 0;
        f.length = paged_length(c, 0);
        const int units = paged_span(f.length, window).units, total = units * times;
        if (units <= most) {
            paged_whole(c, window, times, (int)blockIdx.x, f);
            return f;
        }
        f.per = (int)((unsigned int)(total + (int)gridDim.x - 1) / gridDim.x);
        f.first = (int)blockIdx.x * f.per;
        f.end = f.first + f.per < total ? f.first + f.per : total;
        return f;
    }
    __shared__ int wave_sum_of[4];
    __shared__ bool wave_long[4];
    __shared__ int found[3];
    const int each = (c.sequences + 255) / 256, from = (int)threadIdx.x * each, lo = from < c.sequences ? from : c.sequences;
    const int hi = lo + each < c.sequences ? lo + each : c.sequences;
    int mine = 0, length = 0;
    bool is_long = false;
    for (int s = lo; s < hi; ++s) {
        length = paged_length(c, s);
        const int units = paged_span(length, window).units;
        is_long |= units > most;
        mine += units * times;
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(incl, d);
        if ((int)(threadIdx.x & 63) >= d) incl += o;
    }
    const bool some_long = __ballot(is_long) != 0;
    if ((threadIdx.x & 63) == 63) {
        wave_sum_of[threadIdx.x >> 6] = incl;
        wave_long[threadIdx.x >> 6] = some_long;
    }
    __syncthreads();
    if (!(wave_long[0] || wave_long[1] || wave_long[2] || wave_long[3])) {
        paged_whole(c, window, times, (int)blockIdx.x, f);
        return f;
    }
    int before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < (int)(threadIdx.x >> 6)) before += wave_sum_of[w];
        total += wave_sum_of[w];
    }
    f.per = (int)(((unsigned int)total + gridDim.x - 1) / gridDim.x);
    // (a block behind the last stretch has none, and looks for nothing; blocks times per may pass 2^31)
    const int64_t first = (int64_t)blockIdx.x * f.per, end = first + f.per;
    f.first = first < total ? (int)first : total;
    f.end = end < total ? (int)end : total;
    if (before <= f.first && f.first < before + mine) {
        int s = lo;
        if (each > 1)
            for (; s < hi; ++s) {
                length = paged_length(c, s);
                const int n = paged_span(length, window).units * times;
                if (f.first < before + n) break;
                before += n;
            }
        found[0] = s;
        found[1] = before;
        found[2] = length;
    }
    __syncthreads();
    f.s = found[0];
    f.before = found[1];
    f.length = found[2];
    return f;
}

// Eight 8-bit values as eight of the 16-bit type, exactly.
template <class T>
__device__ __forceinline__ typename T::frag from_e4m3x8(uint2_t d);
template <>
__device__ __forceinline__ half8_t from_e4m3x8<F16>(uint2_t d)
{
    const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d[0], 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d[0], 1.0f, 1);
    const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d[1], 1.0f, 0), e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d[1], 1.0f, 1);
    return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}
template <>
__device__ __forceinline__ bf16x8_t from_e4m3x8<BF16>(uint2_t d)
{
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[0], 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[0], 1.0f, 1);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[1], 1.0f, 0), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[1], 1.0f, 1);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

// N (4 or 8) values next to each other as fp32.
template <class T, bool FP8, int N>
struct ValuePiece {
    static constexpr int kWords = N * (FP8 ? 1 : 2) / 4;
    unsigned int w[kWords];
    __device__ __forceinline__ void load(const char* p)
    {
        if constexpr (kWords == 1) {
            typedef unsigned int word_any_t __attribute__((aligned(1)));
            w[0] = load_global_once<word_any_t>(p);
        } else {
            typedef unsigned int words_t __attribute__((ext_vector_type(kWords)));
            typedef words_t words_any_t __attribute__((aligned(1)));
            const words_t q = load_global_once<words_any_t>(p);
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = q[i];
        }
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float value(int i) const
    {
        if constexpr (FP8) {
            const float2_t two = i % 4 < 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(w[i / 4], false) : __builtin_amdgcn_cvt_pk_f32_fp8(w[i / 4], true);
            return two[i % 2];
        } else if constexpr (__is_same(T, BF16)) {
            return __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        } else {
            return (float)__builtin_bit_cast(half2_t, w[i / 2])[i % 2];
        }
    }
    // Values 2 i and 2 i + 1 in bfloat16, where that has them exactly.
    __device__ __forceinline__ unsigned int pair(int i) const
    {
        if constexpr (FP8)
            return __builtin_bit_cast(unsigned int, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i / 2], 1.0f, 1) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i / 2], 1.0f, 0));
        else
            return w[i];
    }
};

// Wavefronts of a SIMD that the registers are bounded for.
constexpr int attend_waves(int nc, int ht) { return nc <= 2 && ht <= 16 ? 3 : 2; }

// NC: the head's size in 64 columns, rounded up; HT: query heads at a time (16 or 32); EVEN: pages are whole tiles of 16 tokens, and the head's size is NC of 64:
// a tile's place is then the same for the wavefront, and no lane stays without loads (8-bit caches: 138 us, as others 146; 16-bit ones 258 and 260).
template <class T, bool FP8, int NC, int HT, bool EVEN>
__global__ __launch_bounds__(256, attend_waves(NC, HT)) void paged_attend_kernel(AttendArgs a)
{
    typedef typename T::elem elem;
    typedef typename T::frag frag;
    constexpr int kSteps = NC * 2;                   // matrix instructions along a head's values
    constexpr int kLoads = FP8 ? NC : kSteps;        // 16-byte loads of a key's row by a lane
    constexpr int kWide = NC / 2, kNarrow = NC % 2;  // pieces of eight and of four columns of a lane
    constexpr int kCols = NC * 4, kSize = FP8 ? 1 : 2;
    constexpr int kScores = HT / 16;                 // tiles of 16 heads
    constexpr bool kThree = FP8 || __is_same(T, BF16);  // weights in three pieces of bfloat16
    __shared__ float wave_m[4][HT], wave_l[4][HT];
    __shared__ float parts[4][HT][NC * 64 + 4];
    const int lane = threadIdx.x & 63, wave = wave_in_block(), n = lane & 15, g = lane >> 4;
    const PagedView& c = a.c;
    const int D = c.dim;
    const int heads_of_units = c.kv_heads * a.tiles_of_heads;

    PagedStretch stretch = paged_stretch(c, a.window, heads_of_units, a.whole != 0);
    if (stretch.first >= stretch.end) return;
    int s = stretch.s, before = stretch.before, length = stretch.length, end = stretch.end, at = (int)blockIdx.x;
    for (int u = stretch.first; u < end;) {
        const PagedSpan span = paged_span(length, a.window);
        const int rel = u - before, hg = rel / span.units, first = rel - hg * span.units;
        const int left = span.units - first, take = left < end - u ? left : end - u, last = first + take;
        const int kvh = hg / a.tiles_of_heads, head0 = (hg - kvh * a.tiles_of_heads) * HT;

        // ---- queries ----
        frag q[kScores][kSteps];
#pragma unroll
        for (int mt = 0; mt < kScores; ++mt) {
            const int h = head0 + mt * 16 + n;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int d = FP8 ? i / 2 * 64 + g * 16 + i % 2 * 8 : i * 32 + g * 8;
                q[mt][i] = frag{};
                if (h < a.group && d < D) q[mt][i] = load8_any<T>((const elem*)a.q + s * a.q_seq + (kvh * a.group + h) * a.q_head + d);
            }
        }
        const float scale = a.scale_log2 * (FP8 ? c.k_scale[kvh] : 1.0f);
        const char* kh = c.k + kvh * c.k_head;
        const char* vh = c.v + kvh * c.v_head;
        const int* row = c.table + s * c.ld_table;

        float m[kScores], l[kScores];
        float4_t o[kScores][kCols];
#pragma unroll
        for (int mt = 0; mt < kScores; ++mt) {
            m[mt] = -__builtin_inff();
            l[mt] = 0.0f;
        }
#pragma unroll
        for (int mt = 0; mt < kScores; ++mt)
#pragma unroll
            for (int i = 0; i < kCols; ++i) o[mt][i] = float4_t{0, 0, 0, 0};

        // ---- tiles: 16 tokens of each unit ----
        uint4_t k[kLoads];
        ValuePiece<T, FP8, 8> wide[4][kWide ? kWide : 1];
        ValuePiece<T, FP8, 4> narrow[4][kNarrow ? kNarrow : 1];
        unsigned int page_ok = 0;  // a bit for each token of a tile
        // This wavefront's first token of a unit; a unit behind the stretch's end has none.
        auto token_of = [&](int unit) { return unit < last ? span.base + unit * kUnit + wave * 16 : span.end; };
        // Pages: a lane has that of one of the next 64 tiles (EVEN), or of a token of one of the next 4; the group after that is on its way.
        constexpr int kGroup = EVEN ? 64 : 4;
        auto pages_of = [&](int unit) {
            const int first_token = token_of(unit + (EVEN ? lane : g)), token = first_token + (EVEN ? 0 : n);
            return first_token < span.end && token < span.end ? row[c.page_of(token)] : -1;
        };
        int ids = pages_of(first), ids_next = pages_of(first + kGroup);
        // The loads of a unit's tile, in two parts: its place and keys, its values.  A page that is none is read as page 0, and not seen.
        int page = 0, in = 0;
        const unsigned int k_off = n * c.k_tok + g * 16, v_off = g * 4 * c.v_tok + n * (kWide ? 8 : 4) * kSize;
        auto load_keys = [&](int unit) {
            const int token = token_of(unit), i = (unit - first) & (kGroup - 1);
            if (i == 0 && unit != first) {
                ids = ids_next;
                ids_next = pages_of(unit + kGroup);
            }
            if constexpr (EVEN) {
                const int id = __builtin_amdgcn_readlane(ids, i);
                const bool ok = id >= 0 && id < c.pages;
                page_ok = ok ? 0xffffu : 0u;
                page = ok ? id : 0;
                in = token - c.page_of(token) * c.page_size;
                const char* kp = kh + page * c.k_page + in * c.k_tok;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) k[i] = load_global_once<uint4_any_t>(kp + k_off + i * 64);
            } else {
                const int id = __shfl(ids, i * 16 + n);
                const bool ok = id >= 0 && id < c.pages;
                page_ok = (unsigned int)__ballot(ok) & 0xffffu;
                page = ok ? id : 0;
                in = token + n - c.page_of(token + n) * c.page_size;
                const char* kp = kh + page * c.k_page + in * c.k_tok + g * 16;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    k[i] = uint4_t{0, 0, 0, 0};
                    if (i * 64 + g * 16 < D * kSize) k[i] = load_global_once<uint4_any_t>(kp + i * 64);
                }
            }
        };
        auto load_values = [&](int r) {
            if constexpr (EVEN) {
                const char* vp = vh + page * c.v_page + (in + r) * c.v_tok;
#pragma unroll
                for (int i = 0; i < kWide; ++i) wide[r][i].load(vp + v_off + i * 128 * kSize);
                if constexpr (kNarrow) narrow[r][0].load(vp + (kWide ? v_off - n * 4 * kSize + kWide * 128 * kSize : v_off));
            } else {
                const char* vp = vh + __shfl(page, g * 4 + r) * c.v_page + __shfl(in, g * 4 + r) * c.v_tok;
#pragma unroll
                for (int i = 0; i < kWide; ++i) {
                    wide[r][i].clear();
                    if (i * 128 + n * 8 < D) wide[r][i].load(vp + (i * 128 + n * 8) * kSize);
                }
                if constexpr (kNarrow) {
                    narrow[r][0].clear();
                    if (kWide * 128 + n * 4 < D) narrow[r][0].load(vp + (kWide * 128 + n * 4) * kSize);
                }
            }
        };
        if (token_of(first) < span.end) {
            load_keys(first);
#pragma unroll
            for (int r = 0; r < 4; ++r) load_values(r);
        }
        // A tile; `more`: the loads of the next one are issued as its registers become free.
        auto tile = [&](auto more, int unit) {
            constexpr bool kMore = decltype(more)::value;
            const int token = token_of(unit);
            // Tokens that are not the sequence's, or not in the window, or of no page, are left out, whatever lies there.
            unsigned int seen = page_ok;
            if (token < span.first) seen &= 0xffffu << (span.first - token);
            if (token + 16 > span.end) seen &= 0xffffu >> (token + 16 - span.end);

            float4_t sc[kScores];
#pragma unroll
            for (int mt = 0; mt < kScores; ++mt) sc[mt] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                frag kf;
                if constexpr (FP8)
                    kf = from_e4m3x8<T>(i % 2 ? uint2_t{k[i / 2][2], k[i / 2][3]} : uint2_t{k[i / 2][0], k[i / 2][1]});
                else
                    kf = __builtin_bit_cast(frag, k[i]);
#pragma unroll
                for (int mt = 0; mt < kScores; ++mt) sc[mt] = T::mfma(kf, q[mt][i], sc[mt]);
            }
            if constexpr (kMore) load_keys(unit + 1);
#pragma unroll
            for (int mt = 0; mt < kScores; ++mt) sc[mt] *= scale;
            if (seen != 0xffffu) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (seen >> (g * 4 + r) & 1) continue;
#pragma unroll
                    for (int mt = 0; mt < kScores; ++mt) sc[mt][r] = -__builtin_inff();
#pragma unroll
                    for (int i = 0; i < kWide; ++i) wide[r][i].clear();
                    if constexpr (kNarrow) narrow[r][0].clear();
                }
            }
            bool above = false;
#pragma unroll
            for (int mt = 0; mt < kScores; ++mt) above |= fmaxf(fmaxf(sc[mt][0], sc[mt][1]), fmaxf(sc[mt][2], sc[mt][3])) > m[mt] + kLazy;
            if (__ballot(above)) {
                float f[kScores];
#pragma unroll
                for (int mt = 0; mt < kScores; ++mt) {
                    float top = fmaxf(fmaxf(sc[mt][0], sc[mt][1]), fmaxf(sc[mt][2], sc[mt][3]));
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float now = fmaxf(m[mt], top);
                    f[mt] = m[mt] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m[mt] - now);
                    m[mt] = now;
                    l[mt] *= f[mt];
                }
#pragma unroll
                for (int mt = 0; mt < kScores; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float fr = __shfl(f[mt], g * 4 + r);
#pragma unroll
                        for (int i = 0; i < kCols; ++i) o[mt][i][r] *= fr;
                    }
            }
            float p[kScores][4];
#pragma unroll
            for (int mt = 0; mt < kScores; ++mt) {
                const float from = m[mt] == -__builtin_inff() ? 0.0f : m[mt];  // (scores are -inf all then)
#pragma unroll
                for (int r = 0; r < 4; ++r) p[mt][r] = __builtin_amdgcn_exp2f(sc[mt][r] - from);
                l[mt] += (p[mt][0] + p[mt][1]) + (p[mt][2] + p[mt][3]);
            }
            if constexpr (kThree) {
                typedef short short4v_t __attribute__((ext_vector_type(4)));
                auto operand = [](unsigned int w0, unsigned int w1) { return __builtin_bit_cast(short4v_t, uint2_t{w0, w1}); };
                auto halves = [](unsigned int w0, unsigned int w1, bool upper) { return __builtin_amdgcn_perm(w1, w0, upper ? 0x07060302u : 0x05040100u); };
                short4v_t part[3][kScores];
#pragma unroll
                for (int mt = 0; mt < kScores; ++mt)
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        unsigned int b[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            b[r] = __builtin_bit_cast(unsigned int, p[mt][r]);
                            // (what is left, 2^-126 at least: an infinite value times it stays one.  But nothing of a weight that is 0: its value has no part)
                            p[mt][r] = __builtin_amdgcn_fmed3f(p[mt][r] - __builtin_bit_cast(float, b[r] & 0xffff0000u), 0x1p-126f, p[mt][r]);
                        }
                        part[i][mt] = operand(halves(b[0], b[1], true), halves(b[2], b[3], true));
                    }
                // Columns i and i + 1 of a lane, of its four tokens.
                auto add = [&](int i, const unsigned int(&w)[4]) {
                    const short4v_t v[2] = {operand(halves(w[0], w[1], false), halves(w[2], w[3], false)), operand(halves(w[0], w[1], true), halves(w[2], w[3], true))};
#pragma unroll
                    for (int k = 0; k < 3; ++k)
#pragma unroll
                        for (int mt = 0; mt < kScores; ++mt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) o[mt][i + c] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(part[k][mt], v[c], o[mt][i + c], 0, 0, 0);
                };
#pragma unroll
                for (int i = 0; i < kWide; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) add(i * 8 + e * 2, {wide[0][i].pair(e), wide[1][i].pair(e), wide[2][i].pair(e), wide[3][i].pair(e)});
                if constexpr (kNarrow)
#pragma unroll
                    for (int e = 0; e < 2; ++e) add(kWide * 8 + e * 2, {narrow[0][0].pair(e), narrow[1][0].pair(e), narrow[2][0].pair(e), narrow[3][0].pair(e)});
                if constexpr (kMore) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) load_values(r);
                }
                return;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                auto add = [&](int i, float v) {
#pragma unroll
                    for (int mt = 0; mt < kScores; ++mt)
                        o[mt][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[mt][r], v, o[mt][i], 0, 0, 0);
                };
#pragma unroll
                for (int i = 0; i < kWide; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) add(i * 8 + e, wide[r][i].value(e));
                if constexpr (kNarrow)
#pragma unroll
                    for (int e = 0; e < 4; ++e) add(kWide * 8 + e, narrow[r][0].value(e));
                if constexpr (kMore) load_values(r);
            }
        };
        int unit = first;
        for (; token_of(unit + 1) < span.end; ++unit) tile(std::true_type{}, unit);
        if (token_of(unit) < span.end) tile(std::false_type{}, unit);

        // ---- the four wavefronts' parts, joined by all of the block ----
        const int rows = a.group - head0 < HT ? a.group - head0 : HT;
#pragma unroll
        for (int mt = 0; mt < kScores; ++mt) {
            l[mt] += __shfl_xor(l[mt], 16);
            l[mt] += __shfl_xor(l[mt], 32);
            if (g == 0) {
                wave_m[wave][mt * 16 + n] = m[mt];
                wave_l[wave][mt * 16 + n] = l[mt];
            }
        }
#pragma unroll
        for (int mt = 0; mt < kScores; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int h = mt * 16 + g * 4 + r;
                if (h >= rows) continue;
                float* part = parts[wave][h];
#pragma unroll
                for (int i = 0; i < kWide; ++i)
#pragma unroll
                    for (int e = 0; e < 8; e += 4)
                        *reinterpret_cast<float4_t*>(part + i * 128 + n * 8 + e) = float4_t{o[mt][i * 8 + e][r], o[mt][i * 8 + e + 1][r], o[mt][i * 8 + e + 2][r], o[mt][i * 8 + e + 3][r]};
                if constexpr (kNarrow)
                    *reinterpret_cast<float4_t*>(part + kWide * 128 + n * 4) =
                        float4_t{o[mt][kWide * 8][r], o[mt][kWide * 8 + 1][r], o[mt][kWide * 8 + 2][r], o[mt][kWide * 8 + 3][r]};
            }
        __syncthreads();
        const bool complete = first == 0 && last == span.units;
        const float vs = FP8 ? c.v_scale[kvh] : 1.0f;
        const int64_t out0 = (int64_t)s * c.kv_heads * a.group + kvh * a.group + head0;
        float* piece = a.work + ((int64_t)blockIdx.x * 2 + (first == 0 ? 1 : 0)) * HT * (D + 4);
        const int each = D / 4;
        for (int i = threadIdx.x; i < rows * each; i += 256) {
            const int h = i / each, d = (i - h * each) * 4;
            const float top = fmaxf(fmaxf(wave_m[0][h], wave_m[1][h]), fmaxf(wave_m[2][h], wave_m[3][h]));
            float4_t sum = {0, 0, 0, 0};
            float weight = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = wave_m[w][h] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(wave_m[w][h] - top);
                weight += f * wave_l[w][h];
                sum += f * *reinterpret_cast<const float4_t*>(&parts[w][h][d]);
            }
            if (complete) {
                store_attended<T>(a, out0 + h, d, sum, weight, top, vs);
            } else {
                *reinterpret_cast<float4_t*>(piece + h * (D + 4) + d) = sum;
                if (d == 0) *reinterpret_cast<float2_t*>(piece + h * (D + 4) + D) = float2_t{top, weight};
            }
        }
        if (threadIdx.x == 0 && last == span.units) a.pieces[(int64_t)s * heads_of_units + hg] = int2{stretch.whole ? (int)blockIdx.x : (u - first) / stretch.per, (int)blockIdx.x};
        __syncthreads();
        if (stretch.whole) {
            at += (int)gridDim.x;
            paged_whole(c, a.window, heads_of_units, at, stretch);
            s = stretch.s, length = stretch.length, u = stretch.first, end = stretch.end;
            continue;
        }
        u += take;
        if (rel + take == heads_of_units * span.units) {
            before += heads_of_units * span.units;
            if (++s < c.sequences) length = paged_length(c, s);
        }
    }
}

// The pieces of each (sequence, key head) that more than one block worked on, of a head by WAVES wavefronts, an equal share of the pieces each: by one (four heads
// a block), four or sixteen.  A wavefront asks for four pieces at a time, one that is alone for sixteen where there are more, a lane for four columns of each.
template <class T, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void paged_join_kernel(AttendArgs a, int rows)
{
    const PagedView& c = a.c;
    const int D = c.dim, heads = c.kv_heads * a.group, lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : wave_in_block(), d = lane * 4;
    const int at = WAVES == 1 ? (int)blockIdx.x * 4 + wave_in_block() : (int)blockIdx.x;
    if (WAVES == 1 && at >= c.sequences * heads) return;
    const int s = at / heads, h_all = at - s * heads, kvh = h_all / a.group, h_in = h_all - kvh * a.group, tile = h_in / rows, h = h_in - tile * rows;
    const int2 blocks = a.pieces[((int64_t)s * c.kv_heads + kvh) * a.tiles_of_heads + tile];
    if (blocks.x == blocks.y) return;
    // (a piece's place: the block's second where the sequence begins in it, else its first)
    auto part = [&](int b) { return a.work + (((int64_t)b * 2 + (b == blocks.x ? 1 : 0)) * rows + h) * (D + 4); };
    float top = -__builtin_inff(), l = 0.0f;
    float4_t sum = {0, 0, 0, 0};
    auto add = [&](auto count, int b) {
        constexpr int kCount = decltype(count)::value;
        float2_t ml[kCount];
        float4_t v[kCount];
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const float* p = part(b + WAVES * i <= blocks.y ? b + WAVES * i : b);
            ml[i] = *reinterpret_cast<const float2_t*>(p + D);
            v[i] = d < D ? *reinterpret_cast<const float4_t*>(p + d) : float4_t{0, 0, 0, 0};
        }
        float now = top;
#pragma unroll
        for (int i = 0; i < kCount; ++i) now = fmaxf(now, ml[i][0]);
        const float f = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(top - now);
        l *= f;
        sum *= f;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            if (b + WAVES * i > blocks.y) continue;
            const float fi = ml[i][0] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml[i][0] - now);
            l += fi * ml[i][1];
            sum += fi * v[i];
        }
        top = now;
    };
    int b = blocks.x + wave;
    if constexpr (WAVES == 1)
        for (; b + 4 <= blocks.y; b += 16) add(std::integral_constant<int, 16>{}, b);
    for (; b <= blocks.y; b += 4 * WAVES) add(std::integral_constant<int, 4>{}, b);
    const float scale = c.v_scale ? c.v_scale[kvh] : 1.0f;
    if constexpr (WAVES == 1) {
        if (d < D) store_attended<T>(a, at, d, sum, l, top, scale);
    } else {
        __shared__ float wave_m[WAVES], wave_l[WAVES];
        __shared__ float parts[WAVES][256];
        if (lane == 0) {
            wave_m[wave] = top;
            wave_l[wave] = l;
        }
        *reinterpret_cast<float4_t*>(&parts[wave][d]) = sum;
        __syncthreads();
        if (wave != 0 || d >= D) return;
        float all = wave_m[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) all = fmaxf(all, wave_m[w]);
        float weight = 0.0f;
        sum = float4_t{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = wave_m[w] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(wave_m[w] - all);
            weight += f * wave_l[w];
            sum += f * *reinterpret_cast<const float4_t*>(&parts[w][d]);
        }
        store_attended<T>(a, at, d, sum, weight, all, scale);
    }
}
}  // namespace pimhip
