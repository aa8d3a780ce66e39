// A cache of keys and values in pages on gfx950: appending to it with the position rotation on the way, and attention of each
// sequence's new token over it.
//
//   append    a pair (a, b) of a key's or query's first `rotary` values becomes (a c - b w, a w + b c), c and w the cosine and sine of
//             its token's position; the token at position p lies in place p % page_size of page table[sequence, p / page_size]
//   attend    o = sum_j e_j v_j / sum_j e_j,  e_j = exp(scale q . k_j - m),  j over the sequence's last `window` tokens
#pragma once

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
    int sequences, width;
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
    int tokens, q_heads, half;  // half: pairs of a head that are turned
    int items;                  // groups of eight of a token
};

// A block is one token's heads, a thread eight values of one: of a key (query) the eight behind them or half a rotation away are loaded
// beside them, out of the caches as a rule.  Bound by the bytes where tokens are many, else by four dependent loads: the sequence, its length,
// the page, the values.
template <class T, bool FP8, bool INTERLEAVED>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a)
{
    typedef typename T::elem elem;
    const int t = blockIdx.x;
    const int item = blockIdx.y * 256 + threadIdx.x;
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
    int page = -1;
    if (pos >= 0) page = a.c.table[s * a.c.ld_table + a.c.page_of(pos)];
    if (item >= a.items) return;
    const int groups = a.c.dim / 8, head_of_all = item / groups, d = (item - head_of_all * groups) * 8;
    const bool is_k = head_of_all < a.c.kv_heads, is_v = !is_k && head_of_all < 2 * a.c.kv_heads;
    const int head = is_k ? head_of_all : is_v ? head_of_all - a.c.kv_heads : head_of_all - 2 * a.c.kv_heads;
    const bool stored = page >= 0 && page < a.c.pages;
    if (!is_k && !is_v && pos < 0) {  // a query of no sequence
        *reinterpret_cast<uint4_any_t*>((elem*)a.q_out + ((int64_t)t * a.q_heads + head) * a.c.dim + d) = uint4_t{0, 0, 0, 0};
        return;
    }
    if ((is_k || is_v) && !stored) return;
    const elem* x = is_k   ? (const elem*)a.k + t * a.k_token + head * a.k_head
                    : is_v ? (const elem*)a.v + t * a.v_token + head * a.v_head
                           : (const elem*)a.q + t * a.q_token + head * a.q_head;
    const typename T::frag mine = load8_any<T>(x + d);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (float)mine[i];
    if (!is_v && d < 2 * a.half) {
        const float* row = a.angles + pos * a.ld_angles;
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = d / 2 + i;
                if (p < a.half) {
                    const float c = row[p], w = row[a.half + p], u = y[2 * i], v = y[2 * i + 1];
                    y[2 * i] = u * c - v * w;
                    y[2 * i + 1] = u * w + v * c;
                }
            }
        } else {
            // A group may hold values of both halves, and values behind them, where a half is no multiple of eight.
            const bool whole = a.half % 8 == 0;
            typename T::frag other = {};
            if (whole) other = load8_any<T>(x + (d < a.half ? d + a.half : d - a.half));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = d + i;
                if (whole || e < 2 * a.half) {
                    const bool first = e < a.half;
                    const int p = first ? e : e - a.half;
                    const float o = whole ? (float)other[i] : (float)x[first ? e + a.half : e - a.half];
                    const float c = row[p], w = row[a.half + p];
                    y[i] = first ? y[i] * c - o * w : o * w + y[i] * c;
                }
            }
        }
    }
    if (!is_k && !is_v) {
        elem* out = (elem*)a.q_out + ((int64_t)t * a.q_heads + head) * a.c.dim + d;
        const elem r[8] = {T::round(y[0]), T::round(y[1]), T::round(y[2]), T::round(y[3]), T::round(y[4]), T::round(y[5]), T::round(y[6]), T::round(y[7])};
        *reinterpret_cast<uint4_any_t*>(out) = __builtin_bit_cast(uint4_t, r);
        return;
    }
    const int at = pos - a.c.page_of(pos) * a.c.page_size;
    char* out = is_k ? a.c.k + page * a.c.k_page + head * a.c.k_head + (int64_t)at * a.c.k_tok
                     : a.c.v + page * a.c.v_page + head * a.c.v_head + (int64_t)at * a.c.v_tok;
    if constexpr (FP8) {
        const float scale = (is_k ? a.c.k_scale : a.c.v_scale)[head];
        unsigned char r[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const unsigned int two = to_e4m3x2(y[i] / scale, y[i + 1] / scale);
            r[i] = (unsigned char)two;
            r[i + 1] = (unsigned char)(two >> 8);
        }
        typedef uint2_t bytes8_t __attribute__((aligned(1)));
        *reinterpret_cast<bytes8_t*>(out + d) = __builtin_bit_cast(uint2_t, r);
    } else {
        const elem r[8] = {T::round(y[0]), T::round(y[1]), T::round(y[2]), T::round(y[3]), T::round(y[4]), T::round(y[5]), T::round(y[6]), T::round(y[7])};
        *reinterpret_cast<uint4_any_t*>(out + 2 * d) = __builtin_bit_cast(uint4_t, r);
    }
}

// ---- attend ---------------------------------------------------------------------------------------
//
// The tokens of all sequences and key heads lie in a row of units of 64; each block takes an equal stretch of them, so that lengths may differ
// as they like.  A piece of a (sequence, key head) that does not fill it goes to the workspace with its own maximum and sum, and a second
// kernel joins such pieces.  A wavefront takes 16 tokens of a unit at a time:
//   scores    K [16 tokens x dim] . Q^T [dim x 16 heads] on the 16-bit matrix instruction (8-bit keys become Q's type, exactly): a lane has
//             the scores of head l % 16 and tokens 4 (l / 16) + r
//   values    P [16 heads x 4 tokens] . V [4 tokens x 16 columns] on the 32-bit one, for tokens r, 4 + r, 8 + r, 12 + r: a lane's e_j are its
//             operand as they are, unrounded, and V is one that 16 lanes read as one row: nothing is turned or exchanged
// Values lie in registers from memory on; a tile's loads are issued while the one before is worked on.
static constexpr int kUnit = 64;           // tokens that the four wavefronts of a block take together
static constexpr float kLazy = 40.0f;      // a running maximum moves on when a score is above it by so many powers of two

struct AttendArgs {
    PagedView c;
    const void* q;
    void* out;
    float* lse;   // [sequences, heads] or null
    float* work;  // [blocks][2][16 * tiles][dim + 4]
    int64_t q_seq, q_head;  // elements
    int group, tiles_of_heads, window;
    float scale_log2;
};

struct PagedSpan {
    int first, base, end, units;  // tokens first .. end - 1 are seen; tiles begin at base
};
__device__ __forceinline__ PagedSpan paged_span(const PagedView& c, int window, int s)
{
    PagedSpan p;
    p.end = paged_length(c, s);
    p.first = window > 0 && p.end > window ? p.end - window : 0;
    p.base = p.first & ~15;
    const int n = (p.end - p.base + kUnit - 1) / kUnit;
    p.units = n < 1 ? 1 : n;  // (a sequence of no tokens has a result too)
    return p;
}

// Where in the row of units (`times` units for each of a sequence's) a sequence begins, and how many units there are in all, by a block
// of 256.  ask(total) is the unit whose sequence is looked for, or -1 - s for sequence s.
struct PagedFound {
    int64_t before, total;
    int s;
};
template <class F>
__device__ __forceinline__ PagedFound paged_find(const PagedView& c, int window, int64_t times, F ask)
{
    __shared__ int64_t wave_sum_of[4];
    __shared__ int64_t found_before;
    __shared__ int found_s;
    const int each = (c.sequences + 255) / 256, from = (int)threadIdx.x * each, lo = from < c.sequences ? from : c.sequences;
    const int hi = lo + each < c.sequences ? lo + each : c.sequences;
    int64_t mine = 0;
    for (int s = lo; s < hi; ++s) mine += paged_span(c, window, s).units;
    int64_t incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t o = __shfl_up(incl, d);
        if ((int)(threadIdx.x & 63) >= d) incl += o;
    }
    if ((threadIdx.x & 63) == 63) wave_sum_of[threadIdx.x >> 6] = incl;
    __syncthreads();
    int64_t before = incl - mine, total = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < (int)(threadIdx.x >> 6)) before += wave_sum_of[w];
        total += wave_sum_of[w];
    }
    PagedFound f;
    f.total = total * times;
    const int64_t u = ask(f.total);
    const int want = u < 0 ? (int)(-1 - u) : -1;
    if (u < 0 ? lo <= want && want < hi : before * times <= u && u < (before + mine) * times) {
        int s = lo;
        for (; s < hi - 1; ++s) {
            const int n = paged_span(c, window, s).units;
            if (u < 0 ? s == want : u < (before + n) * times) break;
            before += n;
        }
        found_before = before;
        found_s = s;
    }
    __syncthreads();
    f.before = found_before;
    f.s = found_s;
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
        typedef unsigned int words_t __attribute__((ext_vector_type(kWords)));
        typedef words_t words_any_t __attribute__((aligned(1)));
        if constexpr (kWords == 1) {
            typedef unsigned int word_any_t __attribute__((aligned(1)));
            w[0] = load_global<word_any_t>(p);
        } else {
            const words_t q = load_global<words_any_t>(p);
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
        } else if constexpr (sizeof(typename T::elem) == 2 && __is_same(T, BF16)) {
            return __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        } else {
            return (float)__builtin_bit_cast(half2_t, w[i / 2])[i % 2];
        }
    }
};

// NC: the head's size in 64 columns, rounded up; MT: 16 query heads each; ONE: pages are whole tiles of 16 tokens.
template <class T, bool FP8, int NC, int MT, bool ONE>
__global__ __launch_bounds__(256, 2) void paged_attend_kernel(AttendArgs a)
{
    typedef typename T::elem elem;
    typedef typename T::frag frag;
    constexpr int kSteps = NC * 2;                   // matrix instructions along a head's values
    constexpr int kLoads = FP8 ? NC : kSteps;        // 16-byte loads of a key's row by a lane
    constexpr int kWide = NC / 2, kNarrow = NC % 2;  // pieces of eight and of four columns of a lane
    constexpr int kCols = NC * 4, kSize = FP8 ? 1 : 2;
    __shared__ float wave_m[4][16 * MT], wave_l[4][16 * MT];
    __shared__ float parts[2][16 * MT][NC * 64 + 4];
    const int lane = threadIdx.x & 63, wave = wave_in_block(), n = lane & 15, g = lane >> 4;
    const PagedView& c = a.c;
    const int D = c.dim;
    const int64_t heads_of_units = (int64_t)c.kv_heads * a.tiles_of_heads;

    // ---- this block's stretch ----
    int64_t per = 0;
    const PagedFound at = paged_find(c, a.window, heads_of_units, [&](int64_t total) {
        per = (total + gridDim.x - 1) / gridDim.x;
        const int64_t first = blockIdx.x * per;
        return first < total ? first : total - 1;
    });
    int64_t u = blockIdx.x * per;
    const int64_t u_end = u + per < at.total ? u + per : at.total;
    if (u >= u_end) return;
    int s = at.s;
    int64_t before = at.before;

    while (u < u_end) {
        const PagedSpan span = paged_span(c, a.window, s);
        const int rel = (int)(u - before * heads_of_units), hg = rel / span.units, first = rel - hg * span.units;
        const int left = span.units - first, take = left < u_end - u ? left : (int)(u_end - u), last = first + take;
        const int kvh = hg / a.tiles_of_heads, head0 = (hg - kvh * a.tiles_of_heads) * 16 * MT;

        // ---- queries ----
        frag q[MT][kSteps];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
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

        float m[MT], l[MT];
        float4_t o[MT][kCols];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            m[mt] = -__builtin_inff();
            l[mt] = 0.0f;
#pragma unroll
            for (int i = 0; i < kCols; ++i) o[mt][i] = float4_t{0, 0, 0, 0};
        }

        // ---- tiles: 16 tokens of each unit ----
        uint4_t k[kLoads];
        ValuePiece<T, FP8, 8> wide[4][kWide ? kWide : 1];
        ValuePiece<T, FP8, 4> narrow[4][kNarrow ? kNarrow : 1];
        // This wavefront's first token of a unit; a unit behind the stretch's end has none.
        auto token_of = [&](int unit) { return unit < last ? span.base + unit * kUnit + wave * 16 : span.end; };
        // A tile's page (ONE), or the page of each of its 16 tokens (a lane each, the same in the four groups); -1: none.
        auto page_at = [&](int token) {
            const int mine = token + (ONE ? 0 : n);
            return token < span.end && mine < span.end ? row[c.page_of(mine)] : -1;
        };
        // Where they lie: a page that is none is read as page 0, and not seen.
        struct Place {
            int page, in;
            unsigned int ok;  // a bit for each token
        };
        auto place_of = [&](int token, int page) {
            const int mine = token + (ONE ? 0 : n);
            const bool ok = page >= 0 && page < c.pages;
            return Place{ok ? page : 0, mine - c.page_of(mine) * c.page_size, ONE ? (ok ? 0xffffu : 0u) : (unsigned int)__ballot(ok) & 0xffffu};
        };
        auto load_keys = [&](const Place& p) {
            const char* kp = kh + p.page * c.k_page + (int64_t)(p.in + (ONE ? n : 0)) * c.k_tok;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int byte = i * 64 + g * 16;
                k[i] = uint4_t{0, 0, 0, 0};
                if (byte < D * kSize) k[i] = load_global<uint4_any_t>(kp + byte);
            }
        };
        auto load_values = [&](const Place& p, int r) {
            const int page = ONE ? p.page : __shfl(p.page, g * 4 + r), in = ONE ? p.in + g * 4 + r : __shfl(p.in, g * 4 + r);
            const char* vp = vh + page * c.v_page + (int64_t)in * c.v_tok;
#pragma unroll
            for (int i = 0; i < kWide; ++i) {
                wide[r][i].clear();
                if (i * 128 + n * 8 < D) wide[r][i].load(vp + (i * 128 + n * 8) * kSize);
            }
            if constexpr (kNarrow) {
                narrow[r][0].clear();
                if (kWide * 128 + n * 4 < D) narrow[r][0].load(vp + (kWide * 128 + n * 4) * kSize);
            }
        };

        int token = token_of(first), next = token_of(first + 1);
        Place place = place_of(token < span.end ? token : span.base, page_at(token));
        if (token < span.end) {
            load_keys(place);
#pragma unroll
            for (int r = 0; r < 4; ++r) load_values(place, r);
        }
        int page = page_at(next);
        for (int unit = first; token < span.end; ++unit) {
            const bool more = next < span.end;
            const Place then = place_of(more ? next : span.base, page);
            const int next2 = token_of(unit + 2);
            page = page_at(next2);
            // Tokens that are not the sequence's, or not in the window, or of no page, are left out, whatever lies there.
            unsigned int seen = place.ok;
            if (token < span.first) seen &= 0xffffu << (span.first - token);
            if (token + 16 > span.end) seen &= 0xffffu >> (token + 16 - span.end);

            float4_t sc[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) sc[mt] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                frag kf;
                if constexpr (FP8)
                    kf = from_e4m3x8<T>(i % 2 ? uint2_t{k[i / 2][2], k[i / 2][3]} : uint2_t{k[i / 2][0], k[i / 2][1]});
                else
                    kf = __builtin_bit_cast(frag, k[i]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) sc[mt] = T::mfma(kf, q[mt][i], sc[mt]);
            }
            if (more) load_keys(then);
            bool above = false;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                sc[mt] *= scale;
                if (seen != 0xffffu)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[mt][r] = seen >> (g * 4 + r) & 1 ? sc[mt][r] : -__builtin_inff();
#pragma unroll
                for (int r = 0; r < 4; ++r) above |= sc[mt][r] > m[mt] + kLazy;
            }
            if (__ballot(above)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float top = fmaxf(fmaxf(sc[mt][0], sc[mt][1]), fmaxf(sc[mt][2], sc[mt][3]));
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float now = fmaxf(m[mt], top);
                    const float f = m[mt] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m[mt] - now);
                    m[mt] = now;
                    l[mt] *= f;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float fr = __shfl(f, g * 4 + r);
#pragma unroll
                        for (int i = 0; i < kCols; ++i) o[mt][i][r] *= fr;
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float p[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    p[mt] = sc[mt][r] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(sc[mt][r] - m[mt]);
                    l[mt] += p[mt];
                }
                if (seen != 0xffffu && !(seen >> (g * 4 + r) & 1)) {
#pragma unroll
                    for (int i = 0; i < kWide; ++i) wide[r][i].clear();
                    if constexpr (kNarrow) narrow[r][0].clear();
                }
#pragma unroll
                for (int i = 0; i < kWide; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float v = wide[r][i].value(e);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) o[mt][i * 8 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[mt], v, o[mt][i * 8 + e], 0, 0, 0);
                    }
                if constexpr (kNarrow)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = narrow[r][0].value(e);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
                            o[mt][kWide * 8 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[mt], v, o[mt][kWide * 8 + e], 0, 0, 0);
                    }
                if (more) load_values(then, r);
            }
            place = then;
            token = next;
            next = next2;
        }

        // ---- the four wavefronts' parts ----
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            l[mt] += __shfl_xor(l[mt], 16);
            l[mt] += __shfl_xor(l[mt], 32);
            if (g == 0) {
                wave_m[wave][mt * 16 + n] = m[mt];
                wave_l[wave][mt * 16 + n] = l[mt];
            }
        }
        __syncthreads();
        auto column = [&](int i) { return i < kWide * 8 ? i / 8 * 128 + n * 8 + i % 8 : kWide * 128 + n * 4 + i - kWide * 8; };
        float all_l[MT][4], all_m[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int h = mt * 16 + g * 4 + r;
                const float top = fmaxf(fmaxf(wave_m[0][h], wave_m[1][h]), fmaxf(wave_m[2][h], wave_m[3][h]));
                float sum = 0.0f, f = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float fw = wave_m[w][h] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(wave_m[w][h] - top);
                    sum += fw * wave_l[w][h];
                    if (w == wave) f = fw;
                }
                all_m[mt][r] = top;
                all_l[mt][r] = sum;
#pragma unroll
                for (int i = 0; i < kCols; ++i) o[mt][i][r] *= f;
            }
        for (int half = 2; half >= 1; half /= 2) {
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int i = 0; i < kCols; ++i) parts[wave - half][mt * 16 + g * 4 + r][column(i)] = o[mt][i][r];
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int i = 0; i < kCols; ++i) o[mt][i][r] += parts[wave][mt * 16 + g * 4 + r][column(i)];
            }
            __syncthreads();
        }
        if (wave == 0) {
            const bool complete = first == 0 && last == span.units;
            const float vs = FP8 ? c.v_scale[kvh] : 1.0f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int h = head0 + mt * 16 + g * 4 + r;
                    if (h >= a.group) continue;
                    if (complete) {
                        const float f = all_l[mt][r] == 0.0f ? 0.0f : vs / all_l[mt][r];
                        const int64_t at_out = (int64_t)s * c.kv_heads * a.group + kvh * a.group + h;
                        elem* out = (elem*)a.out + at_out * D;
#pragma unroll
                        for (int i = 0; i < kCols; ++i)
                            if (column(i) < D) out[column(i)] = T::round(o[mt][i][r] * f);
                        if (a.lse && n == 0) a.lse[at_out] = (all_m[mt][r] + __builtin_amdgcn_logf(all_l[mt][r])) * 0.6931471805599453f;
                    } else {
                        float* part = a.work + (((int64_t)blockIdx.x * 2 + (first == 0 ? 1 : 0)) * 16 * MT + mt * 16 + g * 4 + r) * (D + 4);
#pragma unroll
                        for (int i = 0; i < kCols; ++i)
                            if (column(i) < D) part[column(i)] = o[mt][i][r];
                        if (n == 0) {
                            part[D] = all_m[mt][r];
                            part[D + 1] = all_l[mt][r];
                        }
                    }
                }
        }
        u += take;
        if (rel + take == heads_of_units * span.units) {
            before += span.units;
            ++s;
        }
    }
}

// The pieces of each (sequence, key head) that more than one block worked on.  `blocks`: those of the kernel before.
template <class T>
__global__ __launch_bounds__(256) void paged_join_kernel(AttendArgs a, int blocks, int rows)
{
    typedef typename T::elem elem;
    const PagedView& c = a.c;
    const int D = c.dim;
    const int hgs = c.kv_heads * a.tiles_of_heads, s = blockIdx.x / hgs, hg = blockIdx.x - s * hgs;
    const PagedFound at = paged_find(c, a.window, hgs, [&](int64_t) { return (int64_t)-1 - s; });
    const int units = paged_span(c, a.window, s).units;
    const int64_t per = (at.total + blocks - 1) / blocks;
    const int64_t u0 = at.before * hgs + (int64_t)hg * units;
    const int b0 = (int)(u0 / per), b1 = (int)((u0 + units - 1) / per);
    if (b0 == b1) return;
    const int kvh = hg / a.tiles_of_heads, head0 = (hg - kvh * a.tiles_of_heads) * rows;
    const int mine = a.group - head0 < rows ? a.group - head0 : rows, each = D / 4;
    const float vs = c.v_scale ? c.v_scale[kvh] : 1.0f;
    for (int i = threadIdx.x; i < mine * each; i += 256) {
        const int h = i / each, d = (i - h * each) * 4;
        // (a piece's place: the block's second where the sequence begins in it, else its first)
        auto part = [&](int b) { return a.work + (((int64_t)b * 2 + (b == b0 ? 1 : 0)) * rows + h) * (D + 4); };
        float top = -__builtin_inff();
        for (int b = b0; b <= b1; ++b) top = fmaxf(top, part(b)[D]);
        float4_t sum = {0, 0, 0, 0};
        float l = 0.0f;
        for (int b = b0; b <= b1; ++b) {
            const float* p = part(b);
            const float f = p[D] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(p[D] - top);
            l += f * p[D + 1];
            sum += f * *reinterpret_cast<const float4_t*>(p + d);
        }
        const float f = l == 0.0f ? 0.0f : vs / l;
        const int64_t at_out = (int64_t)s * c.kv_heads * a.group + kvh * a.group + head0 + h;
        elem* out = (elem*)a.out + at_out * D + d;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = T::round(sum[e] * f);
        if (a.lse && d == 0) a.lse[at_out] = (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
    }
}
}  // namespace pimhip
