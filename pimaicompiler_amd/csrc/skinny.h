// Sums of a few tokens against many rows of weights on the matrix cores: what the products with 4-bit weights and the experts of a
// mixture share.
//
//   acc[row, token] = sum_k w[row, k] * x[token, k]          v_mfma_f32_16x16x32: 16 rows x 16 tokens x 32 k
//
// The weights are read once and are what bounds such a product.  The matrix cores want lane l to hold row l % 16, but a load is
// taken 16 lanes at a time, and 16 lanes in 16 rows are 16 requests: loading operands as they are wanted ran at 3.7 TB/s at the most
// (16384 x 4096 in 4 bits, one token) and, with x alike, at 0.5 TB/s (64 tokens).  So a wavefront loads runs of 128 or 256 bytes of a row, and
// turns them by writing them to LDS and reading them back: memory of its own, no barrier.  A row's 16-byte chunk c lies at
// place c ^ (row % 8) there, which spreads 8 rows' equal chunks over all banks.
//
// k is taken in steps of 128 (four products) and in units: of a unit, lane l has the 32 values from 32 (l / 16) on of each step, the
// products take eight of them each.  The order of k is the same for both operands and otherwise free.  A wavefront asks for a unit of both
// operands behind the products of the one before, and others of its CU fill the wait; x is asked for with its weights, since a
// wavefront's loads come back in order.
#pragma once

#include <type_traits>

#include "mx4_format.h"

namespace pimhip
{
static constexpr int kSkinnyStep = 128;  // values of k of four products

// Orders a wavefront's LDS accesses before and behind it; they are carried out in order, so no instruction is needed.
__device__ __forceinline__ void wave_lds_order()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 16 rows of 16-bit values (weights, or tokens), 128 values a unit: lane l loads chunk l % 16 of rows l / 16 + 4 j.
template <class T>
struct DenseTile {
    static constexpr int kUnit = 128, kLds = 16 * 16;  // (in 16-byte words)
    struct Raw {
        typename T::frag v[4];
    };
    static __device__ __forceinline__ void to_lds(const Raw& w, uint4_t* lds)
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = lane / 16 + 4 * j;
            lds[row * 16 + ((lane & 15) ^ (row & 7))] = __builtin_bit_cast(uint4_t, w.v[j]);
        }
    }
    // This lane's operands of the unit's four products.
    static __device__ __forceinline__ void from_lds(typename T::frag (&f)[4], const uint4_t* lds)
    {
        const int row = threadIdx.x & 15, group = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int o = 0; o < 4; ++o) f[o] = __builtin_bit_cast(typename T::frag, lds[row * 16 + ((group * 4 + o) ^ (row & 7))]);
    }
};

// 16-bit weights, rows of any length at any address of a value.  A tile's rows are addressed from its first one, which all lanes share.
template <class T>
struct DenseWeights {
    typedef DenseTile<T> Tile;
    typedef typename Tile::Raw Raw;
    static constexpr int kUnit = Tile::kUnit, kLds = Tile::kLds;
    struct Rows {
        const char* base;
        unsigned int at[4];  // bytes from there to the lane's four rows' chunks
    };
    struct Operands {
        typename T::frag f[4];
    };
    // Rows first .. first + 15 of a matrix of `count` rows of K values (first is one of them); rows behind its end are its last one again.
    static __device__ __forceinline__ Rows rows(const void* w, int64_t first, int64_t count, int64_t K)
    {
        Rows r;
        const int lane = threadIdx.x & 63, last = (int)(count - 1 - first < 15 ? count - 1 - first : 15);
        r.base = (const char*)w + first * K * 2;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = lane / 16 + 4 * j;
            r.at[j] = (unsigned int)(at < last ? at : last) * (unsigned int)(K * 2) + (lane & 15) * 16;
        }
        return r;
    }
    static __device__ __forceinline__ void load(Raw& w, const Rows& r, int unit)
    {
        const char* p = r.base + (int64_t)unit * (kUnit * 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) w.v[j] = __builtin_bit_cast(typename T::frag, (uint4_t)load_global_once<uint4_any_t>(p + r.at[j]));
    }
    static __device__ __forceinline__ void load_guarded(Raw& w, const Rows& r, int unit, int K)
    {
        const char* p = r.base + (int64_t)unit * (kUnit * 2);
        const int left = K - unit * kUnit - (int)(threadIdx.x & 15) * 8;
#pragma unroll
        for (int j = 0; j < 4; ++j) w.v[j] = left >= 8 ? __builtin_bit_cast(typename T::frag, (uint4_t)load_global<uint4_any_t>(p + r.at[j])) : typename T::frag{};
        if (K % 8 != 0 && left > 0 && left < 8)
#pragma unroll
            for (int j = 0; j < 4; ++j) w.v[j] = load8_guarded<T>(reinterpret_cast<const typename T::elem*>(p + r.at[j]), 0, left);
    }
    static __device__ __forceinline__ void turn(Operands& o, const Raw& w, const Rows&, uint4_t* lds)
    {
        Tile::to_lds(w, lds);
        wave_lds_order();
        Tile::from_lds(o.f, lds);
        wave_lds_order();
    }
    static __device__ __forceinline__ typename T::frag operand(const Operands& o, int, int product) { return o.f[product]; }
};

// 4-bit weights, S steps (of 128 values, four blocks) a unit; T is the type of x.  Lane l loads chunk l % (4 S), a block, of rows
// l / (4 S) + 16 / S j, and of the unit's scale codes S of row l / 4.  Two steps are whole lines of 128 bytes; one step leaves more registers
// to tokens.
template <class T, int S>
struct Mx4Weights {
    static_assert(S == 1 || S == 2, "one or two steps a unit");
    static constexpr int kUnit = S * kSkinnyStep, kRow = 4 * S, kLds = 16 * kRow + 4 * S;  // (rows of 64 S bytes, then their codes)
    typedef typename std::conditional<S == 1, uint8_t, uint16_t>::type Codes;
    struct Rows {
        const uint8_t* base;
        const uint8_t* codes;
        unsigned int at[S], codes_at;  // bytes from there to the lane's rows' blocks and codes
        int top;                       // the largest scale code of row l % 16
    };
    struct Raw {
        uint4_t v[S];
        Codes codes;
    };
    struct Operands {
        uint4_t v[S];    // this lane's block of each step
        float scale[S];
    };
    static __device__ __forceinline__ Rows rows(const uint8_t* packed, const uint8_t* scales, const uint8_t* tops, int64_t ld_scales, int64_t first, int64_t count,
                                                int64_t K)
    {
        Rows r;
        const int lane = threadIdx.x & 63, last = (int)(count - 1 - first < 15 ? count - 1 - first : 15);
        const int64_t pitch = (K + kMxBlock - 1) / kMxBlock * kMxBlockBytes;
        auto row = [&](int i) { return (unsigned int)(i < last ? i : last); };
        r.base = packed + first * pitch;
        r.codes = scales + first * ld_scales;
#pragma unroll
        for (int j = 0; j < S; ++j) r.at[j] = row(lane / kRow + 16 / S * j) * (unsigned int)pitch + lane % kRow * kMxBlockBytes;
        r.codes_at = row(lane / 4) * (unsigned int)ld_scales + (lane & 3) * S;
        r.top = tops[first + row(lane & 15)];
        return r;
    }
    static __device__ __forceinline__ void load(Raw& w, const Rows& r, int unit)
    {
        const uint8_t* p = r.base + (int64_t)unit * (kUnit / 2);
#pragma unroll
        for (int j = 0; j < S; ++j) w.v[j] = load_global_once<uint4_t>(p + r.at[j]);
        w.codes = load_global<Codes>(r.codes + (int64_t)unit * kRow + r.codes_at);  // (whole groups of 16 codes a row)
    }
    static __device__ __forceinline__ void load_guarded(Raw& w, const Rows& r, int unit, int K)
    {
        const int lane = threadIdx.x & 63;
        const uint8_t* p = r.base + (int64_t)unit * (kUnit / 2);
        const bool in = unit * kUnit + lane % kRow * kMxBlock < K;
#pragma unroll
        for (int j = 0; j < S; ++j) w.v[j] = in ? load_global<uint4_t>(p + r.at[j]) : uint4_t{0, 0, 0, 0};
        unsigned int codes = load_global<Codes>(r.codes + (int64_t)unit * kRow + r.codes_at);
        // What lies behind the row's last block may be anything: 0, the one code that is above no row's top.
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (unit * kUnit + ((lane & 3) * S + s) * kMxBlock >= K) codes &= ~(255u << (8 * s));
        w.codes = (Codes)codes;
    }
    static __device__ __forceinline__ int place(int row, int chunk) { return row * kRow + (chunk ^ (S == 2 ? row & 7 : row / 4 & 3)); }
    static __device__ __forceinline__ void turn(Operands& o, const Raw& w, const Rows& r, uint4_t* lds)
    {
        const int lane = threadIdx.x & 63, row = lane & 15, group = lane >> 4;
#pragma unroll
        for (int j = 0; j < S; ++j) lds[place(lane / kRow + 16 / S * j, lane % kRow)] = w.v[j];
        reinterpret_cast<Codes*>(lds + 16 * kRow)[lane] = w.codes;
        wave_lds_order();
        const unsigned int* codes = reinterpret_cast<const unsigned int*>(lds + 16 * kRow) + row * S;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            o.v[s] = lds[place(row, s * 4 + group)];
            o.scale[s] = T::scale((codes[s] >> (8 * group)) & 255u, r.top);
        }
        wave_lds_order();
    }
    static __device__ __forceinline__ typename T::frag operand(const Operands& o, int step, int product) { return T::from_mx4(o.v[step][product], o.scale[step]); }
};

// The tokens of a product, loaded and turned like weights by each wavefront.  WHOLE: their rows are whole groups of eight values.
// (raws: how many loads of a step the tiles of 16 columns make.)
template <class T, bool WHOLE>
struct TurnedTokens {
    typedef DenseTile<T> Tile;
    typedef typename Tile::Raw Raw;
    static constexpr int kLds = Tile::kLds;
    static constexpr int raws(int tiles) { return tiles; }
    struct Rows {
        const typename T::elem* p[4];  // the lane's four rows, at its chunk
    };
    // row(i): the token of column i, as a pointer to its values
    template <class F>
    static __device__ __forceinline__ Rows rows(F row)
    {
        Rows r;
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < 4; ++j) r.p[j] = row(lane / 16 + 4 * j) + (lane & 15) * 8;
        return r;
    }
    static __device__ __forceinline__ void load(Raw& w, const Rows& r, int step)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) w.v[j] = load8_any<T>(r.p[j] + (int64_t)step * kSkinnyStep);
    }
    static __device__ __forceinline__ void load_guarded(Raw& w, const Rows& r, int step, int K)
    {
        const int chunk = threadIdx.x & 15;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (WHOLE)
                w.v[j] = step * kSkinnyStep + chunk * 8 < K ? load8_any<T>(r.p[j] + (int64_t)step * kSkinnyStep) : typename T::frag{};
            else
                w.v[j] = load8_guarded<T>(r.p[j] - chunk * 8, (int64_t)step * kSkinnyStep + chunk * 8, K);
        }
    }
    static __device__ __forceinline__ void turn(typename T::frag (&f)[4], Raw& w, const Rows&, int, int, uint4_t* lds)
    {
        Tile::to_lds(w, lds);
        wave_lds_order();
        Tile::from_lds(f, lds);
        wave_lds_order();
    }
};

// The tokens of a product that fit LDS as a whole: staged once by the block, read by all its wavefronts as the matrix cores want
// them.  A token's row is 16 bytes longer than its values, which spreads eight tokens' equal chunks over all banks.
template <class T>
struct SharedTokens {
    struct Raw {};
    struct Rows {
        const uint4_t* p;
    };
    static constexpr int kLds = 0;
    static constexpr int raws(int tiles) { return tiles; }
    // 16-byte words of a token, of K values filled up to whole units.
    static __host__ __device__ constexpr int pitch(int K, int unit) { return (K + unit - 1) / unit * (unit / 8) + 1; }
    static __device__ __forceinline__ Rows rows(const uint4_t* xs, int token, int pitch) { return {xs + token * pitch + ((threadIdx.x & 63) >> 4) * 4}; }
    template <class F>
    static __device__ __forceinline__ void stage(uint4_t* xs, F row, int n, int K, int pitch)
    {
        const int chunks = pitch - 1;
        for (int i = threadIdx.x; i < n * chunks; i += blockDim.x) {
            const int t = i / chunks, c = i % chunks;
            xs[t * pitch + c] = __builtin_bit_cast(uint4_t, load8_guarded<T>(row(t), (int64_t)c * 8, K));
        }
    }
    static __device__ __forceinline__ void load(Raw&, const Rows&, int) {}
    static __device__ __forceinline__ void load_guarded(Raw&, const Rows&, int, int) {}
    static __device__ __forceinline__ void turn(typename T::frag (&f)[4], Raw&, const Rows& r, int step, int, uint4_t*)
    {
#pragma unroll
        for (int o = 0; o < 4; ++o) f[o] = __builtin_bit_cast(typename T::frag, r.p[step * (kSkinnyStep / 8) + o]);
    }
};

// LDS a wavefront needs for itself, in 16-byte words.
template <class W, class X>
constexpr int kSkinnyLds = W::kLds + X::kLds;

// acc[i][j] += 16 rows i x 16 tokens j over units first, first + stride, ... of K.  `lds`: this wavefront's kSkinnyLds words.
// ready() is called once, behind the first loads of weights: there a block stages what its wavefronts share.
template <class T, class W, class X, int RT, int TT, class R>
__device__ __forceinline__ void skinny_sum(float4_t (&acc)[RT][TT], const typename W::Rows (&w)[RT], const typename X::Rows (&x)[X::raws(TT)], int K, int first, int stride,
                                           uint4_t* lds, R ready)
{
    typedef typename T::frag frag;
    constexpr int S = W::kUnit / kSkinnyStep, XR = X::raws(TT);  // steps of a unit
    const int whole = K / W::kUnit;
    const int mine = first < whole ? (whole - first + stride - 1) / stride : 0;  // this wavefront's whole units
    typename W::Raw wv[RT];
    typename X::Raw xv[S][XR];
    auto ask = [&](int n) {
        const int unit = first + n * stride;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < XR; ++j) X::load(xv[s][j], x[j], unit * S + s);
#pragma unroll
        for (int i = 0; i < RT; ++i) W::load(wv[i], w[i], unit);
    };
    auto products = [&](int unit) {
        typename W::Operands a[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) W::turn(a[i], wv[i], w[i], lds);
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                frag f[4];
                X::turn(f, xv[s][j % XR], x[j % XR], unit * S + s, j, lds + W::kLds);
#pragma unroll
                for (int o = 0; o < 4; ++o)
#pragma unroll
                    for (int i = 0; i < RT; ++i) acc[i][j] = T::mfma(W::operand(a[i], s, o), f[o], acc[i][j]);
            }
    };
    if (mine > 0) ask(0);
    ready();
    for (int n = 0; n + 1 < mine; ++n) {
        products(first + n * stride);
        ask(n + 1);
    }
    if (mine > 0) products(first + (mine - 1) * stride);
    // The unit that K ends in.
    if (K % W::kUnit != 0 && whole % stride == first) {
#pragma unroll
        for (int i = 0; i < RT; ++i) W::load_guarded(wv[i], w[i], whole, K);
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < XR; ++j) X::load_guarded(xv[s][j], x[j], whole * S + s, K);
        products(whole);
    }
}

// Sums of the WK wavefronts of a block, which shared k: tile (i, j) ends up in wavefront (i * TT + j) % WK.  `part` is
// WK * RT * TT * 64 vectors of LDS, which may be the memory the sums were made with.  The order of the sum is the wavefronts'.
template <int RT, int TT, int WK>
__device__ __forceinline__ void skinny_join(float4_t (&acc)[RT][TT], float4_t* part)
{
    const int lane = threadIdx.x & 63, wave = wave_in_block();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) part[((wave * RT + i) * TT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            if ((i * TT + j) % WK != wave) continue;
            float4_t v = part[(i * TT + j) * 64 + lane];
#pragma unroll
            for (int k = 1; k < WK; ++k) v += part[((k * RT + i) * TT + j) * 64 + lane];
            acc[i][j] = v;
        }
}
}  // namespace pimhip
