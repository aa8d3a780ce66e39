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
// products take eight of them each.  The order of k is the same for both operands and otherwise free.  Each wavefront has U units of
// both operands on their way; x is asked for with its weights, since a wavefront's loads come back in order.
#pragma once

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
    struct Rows {
        const typename T::elem* p[4];  // the lane's four rows, at its chunk
    };
    struct Raw {
        typename T::frag v[4];
    };
    template <bool STREAM>
    static __device__ __forceinline__ void load(Raw& w, const Rows& r, int unit)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const typename T::elem* p = r.p[j] + (int64_t)unit * kUnit;
            if constexpr (STREAM)
                w.v[j] = __builtin_bit_cast(typename T::frag, (half8_t)__builtin_nontemporal_load(reinterpret_cast<const half8_any_t*>(p)));
            else
                w.v[j] = load8_any<T>(p);
        }
    }
    // The same where the rows may end inside the unit.
    static __device__ __forceinline__ void load_guarded(Raw& w, const Rows& r, int unit, int K)
    {
        const int chunk = threadIdx.x & 15;
#pragma unroll
        for (int j = 0; j < 4; ++j) w.v[j] = load8_guarded<T>(r.p[j] - chunk * 8, (int64_t)unit * kUnit + chunk * 8, K);
    }
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

// 16-bit weights.
template <class T>
struct DenseWeights {
    typedef DenseTile<T> Tile;
    typedef typename Tile::Raw Raw;
    typedef typename Tile::Rows Rows;
    static constexpr int kUnit = Tile::kUnit, kLds = Tile::kLds;
    struct Operands {
        typename T::frag f[4];
    };
    // Rows first .. first + 15 of a matrix of `count` rows of K values; rows behind its end are its last one again.
    static __device__ __forceinline__ Rows rows(const void* w, int64_t first, int64_t count, int64_t K)
    {
        Rows r;
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t at = first + lane / 16 + 4 * j;
            r.p[j] = (const typename T::elem*)w + (at < count ? at : count - 1) * K + (lane & 15) * 8;
        }
        return r;
    }
    static __device__ __forceinline__ void load(Raw& w, const Rows& r, int unit) { Tile::template load<true>(w, r, unit); }
    static __device__ __forceinline__ void load_guarded(Raw& w, const Rows& r, int unit, int K) { Tile::load_guarded(w, r, unit, K); }
    static __device__ __forceinline__ void turn(Operands& o, const Raw& w, const Rows&, uint4_t* lds)
    {
        Tile::to_lds(w, lds);
        wave_lds_order();
        Tile::from_lds(o.f, lds);
        wave_lds_order();
    }
    static __device__ __forceinline__ typename T::frag operand(const Operands& o, int, int product) { return o.f[product]; }
};

// 4-bit weights, 256 values a unit (two steps); T is the type of x.  Lane l loads chunk l % 8, a block, of rows l / 8 + 8 j, and of the
// unit's scale codes two of row l / 4.
template <class T>
struct Mx4Weights {
    static constexpr int kUnit = 256, kLds = 16 * 8 + 8;  // (rows of 128 bytes, then their codes)
    struct Rows {
        const uint8_t* p[2];
        const uint8_t* codes;
        int top;  // the largest scale code of row l % 16
    };
    struct Raw {
        uint4_t v[2];
        uint16_t codes;
    };
    struct Operands {
        uint4_t v[2];    // this lane's block of each step
        float scale[2];
    };
    static __device__ __forceinline__ Rows rows(const uint8_t* packed, const uint8_t* scales, const uint8_t* tops, int64_t ld_scales, int64_t first, int64_t count,
                                                int64_t K)
    {
        Rows r;
        const int lane = threadIdx.x & 63;
        const int64_t blocks = (K + kMxBlock - 1) / kMxBlock;
        auto row = [&](int i) { return first + i < count ? first + i : count - 1; };
#pragma unroll
        for (int j = 0; j < 2; ++j) r.p[j] = packed + (row(lane / 8 + 8 * j) * blocks + (lane & 7)) * kMxBlockBytes;
        r.codes = scales + row(lane / 4) * ld_scales + (lane & 3) * 2;
        r.top = tops[row(lane & 15)];
        return r;
    }
    static __device__ __forceinline__ void load(Raw& w, const Rows& r, int unit)
    {
#pragma unroll
        for (int j = 0; j < 2; ++j) w.v[j] = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(r.p[j] + (int64_t)unit * (kUnit / 2)));
        w.codes = *reinterpret_cast<const uint16_t*>(r.codes + unit * 8);  // (whole groups of 16 codes a row)
    }
    static __device__ __forceinline__ void load_guarded(Raw& w, const Rows& r, int unit, int K)
    {
        const int lane = threadIdx.x & 63;
        const bool in = unit * kUnit + (lane & 7) * kMxBlock < K;
#pragma unroll
        for (int j = 0; j < 2; ++j) w.v[j] = in ? *reinterpret_cast<const uint4_t*>(r.p[j] + (int64_t)unit * (kUnit / 2)) : uint4_t{0, 0, 0, 0};
        w.codes = *reinterpret_cast<const uint16_t*>(r.codes + unit * 8);
        // What lies behind the row's last block may be anything: any code but "not a number".
        const int left = K - unit * kUnit - (lane & 3) * 2 * kMxBlock;
        if (left <= kMxBlock) w.codes = (uint16_t)((w.codes & 0x00ff) | 0x7f00);
        if (left <= 0) w.codes = 0x7f7f;
    }
    static __device__ __forceinline__ void turn(Operands& o, const Raw& w, const Rows& r, uint4_t* lds)
    {
        const int lane = threadIdx.x & 63, row = lane & 15, group = lane >> 4;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int at = lane / 8 + 8 * j;
            lds[at * 8 + ((lane & 7) ^ (at & 7))] = w.v[j];
        }
        reinterpret_cast<uint16_t*>(lds + 16 * 8)[lane] = w.codes;
        wave_lds_order();
        const uint2_t codes = reinterpret_cast<const uint2_t*>(lds + 16 * 8)[row];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            o.v[h] = lds[row * 8 + ((h * 4 + group) ^ (row & 7))];
            o.scale[h] = T::scale((codes[h] >> (8 * group)) & 255u, r.top);
        }
        wave_lds_order();
    }
    static __device__ __forceinline__ typename T::frag operand(const Operands& o, int step, int product) { return T::from_mx4(o.v[step][product], o.scale[step]); }
};

// The tokens of a product, loaded and turned like weights by each wavefront.
template <class T>
struct TurnedTokens {
    typedef DenseTile<T> Tile;
    typedef typename Tile::Raw Raw;
    typedef typename Tile::Rows Rows;
    static constexpr int kLds = Tile::kLds;
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
    static __device__ __forceinline__ void load(Raw& w, const Rows& r, int step) { Tile::template load<false>(w, r, step); }
    static __device__ __forceinline__ void load_guarded(Raw& w, const Rows& r, int step, int K) { Tile::load_guarded(w, r, step, K); }
    static __device__ __forceinline__ void turn(typename T::frag (&f)[4], const Raw& w, const Rows&, int, uint4_t* lds)
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
    static __device__ __forceinline__ void turn(typename T::frag (&f)[4], const Raw&, const Rows& r, int step, uint4_t*)
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
template <class T, class W, class X, int RT, int TT, int U, class R>
__device__ __forceinline__ void skinny_sum(float4_t (&acc)[RT][TT], const typename W::Rows (&w)[RT], const typename X::Rows (&x)[TT], int K, int first, int stride,
                                           uint4_t* lds, R ready)
{
    typedef typename T::frag frag;
    constexpr int S = W::kUnit / kSkinnyStep;  // steps of a unit
    const int whole = K / W::kUnit;
    const int mine = first < whole ? (whole - first + stride - 1) / stride : 0;  // this wavefront's whole units
    typename W::Raw wv[U][RT];
    typename X::Raw xv[U][S][TT];
    auto ask = [&](int u, int n) {
        const int unit = first + n * stride;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < TT; ++j) X::load(xv[u][s][j], x[j], unit * S + s);
#pragma unroll
        for (int i = 0; i < RT; ++i) W::load(wv[u][i], w[i], unit);
    };
    auto products = [&](const typename W::Raw(&wr)[RT], const typename X::Raw(&xr)[S][TT], int unit) {
        typename W::Operands a[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) W::turn(a[i], wr[i], w[i], lds);
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                frag f[4];
                X::turn(f, xr[s][j], x[j], unit * S + s, lds + W::kLds);
#pragma unroll
                for (int o = 0; o < 4; ++o)
#pragma unroll
                    for (int i = 0; i < RT; ++i) acc[i][j] = T::mfma(W::operand(a[i], s, o), f[o], acc[i][j]);
            }
    };
    // The loop without conditions lets the compiler count loads exactly; what it leaves, fewer than 2 U units, goes by conditions.
    int n = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < mine) ask(u, u);
    ready();
    for (; n + 2 * U <= mine; n += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            products(wv[u], xv[u], first + (n + u) * stride);
            ask(u, n + U + u);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (n + u < mine) products(wv[u], xv[u], first + (n + u) * stride);
        if (n + U + u < mine) ask(u, n + U + u);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (n + U + u < mine) products(wv[u], xv[u], first + (n + U + u) * stride);
    // The unit that K ends in.
    if (K % W::kUnit != 0 && whole % stride == first) {
#pragma unroll
        for (int i = 0; i < RT; ++i) W::load_guarded(wv[0][i], w[i], whole, K);
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < TT; ++j) X::load_guarded(xv[0][s][j], x[j], whole * S + s, K);
        products(wv[0], xv[0], whole);
    }
}

// Sums of the WK wavefronts of a block, which shared k: tile (i, j) ends up in wavefront (i * TT + j) % WK.  `part` is
// WK * RT * TT * 64 vectors of LDS, which may be the memory the sums were made with.  The order of the sum is the wavefronts'.
template <int RT, int TT, int WK>
__device__ __forceinline__ void skinny_join(float4_t (&acc)[RT][TT], float4_t* part)
{
    if constexpr (WK > 1) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
}
}  // namespace pimhip
