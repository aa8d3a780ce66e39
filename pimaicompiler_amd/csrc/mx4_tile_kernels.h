// Products of many tokens with 4-bit weights: tiles of the result, operands through LDS.
#pragma once

#include "mx4_kernels.h"

namespace pimhip
{
// Tile `id` of a product.  Consecutive blocks go to consecutive XCDs, each with an L2 of its own, so an XCD gets a run of tiles: down
// a band of eight token tiles first, then to the next weights.  The 32 tiles that an XCD has at work at a time are about as high as
// wide, so they bring the fewest rows into its L2.
__device__ __forceinline__ void tile_at(int id, int tiles_n, int tiles_t, int64_t& n, int64_t& t)
{
    constexpr int kXcds = 8, kBand = 8;
    const int all = tiles_n * tiles_t, per = all / kXcds, more = all % kXcds, xcd = id % kXcds;
    const int at = xcd * per + (xcd < more ? xcd : more) + id / kXcds;
    const int band = at / (kBand * tiles_n), high = tiles_t - band * kBand < kBand ? tiles_t - band * kBand : kBand;
    const int in = at - band * kBand * tiles_n;
    n = in / high;
    t = band * kBand + in % high;
}

// ---- x in 16 bits, weights in 4 ----------------------------------------------------------------------------------------------
// A block has 16 GN WN rows of weights and 16 GT WT tokens, a wavefront of its GN x GT ones WN x WT tiles of 16 x 16.  Steps of 128 values
// of k, which KS groups of wavefronts take in turn.  Weights stay packed in LDS and are converted on the way to the matrix cores: a quarter of the LDS reads of converted ones.  One
// buffer: the next step's operands wait in registers.  Loads take whole runs of a row (16 lanes in 16 rows would be 16 requests), and a
// row's 16-byte chunks lie in LDS in an order that spreads what 8 lanes read or write over all banks.
//
// 4096 x 16384 x 4096: 528 us, 1.04 PFLOP/s; 1500 x 4096 x 4096: 63 us, 0.80 (this card's library multiplies 16-bit matrices of 8192 at 1.27
// to 1.5).  A block alone takes 1.9 us a step of 256 x 128 x 128: the matrix cores work 0.9 of it, the conversions, one instruction a
// product, take issue slots, LDS is busy 0.75.  Measured and not better: two steps in registers (the same; three: spills), two buffers
// (512, but 1500 tokens 73), 128 rows and tokens and four wavefronts (565), 32 x 128 results a wavefront, half the conversions but twice
// the reads (570), products, reads and conversions told to take turns (594).
template <class T, int WN, int WT, int GN, int GT, int KS>
__global__ __launch_bounds__(64 * GN * GT * KS) void mx4_linear_tile_kernel(const typename T::elem* x, Mx4View w, const typename T::elem* bias, typename T::elem* out,
                                                                       int64_t ld_x, int64_t ld_out, int64_t M, int relu)
{
    constexpr int kThreads = 64 * GN * GT, kN = 16 * GN * WN, kT = 16 * GT * WT, kStep = 128;
    constexpr int kX = kT * 16 / kThreads;   // 16-byte chunks of x a thread brings each step
    constexpr int kW = kN * 4 / kThreads;    // blocks of weights
    static_assert(kX * kThreads == kT * 16 && kW * kThreads == kN * 4, "whole chunks a thread");
    typedef typename T::frag frag;
    // (for each of the KS groups of wavefronts, which take steps of k in turn)
    __shared__ uint4_t xs_[KS][kT * 16];  // chunk c of a row at c ^ (row % 8)
    __shared__ uint4_t ws_[KS][kN * 4];   // block c of a row at c ^ (row / 4 % 4)
    __shared__ float ss_[KS][4][kN];
    const int share = KS == 1 ? 0 : wave_in_block() / (GN * GT), wave = KS == 1 ? wave_in_block() : wave_in_block() % (GN * GT);
    uint4_t *xs = xs_[share], *ws = ws_[share];
    auto ss = ss_[share];
    const int tid = (int)threadIdx.x - share * kThreads, lane = tid & 63, group = lane >> 4, row = lane & 15;
    const int wn = wave % GN * WN, wt = wave / GN * WT;
    int64_t tile_n, tile_t;
    tile_at(blockIdx.x, (int)((w.rows + kN - 1) / kN), (int)((M + kT - 1) / kT), tile_n, tile_t);
    const int64_t n0 = tile_n * kN, t0 = tile_t * kT, K = w.cols;
    const int blocks = (int)((K + kMxBlock - 1) / kMxBlock);

    const typename T::elem* xp[kX];
    const int xc = tid % 16;
#pragma unroll
    for (int i = 0; i < kX; ++i) {
        const int64_t t = t0 + (tid + i * kThreads) / 16;
        xp[i] = x + (t < M ? t : M - 1) * ld_x;
    }
    const uint8_t *wp[kW], *sp[kW];
    int top[kW];
    const int wc = tid % 4;
#pragma unroll
    for (int i = 0; i < kW; ++i) {
        int64_t n = n0 + (tid + i * kThreads) / 4;
        n = n < w.rows ? n : w.rows - 1;
        wp[i] = w.packed + (n * blocks + wc) * kMxBlockBytes;
        sp[i] = w.scales + n * w.ld_scales + wc;
        top[i] = w.tops[n];
    }
    frag xv[kX];
    uint4_t wv[kW];
    unsigned int code[kW];
    auto fetch = [&](int step) {
        const int64_t k0 = (int64_t)step * kStep;
        if (k0 + kStep <= K) {
#pragma unroll
            for (int i = 0; i < kX; ++i) xv[i] = load8_any<T>(xp[i] + k0 + xc * 8);
        } else {
#pragma unroll
            for (int i = 0; i < kX; ++i) xv[i] = load8_guarded<T>(xp[i], k0 + xc * 8, K);
        }
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            wv[i] = uint4_t{0, 0, 0, 0};
            code[i] = 0;  // (above no row's top)
            if (step * 4 + wc < blocks) {
                wv[i] = *reinterpret_cast<const uint4_t*>(wp[i] + (int64_t)step * (4 * kMxBlockBytes));
                code[i] = sp[i][step * 4];
            }
        }
    };
    float4_t acc[WN][WT] = {};
    const int steps = (int)((K + kStep - 1) / kStep);
    if (share < steps) fetch(share);
    for (int s0 = 0; s0 < steps; s0 += KS) {
        const int s = s0 + share;
        if (s0) __syncthreads();
        if (s < steps) {
#pragma unroll
            for (int i = 0; i < kX; ++i) {
                const int r = (tid + i * kThreads) / 16;
                xs[r * 16 + (xc ^ (r & 7))] = __builtin_bit_cast(uint4_t, xv[i]);
            }
#pragma unroll
            for (int i = 0; i < kW; ++i) {
                const int r = (tid + i * kThreads) / 4;
                ws[r * 4 + (wc ^ (r / 4 & 3))] = wv[i];
                ss[wc][r] = T::scale(code[i], top[i]);
            }
        }
        __syncthreads();
        if (s >= steps) continue;
        if (s + KS < steps) fetch(s + KS);
        uint4_t wq[WN];
        float scale[WN];
#pragma unroll
        for (int i = 0; i < WN; ++i) {
            const int r = (wn + i) * 16 + row;
            wq[i] = ws[r * 4 + (group ^ (r / 4 & 3))];
            scale[i] = ss[group][r];
        }
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            frag xf[WT];
#pragma unroll
            for (int j = 0; j < WT; ++j) {
                const int r = (wt + j) * 16 + row;
                xf[j] = __builtin_bit_cast(frag, xs[r * 16 + ((group * 4 + o) ^ (r & 7))]);
            }
#pragma unroll
            for (int i = 0; i < WN; ++i) {
                const frag wf = T::from_mx4(wq[i][o], scale[i]);
#pragma unroll
                for (int j = 0; j < WT; ++j) acc[i][j] = T::mfma(wf, xf[j], acc[i][j]);
            }
        }
    }
    if constexpr (KS > 1) {
        // The groups' sums, in their order.
        static_assert((KS - 1) * GN * GT * WN * WT * 64 <= KS * kT * 16, "the sums fit where the tokens were");
        float4_t* sums = reinterpret_cast<float4_t*>(xs_);
        __syncthreads();
        if (share > 0) {
#pragma unroll
            for (int i = 0; i < WN; ++i)
#pragma unroll
                for (int j = 0; j < WT; ++j) sums[((((share - 1) * GN * GT + wave) * WN + i) * WT + j) * 64 + lane] = acc[i][j];
        }
        __syncthreads();
        if (share > 0) return;
#pragma unroll
        for (int k = 0; k < KS - 1; ++k)
#pragma unroll
            for (int i = 0; i < WN; ++i)
#pragma unroll
                for (int j = 0; j < WT; ++j) acc[i][j] += sums[(((k * GN * GT + wave) * WN + i) * WT + j) * 64 + lane];
    }
#pragma unroll
    for (int i = 0; i < WN; ++i) {
        const int64_t n = n0 + (wn + i) * 16 + group * 4;
        if (n >= w.rows) continue;
        const int count = w.rows - n < 4 ? (int)(w.rows - n) : 4;
        int exponent[4] = {};
        float add[4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < count) {
                exponent[c] = T::exponent(w.tops[n + c]);
                if (bias) add[c] = (float)bias[n + c];
            }
#pragma unroll
        for (int j = 0; j < WT; ++j) {
            const int64_t t = t0 + (wt + j) * 16 + row;
            if (t >= M) continue;
            float4_t v = acc[i][j];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[c] = __builtin_amdgcn_ldexpf(v[c], exponent[c]);
                if (bias) v[c] += add[c];
                if (relu) v[c] = relu_f32(v[c]);
            }
            store4<T>(out + t * ld_out + n, v, count);
        }
    }
}

// ---- both operands in 4 bits -------------------------------------------------------------------------------------------------
// 128 x 128 results a block, a wavefront 64 x 64; steps of 256 values of k: the 128 bytes of a row that are a cache line, two products
// (v_mfma_scale_f32_16x16x128_f8f6f4) a tile.  A lane holds one block of each operand and its scale code.  A step goes from memory
// straight into LDS while the one before is multiplied, operands go from LDS to registers a product ahead, and two blocks of a CU fill
// each other's waits.
//
// 4096 x 16384 x 4096: 177 us, 3.1 PFLOP/s (a loop of the instruction alone reaches 7 to 8.8 here).  Two of these blocks' steps take
// 1.4 us, of which the matrix cores work 0.5 and LDS is read and written 0.7: what is left waits for a step to arrive, which takes a
// microsecond, and LDS holds no more steps.  Measured besides: steps of 128 values, three or four on their way, 227 (half a line is
// a whole request); 256 x 256 results a block, one block a CU, 198 with steps of 128, 226 with steps of 256, and slower by half and
// more where blocks are few; each code word loaded with its step 301 (a row's code is a request, however few bytes it has); k begun in another place by each column of tiles
// the same, and 181 instead of 165 for 4096 x 4096 x 16384 (rows that blocks have in common then leave the L2 before all have read them).
template <class O>
__global__ __launch_bounds__(256, 2) void mx4_matmul_tile_kernel(Mx4View a, Mx4View b, typename O::elem* out, int64_t ld_out)
{
    constexpr int kTile = 128, kRows = 2 * kTile, kPieces = 8;  // (a wavefront brings 64 rows, a load 128 bytes of eight)
    constexpr int kBuffer = kRows * 128, kCodes = kRows * 16;
    // A step: the rows of b, then those of a, block c of row r at c ^ turned(r).  16 lanes of a read have 16 different places of two rows'
    // 256 bytes, whether their rows follow each other or skip four of eight.  Codes come for two steps at a time.
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kBuffer + 2 * kCodes];
    auto turned = [](int r) { return (r >> 1 ^ (r >> 3 & 2)) & 7; };
    // The rows that lane `l` multiplies in tile i of four.  Two tiles of weights take turns, four and four: a lane then has eight neighbours
    // of a row of the result.
    auto weight_row = [](int l, int i) { return (i & 2) * 16 + l / 4 * 8 + (i & 1) * 4 + l % 4; };
    auto token_row = [](int l, int i) { return i * 16 + l; };
    const int lane = threadIdx.x & 63, wave = wave_in_block(), group = lane >> 4, row = lane & 15;
    const int wn = wave % 2 * 64, wt = wave / 2 * 64;
    int64_t tile_n, tile_t;
    tile_at(blockIdx.x, (int)((b.rows + kTile - 1) / kTile), (int)((a.rows + kTile - 1) / kTile), tile_n, tile_t);
    const int64_t n0 = tile_n * kTile, t0 = tile_t * kTile;
    const int blocks = (int)((b.cols + kMxBlock - 1) / kMxBlock), whole = blocks / 8;

    // A wavefront brings rows of one matrix, from `from` on; those behind its end are its last one again.
    const bool weights = wave < 2;
    const Mx4View& m = weights ? b : a;
    const int64_t first = weights ? n0 + wave * 64 : t0 + wave * 64 - kTile, from = first < m.rows ? first : m.rows - 1;
    const int most = (int)(m.rows - 1 - from < 63 ? m.rows - 1 - from : 63);
    const uint8_t *vp = m.packed + from * blocks * kMxBlockBytes, *cp = m.scales + from * m.ld_scales;
    unsigned int v_at[kPieces], c_at;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int r = i * 8 + lane / 8;
        v_at[i] = (unsigned int)((r < most ? r : most) * blocks + ((lane & 7) ^ turned(r))) * kMxBlockBytes;
    }
    const int c_row = weights ? weight_row(row, group) : token_row(row, group);
    c_at = (unsigned int)(c_row < most ? c_row : most) * (unsigned int)m.ld_scales;
    const unsigned int lds0 = (unsigned int)(size_t)(__attribute__((address_space(3))) uint8_t*)lds;
    auto fetch = [&](int step) __attribute__((always_inline)) {
        if (step % 2 == 0) load_lds16(cp + step * 8, c_at, lds0 + 2 * kBuffer + (unsigned int)(step / 2 % 2) * kCodes + (unsigned int)wave * 1024u);
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            load_lds16(vp + (int64_t)step * (8 * kMxBlockBytes), v_at[i], lds0 + (unsigned int)(step % 2) * kBuffer + (unsigned int)(wave * kPieces + i) * 1024u);
    };

    struct Part {  // four tiles' operands, and their codes (byte `group` of what is read) in one register
        uint4_t v[4];
        unsigned int c;
    };
    const unsigned int pick = 0x0c0c0000u | (unsigned int)(group | (group + 4) << 8);  // (0x0c: a byte of zeros)
    const int p_at[2] = {((wn + weight_row(row, 0)) * 8 + (group ^ turned(weight_row(row, 0)))) * 16,
                         ((wn + weight_row(row, 1)) * 8 + (group ^ turned(weight_row(row, 1)))) * 16};
    const int t_at[2] = {((kTile + wt + row) * 8 + (group ^ turned(row))) * 16, ((kTile + wt + 16 + row) * 8 + (group ^ turned(16 + row))) * 16};
    const int pc_at = 2 * kBuffer + (wn + row) * 16, tc_at = 2 * kBuffer + (kTile + wt + row) * 16;
    Part p[2], t[2];
    // Operands of half `half` of a step's k.
    auto read = [&](int step, int half) __attribute__((always_inline)) {
        const int base = step % 2 * kBuffer, word = (step / 2 % 2) * kCodes + (step % 2 * 2 + half) * 4;
        auto part = [&](Part& x, const int(&at)[2], int c_at) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x.v[i] = *reinterpret_cast<const uint4_t*>(lds + base + (at[i & 1] ^ half * 64) + (i & 2) * 2048);
            const unsigned int* q = reinterpret_cast<const unsigned int*>(lds + c_at + word);
            x.c = __builtin_amdgcn_perm(q[64], q[0], pick) | __builtin_amdgcn_perm(q[192], q[128], pick) << 16;
        };
        part(t[half], t_at, tc_at);
        part(p[half], p_at, pc_at);
    };
    float4_t acc[4][4] = {};
    auto multiply = [&](const Part& p, const Part& t) __attribute__((always_inline)) {
        auto wide = [](const uint4_t& q) { return int8v_t{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0}; };
        // (which byte of the codes is part of the instruction)
#define PIMHIP_MX4_STEP(i, j) \
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(p.v[i]), wide(t.v[j]), acc[i][j], 4, 4, i, (int)p.c, j, (int)t.c)
#define PIMHIP_MX4_STEPS(i) PIMHIP_MX4_STEP(i, 0), PIMHIP_MX4_STEP(i, 1), PIMHIP_MX4_STEP(i, 2), PIMHIP_MX4_STEP(i, 3)
        PIMHIP_MX4_STEPS(0), PIMHIP_MX4_STEPS(1), PIMHIP_MX4_STEPS(2), PIMHIP_MX4_STEPS(3);
#undef PIMHIP_MX4_STEPS
#undef PIMHIP_MX4_STEP
    };
    // Half of a step, while the operands of the next half are read, if there is one.
    auto product = [&](int step, int half, bool next) __attribute__((always_inline)) {
        if (next) {
            if (half == 1) {  // everybody has read the step, and the next one is there
                wait_loads_and_barrier<0>();
                if (step + 2 < whole) fetch(step + 2);
            }
            read(step + half, half ^ 1);
        }
        __builtin_amdgcn_sched_barrier(0);  // (the reads stay before the products that they run under)
        multiply(p[half], t[half]);
    };

    if (whole > 0) {
        fetch(0);
        if (whole > 1) {
            fetch(1);
            wait_loads_and_barrier<kPieces>();  // (those of the second step)
        } else {
            wait_loads_and_barrier<0>();
        }
        read(0, 0);
        int s = 0;
        for (; s + 1 < whole; ++s) {
            product(s, 0, true);
            product(s, 1, true);
        }
        product(s, 0, true);
        product(s, 1, false);
        __syncthreads();
    }
    if (blocks % 8 != 0) {
        // The step that K ends in, by way of registers: behind the end zeros, and any code but "not a number".
        const int left = blocks - whole * 8;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            uint4_t q = {0, 0, 0, 0};
            if (((lane & 7) ^ turned(i * 8 + lane / 8)) < left) q = *reinterpret_cast<const uint4_t*>(vp + (int64_t)whole * (8 * kMxBlockBytes) + v_at[i]);
            *reinterpret_cast<uint4_t*>(lds + (wave * kPieces + i) * 1024 + lane * 16) = q;
        }
        const uint64_t in = ((uint64_t)1 << (8 * left)) - 1;
        *reinterpret_cast<uint64_t*>(lds + 2 * kBuffer + wave * 1024 + lane * 16) =
            (*reinterpret_cast<const uint64_t*>(cp + whole * 8 + c_at) & in) | (0x7f7f7f7f7f7f7f7full & ~in);
        __syncthreads();
        read(0, 0);
        product(0, 0, true);
        product(0, 1, false);
    }

    const int64_t n = n0 + wn + group * 8, t_row = t0 + wt + row;
    typename O::elem* to = out + t_row * ld_out + n;
    if (n0 + kTile <= b.rows && t0 + kTile <= a.rows) {
#pragma unroll
        for (int j = 0; j < 4; ++j, to += 16 * ld_out)
#pragma unroll
            for (int i = 0; i < 4; i += 2) store8<O>(to + i * 16, acc[i][j], acc[i + 1][j]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j, to += 16 * ld_out) {
        if (t_row + j * 16 >= a.rows) continue;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const int64_t left = b.rows - n - i * 16;
            if (left >= 8) {
                store8<O>(to + i * 16, acc[i][j], acc[i + 1][j]);
            } else if (left > 0) {
                store4<O>(to + i * 16, acc[i][j], (int)left);
                store4<O>(to + i * 16 + 4, acc[i + 1][j], (int)left - 4);
            }
        }
    }
}
}  // namespace pimhip
