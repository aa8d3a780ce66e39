// Products of many tokens with 4-bit weights: tiles of the result, operands through LDS.
//
// A block has 16 GN WN rows of weights and 16 GT WT tokens, a wavefront of its GN x GT ones WN x WT tiles of 16 x 16.  The next
// step's operands are on their way to registers while the matrix cores work on this one's in LDS (two buffers, one barrier a step).
// Loads take whole runs of a row (16 lanes in 16 rows would be 16 requests), and a row's 16-byte chunks lie in LDS in an order that
// spreads what 8 lanes read or write over all banks.
#pragma once

#include "mx4_kernels.h"

namespace pimhip
{
// Which tile a block has: consecutive blocks go to consecutive XCDs, each with an L2 of its own, so an XCD gets a run of tiles, down
// a column of tokens first: they share the weights' rows.
__device__ __forceinline__ void tile_of_block(int64_t tiles_n, int64_t tiles_t, int64_t& n, int64_t& t)
{
    constexpr int64_t kXcds = 8;
    const int64_t all = tiles_n * tiles_t, id = blockIdx.x;
    const int64_t per = all / kXcds, more = all % kXcds, xcd = id % kXcds;
    const int64_t at = xcd * per + (xcd < more ? xcd : more) + id / kXcds;
    n = at / tiles_t;
    t = at % tiles_t;
}

// ---- x in 16 bits, weights in 4 ----------------------------------------------------------------------------------------------
// Steps of 128 values of k.  Weights stay packed in LDS and are converted on the way to the matrix cores: a quarter of the LDS reads of
// converted ones.  One buffer: the next step's operands wait in registers, and while a block writes them another one of its CU
// computes.
template <class T, int WN, int WT, int GN, int GT>
__global__ __launch_bounds__(64 * GN * GT) void mx4_linear_tile_kernel(const typename T::elem* x, Mx4View w, const typename T::elem* bias, typename T::elem* out,
                                                                       int64_t ld_x, int64_t ld_out, int64_t M, int relu)
{
    constexpr int kThreads = 64 * GN * GT, kN = 16 * GN * WN, kT = 16 * GT * WT, kStep = 128;
    constexpr int kX = kT * 16 / kThreads;   // 16-byte chunks of x a thread brings each step
    constexpr int kW = kN * 4 / kThreads;    // blocks of weights
    static_assert(kX * kThreads == kT * 16 && kW * kThreads == kN * 4, "whole chunks a thread");
    typedef typename T::frag frag;
    __shared__ uint4_t xs[kT * 16];  // chunk c of a row at c ^ (row % 8)
    __shared__ uint4_t ws[kN * 4];   // block c of a row at c ^ (row / 4 % 4)
    __shared__ float ss[4][kN];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_in_block(), group = lane >> 4, row = lane & 15;
    const int wn = wave % GN * WN, wt = wave / GN * WT;
    int64_t tile_n, tile_t;
    tile_of_block((w.rows + kN - 1) / kN, (M + kT - 1) / kT, tile_n, tile_t);
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
            code[i] = 127;
            if (step * 4 + wc < blocks) {
                wv[i] = *reinterpret_cast<const uint4_t*>(wp[i] + (int64_t)step * (4 * kMxBlockBytes));
                code[i] = sp[i][step * 4];
            }
        }
    };
    float4_t acc[WN][WT] = {};
    const int steps = (int)((K + kStep - 1) / kStep);
    fetch(0);
    for (int s = 0; s < steps; ++s) {
        if (s) __syncthreads();
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
        __syncthreads();
        if (s + 1 < steps) fetch(s + 1);
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
#pragma unroll
    for (int i = 0; i < WN; ++i) {
        const int64_t n = n0 + (wn + i) * 16 + group * 4;
        if (n >= w.rows) continue;
        const int count = w.rows - n < 4 ? (int)(w.rows - n) : 4;
        int tops[4] = {};
        float add[4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < count) {
                tops[c] = w.tops[n + c];
                if (bias) add[c] = (float)bias[n + c];
            }
#pragma unroll
        for (int j = 0; j < WT; ++j) {
            const int64_t t = t0 + (wt + j) * 16 + row;
            if (t >= M) continue;
            float4_t v = acc[i][j];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[c] = T::unscale(v[c], tops[c]);
                if (bias) v[c] += add[c];
                if (relu) v[c] = relu_f32(v[c]);
            }
            store4<T>(out + t * ld_out + n, v, count);
        }
    }
}

// ---- both operands in 4 bits -------------------------------------------------------------------------------------------------
// Steps of 128 values of k, one product (v_mfma_scale_f32_16x16x128_f8f6f4) a tile: a lane holds one block of each operand.  The scale
// codes of four tiles' blocks share a 32-bit word of LDS; the instruction picks its byte.
template <class O, int WN, int WT, int GN, int GT>
__global__ __launch_bounds__(64 * GN * GT) void mx4_matmul_tile_kernel(Mx4View a, Mx4View b, typename O::elem* out, int64_t ld_out)
{
    constexpr int kThreads = 64 * GN * GT, kN = 16 * GN * WN, kT = 16 * GT * WT, kRows = kN + kT;
    constexpr int kPieces = kRows * 4 / kThreads;  // blocks of either operand a thread brings each step
    static_assert(kPieces * kThreads == kRows * 4 && kRows <= kThreads && WN % 4 == 0 && WT % 4 == 0, "whole pieces a thread, a row of scales each");
    __shared__ uint4_t values[2][kRows * 4];            // the rows of b, then those of a; block c of a row at c ^ (row / 4 % 4)
    __shared__ unsigned int codes[2][kRows / 64][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_in_block(), group = lane >> 4, row = lane & 15;
    const int wn = wave % GN * WN, wt = wave / GN * WT;
    int64_t tile_n, tile_t;
    tile_of_block((b.rows + kN - 1) / kN, (a.rows + kT - 1) / kT, tile_n, tile_t);
    const int64_t n0 = tile_n * kN, t0 = tile_t * kT;
    const int blocks = (int)((b.cols + kMxBlock - 1) / kMxBlock);
    // Row r of the tile: its matrix, and its row there (the last one again behind the end).
    const uint8_t* vp[kPieces];
    const int vb = tid % 4;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int r = (tid + i * kThreads) / 4;
        const int64_t last = (r < kN ? b.rows : a.rows) - 1, at = r < kN ? n0 + r : t0 + r - kN;
        vp[i] = (r < kN ? b.packed : a.packed) + ((at < last ? at : last) * blocks + vb) * kMxBlockBytes;
    }
    const uint8_t* cp = nullptr;
    if (tid < kRows) {
        const int64_t last = (tid < kN ? b.rows : a.rows) - 1, at = tid < kN ? n0 + tid : t0 + tid - kN;
        cp = (tid < kN ? b.scales : a.scales) + (at < last ? at : last) * (tid < kN ? b.ld_scales : a.ld_scales);
    }
    uint4_t v[kPieces];
    unsigned int c = 0;
    auto fetch = [&](int step) {
        if (step * 4 + 4 <= blocks) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) v[i] = *reinterpret_cast<const uint4_t*>(vp[i] + (int64_t)step * (4 * kMxBlockBytes));
            if (tid < kRows) c = *reinterpret_cast<const unsigned int*>(cp + step * 4);
        } else {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                v[i] = uint4_t{0, 0, 0, 0};
                if (step * 4 + vb < blocks) v[i] = *reinterpret_cast<const uint4_t*>(vp[i] + (int64_t)step * (4 * kMxBlockBytes));
            }
            // (whole groups of 16 codes a row) Behind the row's last block: any code but "not a number".
            if (tid < kRows) {
                c = *reinterpret_cast<const unsigned int*>(cp + step * 4);
                const unsigned int in = (1u << (8 * (blocks - step * 4))) - 1;
                c = (c & in) | (0x7f7f7f7fu & ~in);
            }
        }
    };
    auto put = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int r = (tid + i * kThreads) / 4;
            values[buffer][r * 4 + (vb ^ (r / 4 & 3))] = v[i];
        }
        if (tid < kRows) {
            uint8_t* to = reinterpret_cast<uint8_t*>(&codes[buffer][tid / 64][tid % 16]) + tid / 16 % 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i * 64] = (uint8_t)(c >> (8 * i));
        }
    };
    float4_t acc[WN][WT] = {};
    const int steps = (blocks + 3) / 4;
    fetch(0);
    put(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const int buffer = s & 1;
        if (s + 1 < steps) fetch(s + 1);
        int8v_t af[WT];
        int ac[WT / 4];
#pragma unroll
        for (int j = 0; j < WT; ++j) {
            const uint4_t q = values[buffer][(kN + (wt + j) * 16 + row) * 4 + (group ^ (row / 4))];
            af[j] = int8v_t{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < WT / 4; ++j) ac[j] = (int)codes[buffer][kN / 64 + wt / 4 + j][lane];
#define PIMHIP_MX_PRODUCT(I, J) \
    acc[i4 + I][j4 * 4 + J] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[I], af[j4 * 4 + J], acc[i4 + I][j4 * 4 + J], 4, 4, I, bc, J, ac[j4]);
#define PIMHIP_MX_ROW(I) PIMHIP_MX_PRODUCT(I, 0) PIMHIP_MX_PRODUCT(I, 1) PIMHIP_MX_PRODUCT(I, 2) PIMHIP_MX_PRODUCT(I, 3)
#pragma unroll
        for (int i4 = 0; i4 < WN; i4 += 4) {
            int8v_t bf[4];
            const int bc = (int)codes[buffer][(wn + i4) / 4][lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4_t q = values[buffer][((wn + i4 + i) * 16 + row) * 4 + (group ^ (row / 4))];
                bf[i] = int8v_t{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
            }
#pragma unroll
            for (int j4 = 0; j4 < WT / 4; ++j4) {
                PIMHIP_MX_ROW(0)
                PIMHIP_MX_ROW(1)
                PIMHIP_MX_ROW(2)
                PIMHIP_MX_ROW(3)
            }
        }
#undef PIMHIP_MX_ROW
#undef PIMHIP_MX_PRODUCT
        if (s + 1 < steps) put(buffer ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < WN; ++i) {
        const int64_t n = n0 + (wn + i) * 16 + group * 4;
        if (n >= b.rows) continue;
#pragma unroll
        for (int j = 0; j < WT; ++j) {
            const int64_t t = t0 + (wt + j) * 16 + row;
            if (t < a.rows) store4<O>(out + t * ld_out + n, acc[i][j], b.rows - n < 4 ? (int)(b.rows - n) : 4);
        }
    }
}
}  // namespace pimhip
