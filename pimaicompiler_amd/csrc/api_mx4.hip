// Microscaled 4-bit matrices of the C ABI (include/pimhip.h): quantisation, reading back, and the products with one or both operands in 4 bits.
#include "api_common.h"
#include "mx4_tile_kernels.h"

using namespace pimhip;

namespace
{
constexpr int64_t kMaxCols = 1 << 26;  // (64 rows' bytes are counted in 32 bits)

int check_matrix(const char* name, const PimHipMx4Matrix* m, Mx4View* v)
{
    if (!m) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "%s is null", name);
    if (m->rows < 0 || m->cols < 1 || m->cols > kMaxCols)
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "%s: rows=%lld, cols=%lld (cols in [1, %lld])", name, (long long)m->rows, (long long)m->cols, (long long)kMaxCols);
    const int64_t blocks = (m->cols + kMxBlock - 1) / kMxBlock;
    if (m->ld_scales < blocks || m->ld_scales > kMaxCols || (m->ld_scales & 15))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "%s: ld_scales=%lld must be a multiple of 16 in [%lld, %lld]", name, (long long)m->ld_scales, (long long)blocks,
                    (long long)kMaxCols);
    if (m->rows && (!m->packed || !m->scales || !m->tops)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "%s: packed, scales and tops must be non-null", name);
    if (!aligned16(m->packed) || !aligned16(m->scales)) return fail(PIMHIP_ERR_UNSUPPORTED, "%s: packed and scales must be 16-byte aligned", name);
    *v = Mx4View{(const uint8_t*)m->packed, (const uint8_t*)m->scales, (const uint8_t*)m->tops, m->rows, m->cols, m->ld_scales};
    return PIMHIP_OK;
}

int check_element(const char* name, const void* p, int dtype, bool fp32_too)
{
    if (dtype != PIMHIP_F16 && dtype != PIMHIP_BF16 && !(fp32_too && dtype == PIMHIP_F32)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "dtype=%d", dtype);
    if (!p) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "%s is null", name);
    if (reinterpret_cast<uintptr_t>(p) & (dtype == PIMHIP_F32 ? 3u : 1u)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "%s is not aligned to its elements", name);
    return PIMHIP_OK;
}

// A launch's workgroups, and its threads, which are counted in 32 bits along x.
int check_grid(int64_t x, int64_t y, int threads)
{
    if (x > INT32_MAX || x * threads > UINT32_MAX || y > 65535)
        return fail(PIMHIP_ERR_UNSUPPORTED, "too large for one launch (%lld x %lld workgroups of %d threads)", (long long)x, (long long)y, threads);
    return PIMHIP_OK;
}

// LDS of a launch's staged tokens, in bytes.
template <class T>
int64_t shared_tokens_bytes(int64_t M, int64_t K)
{
    return M * SharedTokens<T>::pitch((int)K, Mx4Weights<T, 2>::kUnit) * 16;
}

template <class T, bool SHARED, int RT, int TT, int WK>
int linear_skinny(void* out, int64_t ld_out, const void* x, int64_t ld_x, int64_t M, const Mx4View& w, const void* bias, int relu, hipStream_t s)
{
    const int64_t gx = (w.rows + 16 * RT - 1) / (16 * RT), gy = (M + 16 * TT - 1) / (16 * TT);
    const int rc = check_grid(gx, gy, 64 * WK);
    if (rc != PIMHIP_OK) return rc;
    mx4_linear_skinny_kernel<T, SHARED, RT, TT, WK><<<dim3((unsigned)gx, (unsigned)gy), 64 * WK, SHARED ? shared_tokens_bytes<T>(M, w.cols) : 0, s>>>(
        (const typename T::elem*)x, w, (const typename T::elem*)bias, (typename T::elem*)out, ld_x, ld_out, M, relu);
    return PIMHIP_OK;
}

template <class T>
int linear(void* out, int64_t ld_out, const void* x, int64_t ld_x, int64_t M, const Mx4View& w, const void* bias, int relu, hipStream_t s)
{
    // Rows a wavefront has at a time, and wavefronts that share k.  More rows read x less often but make fewer blocks, more wavefronts
    // the opposite.  Measured on 16384 x 4096 / 4096 x 4096 / 31999 x 1024, weights that no cache holds, in us:
    //   one token (staged in LDS)   1 tile of 16 rows, 8 wavefronts 10.5 / 4.9 / -      2 tiles, 8: 8.7 / 5.9 / -     (turned by the wavefronts: 12.0 / 5.6)
    //   16 tokens                   1 tile, 8: 16.1 / 6.3 / 12.9      4 tiles, 8: 10.7 / 9.3 / 10.5      4 tiles, 4: 11.3 / 10.4 / 7.3
    //   32 tokens                   1 tile, 8: 24.1 / 8.6 / 17.4      4 tiles, 8: 16.1 / 14.6 / 12.8     4 tiles, 4: 16.8 / 15.7 / 10.0
    //   64 tokens, 32 a block       2 tiles, 8: 36.2 / 9.7 / 28.0     4 tiles, 8: 30.7 / - / -           4 tiles, 4: 27.1 / 15.3 / 19.2
    //   64 tokens, 64 a block       1 tile, 8: 45.3 / 12.5 / 39.9     2 tiles, 8: 28.5 / 14.3 / 25.7     4 tiles, 4: 23.9 / 22.2 / 20.6
    constexpr int64_t kShared = 32 << 10;
    const int64_t tiles16 = (w.rows + 15) / 16;
    const bool long_rows = w.cols > 4 * Mx4Weights<T, 2>::kUnit;
    auto go = [&](auto kernel) { return kernel(out, ld_out, x, ld_x, M, w, bias, relu, s); };
    if (M <= 2 && shared_tokens_bytes<T>(M, w.cols) <= kShared) {
        if (tiles16 < 768) return long_rows ? go(linear_skinny<T, true, 1, 1, 8>) : go(linear_skinny<T, true, 1, 1, 4>);
        return long_rows ? go(linear_skinny<T, true, 2, 1, 8>) : go(linear_skinny<T, true, 2, 1, 4>);
    }
    if (M <= 16) {
        if (tiles16 < 512) return long_rows ? go(linear_skinny<T, false, 1, 1, 8>) : go(linear_skinny<T, false, 1, 1, 4>);
        return long_rows ? go(linear_skinny<T, false, 4, 1, 8>) : go(linear_skinny<T, false, 4, 1, 4>);
    }
    if (M <= 64) {
        if (tiles16 <= 512) return M <= 32 ? go(linear_skinny<T, false, 1, 2, 8>) : go(linear_skinny<T, false, 2, 2, 8>);
        if (!long_rows) return go(linear_skinny<T, false, 4, 2, 4>);
        return M <= 32 ? go(linear_skinny<T, false, 4, 2, 8>) : go(linear_skinny<T, false, 4, 4, 4>);
    }
    // Large tiles read operands less often, small ones fill the card.  Measured, 256 x 128 / 128 x 64, in us: 4096 x 16384 x 4096 532 / 634,
    // 2048 x 4096 x 4096 (256 large tiles) 70 / 86, 1500 x 4608 x 4096 (216) 68 / 84, 1500 x 4096 x 4096 (192) 68 / 65, 200 x 16384 x 4096 (128)
    // 67 / 48, 512 x 4096 x 4096 (64) 67 / 34.
    // The kernel of few tokens ends at 64, where a block of it does; that is not where tiles become faster.  Tiles / that kernel with more blocks of
    // tokens: 64 x 16384 x 4096 35 / 22, 65 x 16384 x 4096 32 / 43, 128 x 16384 x 4096 33 / 45, but 65 x 4096 x 4096 29 / 16, 128 x 4096 x 4096 29 / 17,
    // 200 x 4096 x 4096 29 / 30, 65 x 1024 x 1024 11.0 / 4.4, 512 x 512 x 4096 28 / 9.5, 300 x 300 x 14000 94 / 38, 65 x 17 x 16384 92 / 18: a tile does all of
    // its k in one block, so where tiles are far fewer than CUs the time is that of k, whatever the tokens.
    auto tiled = [&](auto kernel, int rows, int tokens, int threads) {
        const int64_t tiles = ((w.rows + rows - 1) / rows) * ((M + tokens - 1) / tokens);
        const int rc = check_grid(tiles, 1, threads);
        if (rc != PIMHIP_OK) return rc;
        kernel<<<dim3((unsigned)tiles), threads, 0, s>>>((const typename T::elem*)x, w, (const typename T::elem*)bias, (typename T::elem*)out, ld_x, ld_out, M, relu);
        return (int)PIMHIP_OK;
    };
    if (((w.rows + 255) / 256) * ((M + 127) / 128) > 192) return tiled(mx4_linear_tile_kernel<T, 4, 4, 4, 2, 1>, 256, 128, 512);
    // Where every tile has a CU to itself, two groups of wavefronts share its k: 512 x 4096 x 4096 (256 tiles) 31 / 33 us with one group, 300 x 300 x
    // 14000 (15) 94 / 106, 200 x 16384 x 4096 (512) 55 / 48; four groups, 1024 threads: 39 for the first.
    if (((w.rows + 127) / 128) * ((M + 63) / 64) <= 256) return tiled(mx4_linear_tile_kernel<T, 4, 2, 2, 2, 2>, 128, 64, 512);
    return tiled(mx4_linear_tile_kernel<T, 4, 2, 2, 2, 1>, 128, 64, 256);
}

template <class O>
int matmul(void* out, int64_t ld_out, const Mx4View& a, const Mx4View& b, hipStream_t s)
{
    auto run = [&](auto kernel, int RT, int TT, int WK) {
        const int64_t gx = (b.rows + 16 * RT - 1) / (16 * RT), gy = (a.rows + 16 * TT - 1) / (16 * TT);
        const int rc = check_grid(gx, gy, 64 * WK);
        if (rc != PIMHIP_OK) return rc;
        kernel<<<dim3((unsigned)gx, (unsigned)gy), 64 * WK, 0, s>>>(a, b, (typename O::elem*)out, ld_out);
        return (int)PIMHIP_OK;
    };
    // Few rows of a: blocks of 16 to 64 rows of b whose wavefronts share k.  More rows read a less often, fewer make more blocks.  Measured, in us:
    //   16 x 16384 x 4096   16 rows 16.8, 64 rows 12.4      16 x 4096 x 4096   16 rows 5.9, 64 rows 11.4      1 x 4096 x 16384   16 rows 15.1, 64 rows 34
    // From 17 rows of a on, tiles of 128 x 128 (below) where b has 96 of them, else 32 rows of a a block:
    //   32 x 16384 x 4096   tiles 17.7, blocks 18.0      64 x 16384 x 4096   18.0 / 31.2      48 x 8192 x 1024 (64 tiles)   5.7 / 6.0      64 x 4096 x 4096   14.1 / 9.7
    if (a.rows <= 16)
        return (b.rows + 15) / 16 >= 1024 ? run(mx4_matmul_skinny_kernel<O, 4, 1, 8>, 4, 1, 8) : run(mx4_matmul_skinny_kernel<O, 1, 1, 8>, 1, 1, 8);
    const int64_t columns = (b.rows + 127) / 128;
    if (a.rows <= 64 && columns < 96) return a.rows <= 32 ? run(mx4_matmul_skinny_kernel<O, 1, 2, 8>, 1, 2, 8) : run(mx4_matmul_skinny_kernel<O, 2, 2, 8>, 2, 2, 8);
    const int64_t tiles = columns * ((a.rows + 127) / 128);
    const int rc = check_grid(tiles, 1, 256);
    if (rc != PIMHIP_OK) return rc;
    mx4_matmul_tile_kernel<O><<<dim3((unsigned)tiles), 256, 0, s>>>(a, b, (typename O::elem*)out, ld_out);
    return PIMHIP_OK;
}
}  // namespace

extern "C" int pimhip_mx4_quantize(const PimHipMx4Matrix* out, const void* x, int dtype, int64_t ld_x, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    Mx4View v;
    if ((rc = check_matrix("out", out, &v)) != PIMHIP_OK) return rc;
    if (v.rows == 0) return PIMHIP_OK;
    if ((rc = check_element("x", x, dtype, true)) != PIMHIP_OK) return rc;
    if (v.rows > 1 && ld_x < v.cols) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "ld_x=%lld is less than cols=%lld", (long long)ld_x, (long long)v.cols);
    // A row of up to 1024 values is one wavefront's (at most two rounds of 512), a longer one a block's.
    const bool short_rows = v.cols <= 1024;
    const int64_t grid = short_rows ? (v.rows + 3) / 4 : v.rows;
    if ((rc = check_grid(grid, 1, 256)) != PIMHIP_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto type) {
        typedef decltype(type) T;
        auto kernel = short_rows ? mx4_quantize_kernel<T, 1> : mx4_quantize_kernel<T, 4>;
        kernel<<<dim3((unsigned)grid), 256, 0, s>>>((const typename T::elem*)x, v.rows, v.cols, ld_x, (uint8_t*)out->packed, (uint8_t*)out->scales, v.ld_scales,
                                                    (uint8_t*)out->tops);
    };
    dtype == PIMHIP_F16 ? run(F16{}) : dtype == PIMHIP_BF16 ? run(BF16{}) : run(F32{});
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}

extern "C" int pimhip_mx4_find_tops(const PimHipMx4Matrix* m, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    Mx4View v;
    if ((rc = check_matrix("matrix", m, &v)) != PIMHIP_OK) return rc;
    if (v.rows == 0) return PIMHIP_OK;
    if ((rc = check_grid((v.rows + 3) / 4, 1, 256)) != PIMHIP_OK) return rc;
    mx4_tops_kernel<<<dim3((unsigned)((v.rows + 3) / 4)), 256, 0, static_cast<hipStream_t>(stream)>>>(v.scales, v.ld_scales, v.rows, (v.cols + kMxBlock - 1) / kMxBlock,
                                                                                                     (uint8_t*)m->tops);
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}

extern "C" int pimhip_mx4_dequantize(void* out, int dtype, int64_t ld_out, const PimHipMx4Matrix* m, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    Mx4View v;
    if ((rc = check_matrix("matrix", m, &v)) != PIMHIP_OK) return rc;
    if (v.rows == 0) return PIMHIP_OK;
    if ((rc = check_element("out", out, dtype, true)) != PIMHIP_OK) return rc;
    if (v.rows > 1 && ld_out < v.cols) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "ld_out=%lld is less than cols=%lld", (long long)ld_out, (long long)v.cols);
    const dim3 grid((unsigned)((v.cols + 2047) / 2048), (unsigned)(v.rows < 65535 ? v.rows : 65535));
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto type) {
        typedef decltype(type) T;
        mx4_dequantize_kernel<T><<<grid, 256, 0, s>>>(v.packed, v.scales, v.rows, v.cols, v.ld_scales, (typename T::elem*)out, ld_out);
    };
    dtype == PIMHIP_F16 ? run(F16{}) : dtype == PIMHIP_BF16 ? run(BF16{}) : run(F32{});
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}

extern "C" int pimhip_mx4_linear(void* out, int64_t ld_out, const void* x, int64_t ld_x, int dtype, int64_t tokens, const PimHipMx4Matrix* weight,
                                 const void* bias, int act, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    Mx4View w;
    if ((rc = check_matrix("weight", weight, &w)) != PIMHIP_OK) return rc;
    if (tokens < 0) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "tokens=%lld", (long long)tokens);
    if (act != PIMHIP_ACT_NONE && act != PIMHIP_ACT_RELU) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "act=%d", act);
    if (tokens == 0 || w.rows == 0) return PIMHIP_OK;
    if ((rc = check_element("x", x, dtype, false)) != PIMHIP_OK || (rc = check_element("out", out, dtype, false)) != PIMHIP_OK) return rc;
    if (bias && (rc = check_element("bias", bias, dtype, false)) != PIMHIP_OK) return rc;
    if (tokens > 1 && (ld_x < w.cols || ld_out < w.rows))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "ld_x=%lld is less than cols=%lld, or ld_out=%lld less than rows=%lld", (long long)ld_x, (long long)w.cols,
                    (long long)ld_out, (long long)w.rows);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int relu = act == PIMHIP_ACT_RELU;
    rc = dtype == PIMHIP_F16 ? linear<F16>(out, ld_out, x, ld_x, tokens, w, bias, relu, s) : linear<BF16>(out, ld_out, x, ld_x, tokens, w, bias, relu, s);
    if (rc != PIMHIP_OK) return rc;
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}

extern "C" int pimhip_mx4_matmul(void* out, int64_t ld_out, int dtype, const PimHipMx4Matrix* a, const PimHipMx4Matrix* b, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    Mx4View va, vb;
    if ((rc = check_matrix("a", a, &va)) != PIMHIP_OK || (rc = check_matrix("b", b, &vb)) != PIMHIP_OK) return rc;
    if (va.cols != vb.cols) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "a has %lld columns, b %lld", (long long)va.cols, (long long)vb.cols);
    if (va.rows == 0 || vb.rows == 0) return PIMHIP_OK;
    if ((rc = check_element("out", out, dtype, true)) != PIMHIP_OK) return rc;
    if (va.rows > 1 && ld_out < vb.rows) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "ld_out=%lld is less than the %lld rows of b", (long long)ld_out, (long long)vb.rows);
    hipStream_t s = static_cast<hipStream_t>(stream);
    rc = dtype == PIMHIP_F16 ? matmul<F16>(out, ld_out, va, vb, s) : dtype == PIMHIP_BF16 ? matmul<BF16>(out, ld_out, va, vb, s) : matmul<F32>(out, ld_out, va, vb, s);
    if (rc != PIMHIP_OK) return rc;
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}
