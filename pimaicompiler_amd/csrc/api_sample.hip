// Sampling, of the C ABI (include/pimhip.h).
#include "api_common.h"
#include "sample_kernels.h"

#include <type_traits>

using namespace pimhip;

namespace
{
// Values are counted (16-bit rows) where a row may need it, with a top_p or a top_k above the list's: it takes a CU for one row and some 15 us, whatever
// the row's length.  A nucleus of half of 32000 tokens, in us, counted and not: 64 rows 40 and 53, of 16000 38 and 35; a peaked one of 32000
// 27 and 27.  Where CUs have several rows each: 512 rows of 32000 82 and 80, of 64000 99 and 135, peaked ones 72 and 54.
constexpr int kCountFrom = 24576, kCountFromMany = 49152;

// Threads of a block.  One row a CU: 256 while that is enough (4000 tokens: 13.7 us with any number), 512, and 1024 for long ones (64 rows
// with top_k 40, of 16000: 15.8 and 16.5 us with 512 and 1024; of 100003: 27.9 and 25.5).  Two rows of 512 threads share a CU (512 rows of 32000: 26.0 with 512,
// 26.7 with 256, 38 with 1024), four of 256 as long as their largest values leave LDS for that (2000 rows of 8000: 41.7 with 256, 64.8 with 512; 1024 of
// 32000 38.3 and 44.0, of 64000 69.7 and 62.4).
int threads_of(int64_t rows, int64_t vocab, int num_cus)
{
    constexpr int kMiddle = 32768;
    if (vocab <= 4096 || (vocab <= kMiddle && rows > 2 * (int64_t)num_cus)) return 256;
    return vocab <= kMiddle || rows > num_cus ? 512 : 1024;
}
}  // namespace

extern "C" int pimhip_sample_tokens(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab, const float* uniform, const PimHipSampleSettings* settings,
                                    int64_t* tokens, float* logp, void* stream)
{
    DeviceState* st = nullptr;
    const int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > kSampleMost)
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "rows=%lld, vocab=%lld (at most %d)", (long long)rows, (long long)vocab, kSampleMost);
    if (dtype != PIMHIP_F16 && dtype != PIMHIP_BF16 && dtype != PIMHIP_F32) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "dtype=%d", dtype);
    if (!settings) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "settings must be non-null");
    const bool count = dtype != PIMHIP_F32 && vocab > (rows > st->num_cus ? kCountFromMany : kCountFrom) &&
                       (settings->top_ks || settings->top_k <= 0 || settings->top_k > kListMost / 2) &&
                       (settings->top_ks || settings->top_ps || settings->top_p < 1.0f || settings->top_k > 0);
    const int threads = count ? 1024 : threads_of(rows, vocab, st->num_cus);
    if (rows * threads > UINT32_MAX) return fail(PIMHIP_ERR_UNSUPPORTED, "%lld rows are too many for one launch", (long long)rows);
    if (rows == 0) return PIMHIP_OK;
    if (!logits || (rows > 1 && ld < vocab)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "logits is null, or ld=%lld is less than vocab=%lld", (long long)ld, (long long)vocab);
    if (!uniform || !tokens || !logp) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "uniform, tokens and logp must be non-null");
    auto off = [](const void* p, uintptr_t size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; };
    if (off(logits, dtype == PIMHIP_F32 ? 4 : 2) || off(uniform, 4) || off(tokens, 8) || off(logp, 4) || off(settings->temperatures, 4) || off(settings->top_ks, 4) ||
        off(settings->top_ps, 4) || off(settings->min_ps, 4))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its elements");
    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits, a.ld = ld, a.uniform = uniform;
    a.temperatures = settings->temperatures, a.top_ks = settings->top_ks, a.top_ps = settings->top_ps, a.min_ps = settings->min_ps;
    a.temperature = settings->temperature, a.top_k = settings->top_k, a.top_p = settings->top_p, a.min_p = settings->min_p;
    a.tokens = tokens, a.logp = logp, a.V = (int)vocab;
    a.shift = 45;
    while (vocab > (int64_t)1 << (62 - a.shift)) --a.shift;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto type) {
        typedef decltype(type) T;
        auto launch = [&](auto threads, auto counts) {
            constexpr int kThreads = decltype(threads)::value;
            constexpr bool kCount = decltype(counts)::value;
            sample_kernel<T, kThreads, kCount><<<dim3((unsigned)rows), kThreads, sample_shared_bytes<T, kThreads, kCount>(a.V), s>>>(a);
        };
        typedef std::integral_constant<int, 256> T256;
        typedef std::integral_constant<int, 512> T512;
        typedef std::integral_constant<int, 1024> T1024;
        if constexpr (!std::is_same<T, F32>::value) {
            if (count) return launch(T1024{}, std::true_type{});
        }
        threads == 256 ? launch(T256{}, std::false_type{}) : threads == 512 ? launch(T512{}, std::false_type{}) : launch(T1024{}, std::false_type{});
    };
    dtype == PIMHIP_F16 ? run(F16{}) : dtype == PIMHIP_BF16 ? run(BF16{}) : run(F32{});
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}
