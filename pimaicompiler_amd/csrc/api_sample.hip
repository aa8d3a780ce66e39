// Sampling, of the C ABI (include/pimhip.h).
#include "api_common.h"
#include "sample_kernels.h"

#include <type_traits>

using namespace pimhip;

namespace
{
// Values are counted (16-bit rows) where a row may need it, with a top_p or a top_k above the list's: it takes a CU for one row and some 15 us, whatever
// the row's length.  A nucleus of half of 32000 tokens, in us, counted and not: 64 rows 40 and 44, of 16000 38 and 30; a peaked one of 32000
// 27 and 25.  Where CUs have several rows each: 512 rows of 32000 80 and 73, of 64000 98 and 121, peaked ones 68 and 53.
constexpr int kCountFrom = 24576, kCountFromMany = 49152;

// The first pass by all CUs, in a launch of its own, where rows are few and long.  In us, without and with it: one row of 131072 with nothing cut off 36 and 15,
// with top_k 40 24.5 and 19.4, with a peaked nucleus 43 and 19, a flat one 57 and 68 (it is counted after all; in fp32 128 and 107); one of 32000 with top_k
// 40 15.8 and 17.8; 64 rows of 100003 33 and 22, with top_k 40 23.7 and 22.7; 128 of them with top_k 40 24 and 26, of 200000, whose pieces' largest
// values do not fit into LDS, 43 and 33.
constexpr int kPartsFrom = 49152;

// Threads of a block.  One row a CU: 256 while that is enough (4000 tokens: 13.3 us, with 512 13.0, with 1024 14.5), 512, and 1024 for long ones (64 rows
// with top_k 40, of 16000: 14.4 and 15.6 us with 512 and 1024; of 100003: 26.7 and 23.9).  Two rows of 512 threads share a CU (512 rows of 32000: 22.4 with 512,
// 24.6 with 256, 34 with 1024), four of 256 as long as their largest values leave LDS for that (2000 rows of 8000: 36 with 256, 58 with 512; 1024 of
// 32000 32 and 39, of 64000 65 and 57).
int threads_of(int64_t rows, int64_t vocab, int num_cus)
{
    constexpr int kMiddle = 32768;
    if (vocab <= 4096 || (vocab <= kMiddle && rows > 2 * (int64_t)num_cus)) return 256;
    return vocab <= kMiddle || rows > num_cus ? 512 : 1024;
}

// How a call is worked out.
struct SampleCut {
    bool count, parts;
    int threads, segments;
    int64_t ld_tops;
    uint64_t best_at, sums_at, bytes;  // of the workspace: the pieces' largest values come first
};
int cut_of(int dtype, int64_t rows, int64_t vocab, const PimHipSampleSettings* settings, int num_cus, SampleCut* cut)
{
    if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > kSampleMost)
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "rows=%lld, vocab=%lld (at most %d)", (long long)rows, (long long)vocab, kSampleMost);
    if (dtype != PIMHIP_F16 && dtype != PIMHIP_BF16 && dtype != PIMHIP_F32) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "dtype=%d", dtype);
    if (!settings) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "settings must be non-null");
    const bool many_k = !settings->top_ks && settings->top_k > kListMost / 2;
    cut->count = dtype != PIMHIP_F32 && vocab > (rows > num_cus ? kCountFromMany : kCountFrom) && (settings->top_ks || settings->top_k <= 0 || many_k) &&
                 (settings->top_ks || settings->top_ps || settings->top_p < 1.0f || settings->top_k > 0);
    cut->threads = cut->count ? 1024 : threads_of(rows, vocab, num_cus);
    if (rows * cut->threads > UINT32_MAX) return fail(PIMHIP_ERR_UNSUPPORTED, "%lld rows are too many for one launch", (long long)rows);
    cut->parts = rows > 0 && 2 * rows <= num_cus && vocab > (4 * rows <= num_cus ? kPartsFrom : kTopsMost) && cut->threads == 1024 && !(cut->count && many_k);
    cut->segments = (int)((vocab + kSegment - 1) / kSegment);
    cut->ld_tops = ((vocab + 7) / 8 + 7) / 8 * 8;
    cut->best_at = (uint64_t)rows * cut->ld_tops * sizeof(unsigned short);
    cut->sums_at = cut->best_at + (uint64_t)rows * cut->segments * sizeof(unsigned long long);
    cut->bytes = cut->parts ? cut->sums_at + (uint64_t)rows * cut->segments * sizeof(double) : 0;
    return PIMHIP_OK;
}
}  // namespace

extern "C" int pimhip_sample_workspace_bytes(int dtype, int64_t rows, int64_t vocab, const PimHipSampleSettings* settings, uint64_t* bytes)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    SampleCut cut;
    if ((rc = cut_of(dtype, rows, vocab, settings, st->num_cus, &cut)) != PIMHIP_OK) return rc;
    if (!bytes) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = cut.bytes;
    return PIMHIP_OK;
}

extern "C" int pimhip_sample_tokens(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab, const float* uniform, const PimHipSampleSettings* settings,
                                    int64_t* tokens, float* logp, void* workspace, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    SampleCut cut;
    if ((rc = cut_of(dtype, rows, vocab, settings, st->num_cus, &cut)) != PIMHIP_OK) return rc;
    if (rows == 0) return PIMHIP_OK;
    if (!logits || (rows > 1 && ld < vocab)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "logits is null, or ld=%lld is less than vocab=%lld", (long long)ld, (long long)vocab);
    if (!uniform || !tokens || !logp) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "uniform, tokens and logp must be non-null");
    auto off = [](const void* p, uintptr_t size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; };
    if (off(logits, dtype == PIMHIP_F32 ? 4 : 2) || off(uniform, 4) || off(tokens, 8) || off(logp, 4) || off(settings->temperatures, 4) || off(settings->top_ks, 4) ||
        off(settings->top_ps, 4) || off(settings->min_ps, 4))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its elements");
    if (cut.parts && (!workspace || off(workspace, 16))) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "workspace must be non-null and aligned to 16 bytes");
    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits, a.ld = ld, a.uniform = uniform;
    a.temperatures = settings->temperatures, a.top_ks = settings->top_ks, a.top_ps = settings->top_ps, a.min_ps = settings->min_ps;
    a.temperature = settings->temperature, a.top_k = settings->top_k, a.top_p = settings->top_p, a.min_p = settings->min_p;
    a.tokens = tokens, a.logp = logp, a.V = (int)vocab;
    a.shift = 45;
    while (vocab > (int64_t)1 << (62 - a.shift)) --a.shift;
    if (cut.parts) {
        char* w = static_cast<char*>(workspace);
        a.part_tops = reinterpret_cast<unsigned short*>(w), a.ld_tops = cut.ld_tops;
        a.part_best = reinterpret_cast<unsigned long long*>(w + cut.best_at), a.part_sums = reinterpret_cast<double*>(w + cut.sums_at);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto type) {
        typedef decltype(type) T;
        auto launch = [&](auto threads, auto counts, auto parts) {
            constexpr int kThreads = decltype(threads)::value;
            constexpr bool kCount = decltype(counts)::value;
            sample_kernel<T, kThreads, kCount, decltype(parts)::value><<<dim3((unsigned)rows), kThreads, sample_shared_bytes<T, kThreads, kCount>(a.V), s>>>(a);
        };
        typedef std::integral_constant<int, 256> T256;
        typedef std::integral_constant<int, 512> T512;
        typedef std::integral_constant<int, 1024> T1024;
        constexpr std::true_type yes;
        constexpr std::false_type no;
        constexpr std::integral_constant<bool, !std::is_same<T, F32>::value> short_values;
        if (cut.parts) {
            sample_parts_kernel<T><<<dim3((unsigned)(cut.segments + 3) / 4, (unsigned)rows), 256, 0, s>>>(a);
            return launch(T1024{}, short_values, yes);
        }
        if constexpr (short_values) {
            if (cut.count) return launch(T1024{}, yes, no);
        }
        cut.threads == 256 ? launch(T256{}, no, no) : cut.threads == 512 ? launch(T512{}, no, no) : launch(T1024{}, no, no);
    };
    dtype == PIMHIP_F16 ? run(F16{}) : dtype == PIMHIP_BF16 ? run(BF16{}) : run(F32{});
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}
