// Log probabilities of tokens with entropy and alternatives, of the C ABI (include/pimhip.h).
#include "api_common.h"
#include "logprob_kernels.h"

using namespace pimhip;

extern "C" int pimhip_token_log_probs(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab, const void* tokens, int tokens_int64, int top,
                                      float* logp, float* entropy, float* top_logp, int* top_ids, void* stream)
{
    DeviceState* st = nullptr;
    const int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > INT32_MAX - 8)
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "rows=%lld, vocab=%lld", (long long)rows, (long long)vocab);
    if (dtype != PIMHIP_F16 && dtype != PIMHIP_BF16 && dtype != PIMHIP_F32) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "dtype=%d", dtype);
    if (top < 0 || top > kTopMost || top > vocab) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "top=%d not in [0, min(%d, vocab)]", top, kTopMost);
    const int threads = vocab <= 1024 ? 64 : vocab <= 8192 ? 256 : 1024;
    if (rows * threads > UINT32_MAX) return fail(PIMHIP_ERR_UNSUPPORTED, "%lld rows are too many for one launch", (long long)rows);
    if (rows == 0) return PIMHIP_OK;
    if (!logits || (rows > 1 && ld < vocab)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "logits is null, or ld=%lld is less than vocab=%lld", (long long)ld, (long long)vocab);
    if (reinterpret_cast<uintptr_t>(logits) & (dtype == PIMHIP_F32 ? 3u : 1u)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "logits is not aligned to its elements");
    if ((logp != nullptr) != (tokens != nullptr)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "logp goes with tokens: both or neither");
    if (top > 0 && (!top_logp || !top_ids)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "top_logp and top_ids must be non-null where top is not 0");
    LogProbArgs a{logits, tokens, logp, entropy, top_logp, top_ids, vocab, ld, top, tokens_int64 ? 1 : 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto type) {
        typedef decltype(type) T;
        if (threads == 64)
            token_log_probs_kernel<T, 64><<<dim3((unsigned)rows), 64, 0, s>>>(a);
        else if (threads == 256)
            token_log_probs_kernel<T, 256><<<dim3((unsigned)rows), 256, 0, s>>>(a);
        else
            token_log_probs_kernel<T, 1024><<<dim3((unsigned)rows), 1024, 0, s>>>(a);
    };
    dtype == PIMHIP_F16 ? run(F16{}) : dtype == PIMHIP_BF16 ? run(BF16{}) : run(F32{});
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}
