// The mixture-of-experts layer for a few tokens of the C ABI (include/pimhip.h).
#include "api_common.h"
#include "moe_layer_kernels.h"

using namespace pimhip;

namespace
{
struct Plan {
    uintptr_t number = 0;  // what a PimHipMoeLayerPlan* holds
    int device = 0;
    int num_experts = 0, top_k = 0;
    int64_t d_model = 0, d_ff = 0;
    int dtype = 0, act = 0, gated = 0, renormalize = 0, mx4 = 0;
    int64_t ld_s1 = 0, ld_s2 = 0;
    const void* router_w = nullptr;
    const void* router_b = nullptr;
    ExpertPointers* experts = nullptr;  // device, [E]
};

// A plan's handle is its number and no address, which the next plan might get: the handle of a destroyed plan is no other's.
std::vector<Plan*> g_moe_layer_plans;
uintptr_t g_moe_layer_plans_made = 0;

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
int64_t hidden_pitch(const Plan* p) { return (p->d_ff + 7) / 8 * 8; }
size_t hidden_bytes(const Plan* p, int tokens) { return round256((size_t)tokens * p->top_k * hidden_pitch(p) * 4); }
size_t part_bytes(const Plan* p, int tokens) { return round256((size_t)tokens * p->top_k * p->d_model * sizeof(float)); }

size_t counter_bytes(const Plan* p) { return round256((size_t)(p->d_model + 15) / 16 * sizeof(unsigned int)); }
int64_t most_pitch(const Plan* p) { return (p->d_ff + 255) / 256 * 16; }
size_t most_bytes(const Plan* p, int tokens) { return (size_t)tokens * p->top_k * most_pitch(p); }

Plan* find_locked(const PimHipMoeLayerPlan* handle)
{
    for (Plan* p : g_moe_layer_plans)
        if (p->number == reinterpret_cast<uintptr_t>(handle)) return p;
    return nullptr;
}

// A plan that shutting the library down, or its owner, has destroyed is refused.
int find_plan(const PimHipMoeLayerPlan* handle, Plan** plan)
{
    std::lock_guard<std::mutex> lock(g_mutex);
    *plan = find_locked(handle);
    return *plan ? (int)PIMHIP_OK : fail(PIMHIP_ERR_INVALID_ARGUMENT, "unknown or already destroyed expert layer plan");
}

int destroy_moe_layer_plan_locked(Plan* plan)
{
    if (!plan) return PIMHIP_OK;
    int prev = -1;
    hipGetDevice(&prev);
    hipSetDevice(plan->device);
    hipDeviceSynchronize();
    if (plan->experts) hipFree(plan->experts);
    if (prev >= 0) hipSetDevice(prev);
    for (size_t i = 0; i < g_moe_layer_plans.size(); ++i) {
        if (g_moe_layer_plans[i] == plan) {
            g_moe_layer_plans.erase(g_moe_layer_plans.begin() + i);
            break;
        }
    }
    delete plan;
    return PIMHIP_OK;
}

// LDS that staging `columns` of a product over K values takes, in bytes (weights of T's units).
template <class T, bool MX>
unsigned int shared_bytes(int columns, int K)
{
    return (unsigned int)(columns * SharedTokens<T>::pitch(K, ExpertWeights<T, MX, 1>::W::kUnit) * 16);
}

template <class T, bool MX, bool SHARED, bool GATED, int F, int TT>
void launch_first(const MoeLayerArgs& a, unsigned int bytes, hipStream_t s)
{
    constexpr int WK = 4;
    moe_layer_first_kernel<T, MX, SHARED, GATED, F, WK, TT>
        <<<dim3((unsigned)((a.d_ff + 16 * F - 1) / (16 * F)), (unsigned)a.E, (unsigned)((a.tokens + 16 * TT - 1) / (16 * TT))), 64 * WK, SHARED ? bytes : 0, s>>>(a);
}

// `most`: LDS that staged columns may take.
template <class T, bool MX, int RT, int WK, bool FEW>
void launch_second(const MoeLayerArgs& a, unsigned int most, hipStream_t s)
{
    typedef SecondColumns<T, MX, true, FEW> C;
    const dim3 grid((unsigned)((a.d_model + 16 * RT - 1) / (16 * RT)), (unsigned)a.E, (unsigned)((a.tokens + C::kPairs - 1) / C::kPairs));
    const unsigned int bytes = shared_bytes<T, MX>((a.tokens < 16 ? a.tokens : 16) * C::kPieces, a.d_ff);
    if (bytes <= most)
        moe_layer_second_kernel<T, MX, true, RT, WK, FEW><<<grid, 64 * WK, bytes, s>>>(a);
    else
        moe_layer_second_kernel<T, MX, false, RT, WK, FEW><<<grid, 64 * WK, 0, s>>>(a);
}

template <class T, bool MX>
void launch(const Plan* p, MoeLayerArgs& a, hipStream_t s)
{
    moe_layer_router_kernel<T><<<dim3((unsigned)a.tokens), kRouterThreads, 0, s>>>(a);
    // Columns are staged as a whole where tokens are one or two, or where an expert has many and 16 of them leave a CU room for three
    // blocks (the second product of one token and 4096 hidden values in three pieces, 24 KB: 18.2 us a call, 21.7 turned).
    const bool many = a.tokens > 16;
    const unsigned int most = many ? 40 << 10 : a.tokens <= 2 ? 26 << 10 : 0;
    // With many tokens a block has twice the rows: their values are read, and turned or staged, half as often (64 tokens through 8 gated 4-bit
    // experts 1024 -> 4096: 29.8 -> 20.8 us; one token through 2 of 8 experts 1024 -> 4096 in fp16, where blocks are few: 6.1 -> 7.9).
    const unsigned int staged = shared_bytes<T, MX>(a.tokens < 16 ? a.tokens : 16, a.d_model);
    auto first = [&](auto shared) {
        constexpr bool S = decltype(shared)::value;
        if (many)
            p->gated ? launch_first<T, MX, S, true, 2, 1>(a, staged, s) : launch_first<T, MX, S, false, 4, 1>(a, staged, s);
        else
            p->gated ? launch_first<T, MX, S, true, 1, 1>(a, staged, s) : launch_first<T, MX, S, false, 2, 1>(a, staged, s);
    };
    // Where experts have more than 16 pairs, which some have from 10 on the average on, 32 of them a block read their weights half as often.
    // In us a call, 32 / 16 pairs a block, 64 tokens through 8 experts 1024 -> 4096, two chosen: gated in 4 bits 44.4 / 48.7, gated fp16 63 / 73, fp16
    // 49.5 / 52.8; 16 tokens through both of 2 experts 512 -> 1024, which have 16 pairs at the most, 17.6 / 14.8.
    const int pairs = a.tokens * a.top_k;
    if (many && pairs > 10 * a.E)
        p->gated ? launch_first<T, MX, false, true, 2, 2>(a, 0, s) : launch_first<T, MX, false, false, 4, 2>(a, 0, s);
    else
        staged <= most ? first(std::true_type{}) : first(std::false_type{});
    // Blocks of the second product that have something to read.  Where they fill the card several times over a block has two tiles of
    // rows and four wavefronts, else eight wavefronts share its long k.  The pieces of 8 pairs (fp16) or 5 (bfloat16) are a tile; 16 pairs in a tile a
    // piece read an expert's weights less often where experts have many pairs, and turn and multiply more where they have few.  In us a call, 16 / 8 or 5
    // pairs a block, by pairs an expert on the average, 8 gated experts 1024 -> 4096, two chosen, and 64 of 2048 -> 1024, six chosen:
    //   fp16        3.3: 44.8 / 42.6   5: 48.5 / 48.5   6: 49.3 / 53.6   16: 63 / 69
    //   bfloat16    2.5: 44.1 / 42.0   3.3: 44.5 / 46.9   4.3: 46.3 / 54.1   16: 58 / 84      64 experts   2.3: 160 / 158   3.8: 169 / 174   6: 182 / 224
    //   4 bits, fp16 x    6: 36.0 / 32.0   7: 37.6 / 37.1   8: 37.2 / 37.6   16: 43.7 / 50.4
    //   4 bits, bfloat16 x    6: 36.9 / 33.3   7: 38.2 / 34.8   8: 37.5 / 35.8   16: 43.8 / 49.9      64 experts   3.8: 95.6 / 90.0   6: 107.6 / 128.2
    const int64_t blocks = (int64_t)((a.d_model + 15) / 16) * (a.E < pairs ? a.E : pairs);
    const int border = MX ? (blocks >= 2048 ? 5 : 7) : Pieces<T>::kCount > 2 ? 3 : 5;
    if (pairs > border * a.E) {
        if constexpr (!MX) {
            // (16-bit weights are four times the bytes: 64 tokens through 8 fp16 experts 1024 -> 4096 49.5 with eight wavefronts and a tile, 53.7 with two
            // tiles and four; in 4 bits 48.4 / 44.4, the values being turned for each tile of rows)
            if (blocks < 2048) return launch_second<T, MX, 1, 8, false>(a, most, s);
        }
        launch_second<T, MX, 2, 4, false>(a, most, s);
    } else if (blocks >= 2048)
        launch_second<T, MX, 2, 4, true>(a, most, s);
    else if (many)
        launch_second<T, MX, 2, 8, true>(a, most, s);
    else
        launch_second<T, MX, 1, 8, true>(a, most, s);
}
}  // namespace

namespace pimhip
{
void destroy_all_moe_layer_plans_locked()
{
    while (!g_moe_layer_plans.empty()) destroy_moe_layer_plan_locked(g_moe_layer_plans.back());
}
}  // namespace pimhip

extern "C" int pimhip_moe_layer_plan_create(PimHipMoeLayerPlan** plan_out, const PimHipMoeLayerDesc* d, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    if (!plan_out || !d || !d->router_w) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "plan, desc and router_w must be non-null");
    if (d->dtype != PIMHIP_F16 && d->dtype != PIMHIP_BF16) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "dtype=%d", d->dtype);
    if (d->num_experts < 1 || d->num_experts > kMoeLayerExperts)
        return fail(PIMHIP_ERR_UNSUPPORTED, "num_experts=%d not in [1, %d]", d->num_experts, kMoeLayerExperts);
    if (d->top_k < 1 || d->top_k > kMoeLayerTopK || d->top_k > d->num_experts)
        return fail(PIMHIP_ERR_UNSUPPORTED, "top_k=%d not in [1, min(%d, num_experts)]", d->top_k, kMoeLayerTopK);
    constexpr int64_t kMost = 1 << 20;
    if (d->d_model < 8 || d->d_model > kMost || (d->d_model & 7) || d->d_ff < 1 || d->d_ff > kMost)
        return fail(PIMHIP_ERR_UNSUPPORTED, "d_model=%lld must be a multiple of 8, d_model and d_ff=%lld at most %lld", (long long)d->d_model, (long long)d->d_ff,
                    (long long)kMost);
    if (d->act != PIMHIP_EXPERT_NONE && d->act != PIMHIP_EXPERT_RELU && d->act != PIMHIP_EXPERT_SILU) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "act=%d", d->act);
    const bool mx = d->w1_mx4 || d->w2_mx4;
    if (mx ? (!d->w1_mx4 || !d->w2_mx4) : (!d->w1 || !d->w2))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "either w1 and w2 or w1_mx4 and w2_mx4 must be non-null");
    if (!aligned16(d->router_w)) return fail(PIMHIP_ERR_UNSUPPORTED, "router_w must be 16-byte aligned");
    const int64_t rows1 = d->gated ? 2 * d->d_ff : d->d_ff;
    ExpertPointers table[kMoeLayerExperts];
    for (int e = 0; e < d->num_experts; ++e) {
        ExpertPointers& p = table[e];
        memset(&p, 0, sizeof(p));
        if (mx) {
            const PimHipMx4Matrix *m1 = d->w1_mx4 + e, *m2 = d->w2_mx4 + e;
            if (m1->rows != rows1 || m1->cols != d->d_model || m2->rows != d->d_model || m2->cols != d->d_ff)
                return fail(PIMHIP_ERR_INVALID_ARGUMENT, "expert %d: w1 must be [%lld, %lld] and w2 [%lld, %lld]", e, (long long)rows1, (long long)d->d_model,
                            (long long)d->d_model, (long long)d->d_ff);
            for (const PimHipMx4Matrix* m : {m1, m2}) {
                if (!m->packed || !m->scales || !m->tops || !aligned16(m->packed) || !aligned16(m->scales) || (m->ld_scales & 15) ||
                    m->ld_scales < (m->cols + 31) / 32 || m->ld_scales > INT32_MAX / 16 || m->ld_scales != (m == m1 ? d->w1_mx4 : d->w2_mx4)->ld_scales)
                    return fail(PIMHIP_ERR_INVALID_ARGUMENT, "expert %d: a 4-bit matrix is null, not 16-byte aligned, or has another pitch of scales", e);
            }
            p.w1 = m1->packed, p.s1 = m1->scales, p.t1 = m1->tops;
            p.w2 = m2->packed, p.s2 = m2->scales, p.t2 = m2->tops;
        } else {
            p.w1 = d->w1[e], p.w2 = d->w2[e];
            if (!p.w1 || !p.w2) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "w1[%d] / w2[%d] is null", e, e);
            if (!aligned16(p.w1) || !aligned16(p.w2)) return fail(PIMHIP_ERR_UNSUPPORTED, "the weights of expert %d must be 16-byte aligned", e);
        }
        p.b1 = d->b1 ? d->b1[e] : nullptr;
        p.b2 = d->b2 ? d->b2[e] : nullptr;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    PIMHIP_HIP_CHECK(hipStreamIsCapturing(s, &capture));
    if (capture != hipStreamCaptureStatusNone) return fail(PIMHIP_ERR_UNSUPPORTED, "a plan allocates: create it before the capture");
    Plan* plan = new (std::nothrow) Plan();
    if (!plan) return fail(PIMHIP_ERR_HIP, "out of host memory");
    hipGetDevice(&plan->device);
    plan->num_experts = d->num_experts, plan->top_k = d->top_k, plan->d_model = d->d_model, plan->d_ff = d->d_ff;
    plan->dtype = d->dtype, plan->act = d->act, plan->gated = d->gated ? 1 : 0, plan->renormalize = d->renormalize ? 1 : 0, plan->mx4 = mx;
    plan->ld_s1 = mx ? d->w1_mx4->ld_scales : 0, plan->ld_s2 = mx ? d->w2_mx4->ld_scales : 0;
    plan->router_w = d->router_w, plan->router_b = d->router_b;
    const size_t bytes = (size_t)d->num_experts * sizeof(ExpertPointers);
    hipError_t err = hipMalloc(reinterpret_cast<void**>(&plan->experts), bytes);
    if (err == hipSuccess) err = hipMemcpyAsync(plan->experts, table, bytes, hipMemcpyHostToDevice, s);
    if (err == hipSuccess) err = hipStreamSynchronize(s);  // (table goes out of scope)
    std::lock_guard<std::mutex> lock(g_mutex);
    if (err != hipSuccess) {
        destroy_moe_layer_plan_locked(plan);
        return fail(PIMHIP_ERR_HIP, "the table of experts could not be set up: %s", hipGetErrorString(err));
    }
    try {
        g_moe_layer_plans.push_back(plan);
        plan->number = ++g_moe_layer_plans_made;
    } catch (...) {
        destroy_moe_layer_plan_locked(plan);
        return fail(PIMHIP_ERR_HIP, "out of host memory");
    }
    *plan_out = reinterpret_cast<PimHipMoeLayerPlan*>(plan->number);
    return PIMHIP_OK;
}

extern "C" int pimhip_moe_layer_plan_destroy(PimHipMoeLayerPlan* handle)
{
    if (!handle) return PIMHIP_OK;
    std::lock_guard<std::mutex> lock(g_mutex);
    Plan* plan = find_locked(handle);
    if (!plan) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "unknown or already destroyed expert layer plan");
    return destroy_moe_layer_plan_locked(plan);
}

extern "C" int pimhip_moe_layer_workspace_bytes(const PimHipMoeLayerPlan* handle, int tokens, uint64_t* bytes)
{
    if (!handle || !bytes) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "plan and bytes must be non-null");
    Plan* plan;
    const int rc = find_plan(handle, &plan);
    if (rc != PIMHIP_OK) return rc;
    if (tokens < 0 || tokens > kMoeLayerTokens) return fail(PIMHIP_ERR_UNSUPPORTED, "tokens=%d not in [0, %d]", tokens, kMoeLayerTokens);
    *bytes = hidden_bytes(plan, tokens) + part_bytes(plan, tokens) + counter_bytes(plan) + most_bytes(plan, tokens);
    return PIMHIP_OK;
}

extern "C" int pimhip_moe_layer_forward(PimHipMoeLayerPlan* handle, const void* x, int64_t ld_x, int tokens, void* y, int* experts, float* shares,
                                        void* workspace, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    if (!handle) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "plan is null");
    Plan* plan;
    if ((rc = find_plan(handle, &plan)) != PIMHIP_OK) return rc;
    int dev = -1;
    PIMHIP_HIP_CHECK(hipGetDevice(&dev));
    if (dev != plan->device) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "plan belongs to device %d, current device is %d", plan->device, dev);
    if (tokens < 0 || tokens > kMoeLayerTokens) return fail(PIMHIP_ERR_UNSUPPORTED, "tokens=%d not in [0, %d]", tokens, kMoeLayerTokens);
    if (tokens == 0) return PIMHIP_OK;
    if (!x || !y || !experts || !shares || !workspace) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "x, y, experts, shares and workspace must be non-null");
    if (!aligned16(workspace)) return fail(PIMHIP_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(x) & 1u) || (reinterpret_cast<uintptr_t>(y) & 1u) || (reinterpret_cast<uintptr_t>(experts) & 3u) ||
        (reinterpret_cast<uintptr_t>(shares) & 3u))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "x, y, experts and shares must be aligned to their elements");
    if (tokens > 1 && (ld_x < plan->d_model || ld_x > INT32_MAX)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "ld_x=%lld", (long long)ld_x);
    MoeLayerArgs a;
    memset(&a, 0, sizeof(a));
    a.experts = plan->experts;
    a.x = x, a.router_w = plan->router_w, a.router_b = plan->router_b, a.y = y;
    a.chosen = experts, a.share = shares;
    a.h = static_cast<float*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + hidden_bytes(plan, tokens));
    a.counters = reinterpret_cast<unsigned int*>(static_cast<char*>(workspace) + hidden_bytes(plan, tokens) + part_bytes(plan, tokens));
    a.tokens = tokens, a.E = plan->num_experts, a.top_k = plan->top_k, a.d_model = (int)plan->d_model, a.d_ff = (int)plan->d_ff;
    a.h_most = reinterpret_cast<uint8_t*>(a.counters) + counter_bytes(plan);
    a.counters_used = (a.d_model + 15) / 16;
    a.ld_h = (int)hidden_pitch(plan), a.ld_most = (int)most_pitch(plan);
    a.ld_x = tokens > 1 ? (int)ld_x : 0;
    a.ld_s1 = (int)plan->ld_s1, a.ld_s2 = (int)plan->ld_s2;
    a.act = plan->act, a.renormalize = plan->renormalize;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f16 = plan->dtype == PIMHIP_F16;
    if (plan->mx4)
        f16 ? launch<F16, true>(plan, a, s) : launch<BF16, true>(plan, a, s);
    else
        f16 ? launch<F16, false>(plan, a, s) : launch<BF16, false>(plan, a, s);
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}
