// A paged cache of keys and values, of the C ABI (include/pimhip.h).
#include "api_common.h"
#include "paged_kernels.h"

using namespace pimhip;

namespace
{
constexpr int kDimMost = 256;

bool element_aligned(const void* p, unsigned int size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) == 0; }

// What both entry points ask of the cache and the batch, and the view of them that kernels take.
int view_of(const PimHipPagedCache* cache, const PimHipPagedBatch* batch, PagedView* view)
{
    if (!cache || !batch) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "cache and batch must be non-null");
    const PimHipPagedCache& c = *cache;
    const bool fp8 = c.dtype == PIMHIP_F8E4M3;
    if (!fp8 && c.dtype != PIMHIP_F16 && c.dtype != PIMHIP_BF16) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "cache dtype=%d", c.dtype);
    if (c.pages < 1 || c.pages > INT32_MAX || c.kv_heads < 1 || c.kv_heads > 65535 || c.page_size < 1 || c.page_size > 65536)
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "pages=%lld, kv_heads=%d, page_size=%d", (long long)c.pages, c.kv_heads, c.page_size);
    if (c.head_dim < 1 || c.head_dim > kDimMost || c.head_dim % (fp8 ? 16 : 8))
        return fail(PIMHIP_ERR_UNSUPPORTED, "head_dim=%d is no multiple of %d up to %d", c.head_dim, fp8 ? 16 : 8, kDimMost);
    const int size = fp8 ? 1 : 2;
    if (!c.k || !c.v || !element_aligned(c.k, size) || !element_aligned(c.v, size))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "k and v must be non-null and aligned to their elements");
    if (fp8 ? !c.k_scale || !c.v_scale || !element_aligned(c.k_scale, 4) || !element_aligned(c.v_scale, 4) : c.k_scale || c.v_scale)
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "scales go with 8-bit caches: both or neither");
    for (const int64_t* s : {c.k_strides, c.v_strides}) {
        if (s[0] < 0 || s[1] < 0 || s[2] < 0 || s[2] > (int64_t)INT32_MAX / 2 / c.page_size || s[0] > INT64_MAX / 4 / c.pages || s[1] > INT64_MAX / 4 / c.kv_heads)
            return fail(PIMHIP_ERR_UNSUPPORTED, "strides %lld, %lld, %lld", (long long)s[0], (long long)s[1], (long long)s[2]);
    }
    const PimHipPagedBatch& b = *batch;
    if (b.sequences < 0 || b.sequences > (1 << 20) || b.table_width < 1 || (int64_t)b.table_width * c.page_size > INT32_MAX - 256 || (b.sequences > 1 && b.ld_table < b.table_width))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "sequences=%d, table_width=%d, ld_table=%lld", b.sequences, b.table_width, (long long)b.ld_table);
    if (b.sequences > 0 && (!b.page_table || !b.lengths || !element_aligned(b.page_table, 4) || !element_aligned(b.lengths, 4)))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "page_table and lengths must be non-null and aligned to their elements");
    PagedView& v = *view;
    v.k = static_cast<char*>(c.k), v.v = static_cast<char*>(c.v);
    v.k_scale = c.k_scale, v.v_scale = c.v_scale;
    v.k_page = c.k_strides[0] * size, v.k_head = c.k_strides[1] * size, v.k_tok = (int)c.k_strides[2] * size;
    v.v_page = c.v_strides[0] * size, v.v_head = c.v_strides[1] * size, v.v_tok = (int)c.v_strides[2] * size;
    v.pages = (int)c.pages, v.page_size = c.page_size, v.kv_heads = c.kv_heads, v.dim = c.head_dim;
    v.table = b.page_table, v.lengths = b.lengths, v.ld_table = b.ld_table;
    v.sequences = b.sequences, v.most = b.table_width * c.page_size;
    int log = 0;
    while (1 << log < c.page_size) ++log;
    v.shift = 31 + log, v.magic = (unsigned int)((((uint64_t)1 << v.shift) + c.page_size - 1) / c.page_size);
    return PIMHIP_OK;
}

int check_rows(const char* name, const PimHipPagedRows& r)
{
    if (!r.data || !element_aligned(r.data, 2)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "%s must be non-null and aligned to its elements", name);
    if (r.token_stride < 0 || r.head_stride < 0) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "%s has strides %lld, %lld", name, (long long)r.token_stride, (long long)r.head_stride);
    return PIMHIP_OK;
}

// How an attention call is cut: query heads at a time, their tiles of a key head, blocks of its grid.
struct AttendCut {
    int heads, tiles_of_heads, blocks;
};
int cut_of(const PagedView& v, int group, int num_cus, AttendCut* cut)
{
    const int nc = (v.dim + 63) / 64;
    // (for heads longer than 128 the registers do not hold the sums of 32 query heads)
    cut->heads = group > 16 && nc <= 2 ? 32 : 16;
    cut->tiles_of_heads = (group + cut->heads - 1) / cut->heads;
    const int64_t heads = (int64_t)v.kv_heads * cut->tiles_of_heads, units = (v.most + 15 + kUnit - 1) / kUnit;
    if (units * v.sequences > INT32_MAX / heads / 2 || (int64_t)v.sequences * v.kv_heads * group > (1 << 23))
        return fail(PIMHIP_ERR_UNSUPPORTED, "%d sequences of up to %d tokens with %d key heads are too many for one launch", v.sequences, v.most, v.kv_heads);
    const int64_t most = (int64_t)v.sequences * heads * units, wanted = attend_waves(nc, cut->heads) * (int64_t)num_cus;
    cut->blocks = (int)(most < wanted ? most : wanted);
    return PIMHIP_OK;
}

uint64_t part_bytes(const AttendCut& cut, int dim) { return (uint64_t)cut.blocks * 2 * cut.heads * (dim + 4) * sizeof(float); }

template <class T, bool FP8, int NC, int HT>
void launch_attend(const AttendArgs& a, int blocks, hipStream_t s)
{
    if (a.c.page_size % 16 == 0 && a.c.dim == 64 * NC)
        paged_attend_kernel<T, FP8, NC, HT, true><<<dim3(blocks), 256, 0, s>>>(a);
    else
        paged_attend_kernel<T, FP8, NC, HT, false><<<dim3(blocks), 256, 0, s>>>(a);
}
template <class T, bool FP8, int NC>
void launch_attend(const AttendArgs& a, const AttendCut& cut, hipStream_t s)
{
    if constexpr (NC <= 2) {
        if (cut.heads == 32) return launch_attend<T, FP8, NC, 32>(a, cut.blocks, s);
    }
    launch_attend<T, FP8, NC, 16>(a, cut.blocks, s);
}
template <class T, bool FP8>
void launch_attend(const AttendArgs& a, const AttendCut& cut, hipStream_t s)
{
    const int nc = (a.c.dim + 63) / 64;
    nc == 1   ? launch_attend<T, FP8, 1>(a, cut, s)
    : nc == 2 ? launch_attend<T, FP8, 2>(a, cut, s)
    : nc == 3 ? launch_attend<T, FP8, 3>(a, cut, s)
              : launch_attend<T, FP8, 4>(a, cut, s);
}
template <class T>
void launch_attend(const AttendArgs& a, const AttendCut& cut, int num_cus, hipStream_t s)
{
    a.c.k_scale ? launch_attend<T, true>(a, cut, s) : launch_attend<T, false>(a, cut, s);
    if (a.whole) return;
    // One wavefront a head where heads are many (64 sequences, 192 heads each: 276 us, with four 286), sixteen where they are few and may have more
    // than 32 parts (one sequence of 131071 tokens, 96 of them: 92.9 us, with four 94.8), else four (32 heads of 16 parts: 9.9 us, with one 10.8).
    const int heads = a.c.sequences * a.c.kv_heads * a.group;
    if (heads > 2 * num_cus)
        paged_join_kernel<T, 1><<<dim3((heads + 3) / 4), 256, 0, s>>>(a, cut.heads);
    else if (cut.blocks > 32 * (int64_t)a.c.sequences * a.c.kv_heads * a.tiles_of_heads)
        paged_join_kernel<T, 16><<<dim3(heads), 1024, 0, s>>>(a, cut.heads);
    else
        paged_join_kernel<T, 4><<<dim3(heads), 256, 0, s>>>(a, cut.heads);
}
}  // namespace

extern "C" int pimhip_paged_append(const PimHipPagedCache* cache, const PimHipPagedBatch* batch, const int* starts, int64_t tokens, const PimHipPagedRows* k,
                                   const PimHipPagedRows* v, const PimHipPagedRows* q, int q_heads, void* q_out, int dtype, const float* angles,
                                   int64_t angle_rows, int64_t ld_angles, int rotary_dim, int interleaved, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    AppendArgs a;
    memset(&a, 0, sizeof(a));
    if ((rc = view_of(cache, batch, &a.c)) != PIMHIP_OK) return rc;
    if (dtype != PIMHIP_F16 && dtype != PIMHIP_BF16) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "dtype=%d", dtype);
    if (cache->dtype != dtype && cache->dtype != PIMHIP_F8E4M3) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "a cache of type %d takes no tokens of type %d", cache->dtype, dtype);
    if (tokens < 0 || tokens > (1 << 23) || (!starts && tokens != batch->sequences))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "tokens=%lld for %d sequences", (long long)tokens, batch->sequences);
    if (starts && !element_aligned(starts, 4)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "starts is not aligned to its elements");
    if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > cache->head_dim) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "rotary_dim=%d", rotary_dim);
    if (rotary_dim > 0 && (!angles || !element_aligned(angles, 4) || angle_rows < a.c.most || ld_angles < rotary_dim))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "angles must be [%d or more, %d], got %lld rows with a pitch of %lld", a.c.most, rotary_dim, (long long)angle_rows,
                    (long long)ld_angles);
    if (q && (q_heads < 1 || q_heads > 65535 || !q_out || !element_aligned(q_out, 2))) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "q_heads=%d, or q_out is null", q_heads);
    if (cache->k == cache->v) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "keys and values of the cache are the same memory");
    if (tokens == 0) return PIMHIP_OK;
    if (!k || !v) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "k and v must be non-null");
    if ((rc = check_rows("k", *k)) != PIMHIP_OK || (rc = check_rows("v", *v)) != PIMHIP_OK || (q && (rc = check_rows("q", *q)) != PIMHIP_OK)) return rc;
    a.starts = starts;
    a.k = k->data, a.k_token = k->token_stride, a.k_head = k->head_stride;
    a.v = v->data, a.v_token = v->token_stride, a.v_head = v->head_stride;
    if (q) a.q = q->data, a.q_token = q->token_stride, a.q_head = q->head_stride, a.q_out = q_out, a.q_heads = q_heads;
    a.angles = angles, a.ld_angles = ld_angles, a.half = rotary_dim / 2;
    a.items = (2 * a.c.kv_heads + a.q_heads) * (a.c.dim / 8);
    // Blocks of one group a thread for a step's tokens, of four where there are tokens enough for every CU (32 + 8 + 8 heads of 128 in bfloat16, one and
    // four: 512 tokens 5.5 and 6.3 us, 1024 9.5 and 9.1, 4096 24.2 and 24.7, 8001 53 and 47.5, 16000 104 and 91).
    const bool many = tokens >= 4 * (int64_t)st->num_cus;
    const dim3 grid((unsigned)tokens, (unsigned)(a.items + 255) / 256), grid4((unsigned)tokens, (unsigned)(a.items + 1023) / 1024);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto type, auto fp8) {
        typedef decltype(type) T;
        constexpr bool kFp8 = decltype(fp8)::value;
        if (interleaved)
            many ? paged_append_kernel<T, kFp8, true, 4><<<grid4, 256, 0, s>>>(a) : paged_append_kernel<T, kFp8, true, 1><<<grid, 256, 0, s>>>(a);
        else
            many ? paged_append_kernel<T, kFp8, false, 4><<<grid4, 256, 0, s>>>(a) : paged_append_kernel<T, kFp8, false, 1><<<grid, 256, 0, s>>>(a);
    };
    auto run_type = [&](auto type) { cache->dtype == PIMHIP_F8E4M3 ? run(type, std::true_type{}) : run(type, std::false_type{}); };
    dtype == PIMHIP_F16 ? run_type(F16{}) : run_type(BF16{});
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}

extern "C" int pimhip_paged_attend_workspace_bytes(const PimHipPagedCache* cache, const PimHipPagedBatch* batch, int q_heads, uint64_t* bytes)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    PagedView v;
    if ((rc = view_of(cache, batch, &v)) != PIMHIP_OK) return rc;
    if (!bytes || q_heads < 1 || q_heads % v.kv_heads || q_heads > 65535) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "q_heads=%d with %d key heads, or bytes is null", q_heads, v.kv_heads);
    AttendCut cut;
    if ((rc = cut_of(v, q_heads / v.kv_heads, st->num_cus, &cut)) != PIMHIP_OK) return rc;
    *bytes = part_bytes(cut, v.dim) + (uint64_t)v.sequences * v.kv_heads * cut.tiles_of_heads * sizeof(int2);
    return PIMHIP_OK;
}

extern "C" int pimhip_paged_attend(const PimHipPagedCache* cache, const PimHipPagedBatch* batch, const PimHipPagedRows* q, int q_heads, int dtype, float scale,
                                   int window, void* out, float* lse, void* workspace, void* stream)
{
    DeviceState* st = nullptr;
    int rc = current_device_state(&st);
    if (rc != PIMHIP_OK) return rc;
    AttendArgs a;
    memset(&a, 0, sizeof(a));
    if ((rc = view_of(cache, batch, &a.c)) != PIMHIP_OK) return rc;
    if (dtype != PIMHIP_F16 && dtype != PIMHIP_BF16) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "dtype=%d", dtype);
    if (cache->dtype != dtype && cache->dtype != PIMHIP_F8E4M3) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "a cache of type %d takes no queries of type %d", cache->dtype, dtype);
    if (q_heads < 1 || q_heads % a.c.kv_heads || q_heads > 65535) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "q_heads=%d with %d key heads", q_heads, a.c.kv_heads);
    a.scale_log2 = scale * 1.4426950408889634f;
    if (window < 0 || !(a.scale_log2 - a.scale_log2 == 0.0f)) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "window=%d, scale=%g", window, (double)scale);
    AttendCut cut;
    if ((rc = cut_of(a.c, q_heads / a.c.kv_heads, st->num_cus, &cut)) != PIMHIP_OK) return rc;
    if (a.c.sequences == 0) return PIMHIP_OK;
    if (!q || !out || !workspace) return fail(PIMHIP_ERR_INVALID_ARGUMENT, "q, out and workspace must be non-null");
    if ((rc = check_rows("q", *q)) != PIMHIP_OK) return rc;
    if (!element_aligned(out, 2) || !element_aligned(lse, 4) || !aligned16(workspace))
        return fail(PIMHIP_ERR_INVALID_ARGUMENT, "out and lse must be aligned to their elements, workspace to 16 bytes");
    a.q = q->data, a.q_seq = q->token_stride, a.q_head = q->head_stride;
    a.out = out, a.lse = lse, a.work = static_cast<float*>(workspace);
    a.pieces = reinterpret_cast<int2*>(static_cast<char*>(workspace) + part_bytes(cut, a.c.dim));
    a.group = q_heads / a.c.kv_heads, a.tiles_of_heads = cut.tiles_of_heads, a.window = window;
    // Sequences of a few units, by the room they have or by the window, are not cut, and nothing is joined.
    const int64_t seen = window > 0 && window < a.c.most ? (int64_t)window + 15 : a.c.most;
    const int64_t heads = (int64_t)a.c.sequences * a.c.kv_heads * cut.tiles_of_heads;
    if (seen <= paged_whole_units(heads, true) * (int64_t)kUnit) {
        a.whole = 1;
        cut.blocks = (int)heads;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    dtype == PIMHIP_F16 ? launch_attend<F16>(a, cut, st->num_cus, s) : launch_attend<BF16>(a, cut, st->num_cus, s);
    PIMHIP_HIP_CHECK(hipGetLastError());
    return PIMHIP_OK;
}
