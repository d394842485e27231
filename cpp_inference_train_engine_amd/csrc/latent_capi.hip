// C ABI of the 8-bit latent cache and of planned attention (include/mla_hip.h): validation and
// launches.
#include "mla_capi_util.hpp"
#include "mla_hip.h"
#include "mla_latent.hpp"
#include "mla_q8.hpp"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <string>

using namespace mla;

namespace {

bool misaligned(std::initializer_list<const void*> ptrs) {
    uintptr_t u = 0;
    for (const void* p : ptrs)
        u |= reinterpret_cast<uintptr_t>(p);
    return (u & 15) != 0;
}

int invalid(const char* fn, const std::string& what) {
    return fail(MLA_ERR_INVALID_ARGUMENT, std::string(fn) + ": " + what);
}

// Shape and dtype of an 8-bit cache; MLA_OK or an error status.
int q8_shape(const char* fn, int kv_rank, int rope_dim, int page_size, int dtype,
             int num_pool_pages) {
    if (kv_rank < 1 || rope_dim < 0 || page_size < 1 || num_pool_pages < 0 ||
        (dtype != MLA_DTYPE_F16 && dtype != MLA_DTYPE_BF16))
        return invalid(fn, "invalid argument");
    if (!q8_supported(page_size, kv_rank, rope_dim))
        return fail(MLA_ERR_UNSUPPORTED,
                    std::string(fn) + ": page_size must be a multiple of 16 up to 65,536, kv_rank of "
                                      "32 up to 512, rope_dim of 8 up to 64");
    return MLA_OK;
}

constexpr long long kMaxSegments = 1 << 22;

int plan_scalars(const char* fn, int B, int rows, int n_heads, int kv_rank, int page_size,
                 int max_q_len, int n_groups) {
    if (B < 0 || rows < 0 || n_heads < 1 || kv_rank < 1 || page_size < 1 || max_q_len < 1 ||
        n_groups < 0 || n_groups > B || (long long)B + n_groups > kMaxSegments ||
        (long long)rows * n_heads > (1LL << 30))
        return invalid(fn, "invalid argument");
    const PlanShape p = plan_shape(B, n_groups, rows, n_heads, kv_rank, max_q_len);
    // (a launch has fewer than 2^32 threads)
    if (p.max_parts > 0x7fffffffLL || p.words > (1LL << 40) ||
        (long long)p.max_jobs_k * kThreadsK > 0xffffffffLL ||
        (long long)p.max_jobs_r * kThreadsR > 0xffffffffLL)
        return invalid(fn, "the batch is too large for one plan");
    return MLA_OK;
}

size_t workspace_size(const PlanShape& p) {
    return (((size_t)p.max_parts * (p.kv_rank + 2)) * sizeof(float) + 255) & ~(size_t)255;
}

}  // namespace

extern "C" {

size_t mla_q8_page_bytes(int page_size, int kv_rank, int rope_dim) {
    return q8_supported(page_size, kv_rank, rope_dim)
               ? (size_t)q8_page_bytes(page_size, kv_rank, rope_dim)
               : 0;
}

int mla_append_latent_q8(void* stream, int T, int kv_rank, int rope_dim, int page_size, int dtype,
                         const float* ckv, const float* krope, const int32_t* slot_mapping,
                         int num_pool_pages, void* pages) {
    const char* fn = "mla_append_latent_q8";
    if (T < 0)
        return invalid(fn, "invalid argument");
    if (int st = q8_shape(fn, kv_rank, rope_dim, page_size, dtype, num_pool_pages))
        return st;
    if (T == 0)
        return MLA_OK;
    if (!ckv || (rope_dim > 0 && !krope) || !slot_mapping || !pages)
        return invalid(fn, "null buffer");
    if (misaligned({pages}))
        return invalid(fn, "pages must lie at a multiple of 16 bytes");
    Q8Args a{};
    a.T = T;
    a.kv_rank = kv_rank;
    a.rope_dim = rope_dim;
    a.page_size = page_size;
    a.num_pool_pages = num_pool_pages;
    a.ckv = ckv;
    a.krope = krope;
    a.slot_mapping = slot_mapping;
    a.pages = static_cast<uint8_t*>(pages);
    return gpu_status(launch_append_q8(a, dtype, static_cast<hipStream_t>(stream)), fn);
}

int mla_read_latent_q8(void* stream, int T, int kv_rank, int rope_dim, int page_size, int dtype,
                       const int32_t* slot_mapping, int num_pool_pages, const void* pages,
                       void* ckv, void* krope) {
    const char* fn = "mla_read_latent_q8";
    if (T < 0)
        return invalid(fn, "invalid argument");
    if (int st = q8_shape(fn, kv_rank, rope_dim, page_size, dtype, num_pool_pages))
        return st;
    if (T == 0)
        return MLA_OK;
    if (!ckv || (rope_dim > 0 && !krope) || !slot_mapping || !pages)
        return invalid(fn, "null buffer");
    if (misaligned({pages, ckv, krope}))
        return invalid(fn, "pages, ckv and krope must lie at multiples of 16 bytes");
    Q8Args a{};
    a.T = T;
    a.kv_rank = kv_rank;
    a.rope_dim = rope_dim;
    a.page_size = page_size;
    a.num_pool_pages = num_pool_pages;
    a.slot_mapping = slot_mapping;
    a.pages = static_cast<uint8_t*>(const_cast<void*>(pages));
    a.ckv16 = static_cast<uint16_t*>(ckv);
    a.krope16 = static_cast<uint16_t*>(krope);
    return gpu_status(launch_read_q8(a, dtype, static_cast<hipStream_t>(stream)), fn);
}

size_t mla_attention_plan_bytes(int B, int rows, int n_heads, int kv_rank, int max_q_len,
                                int n_groups) {
    if (plan_scalars("mla_attention_plan_bytes", B, rows, n_heads, kv_rank, 1, max_q_len, n_groups))
        return 0;
    return (size_t)plan_shape(B, n_groups, rows, n_heads, kv_rank, max_q_len).words *
           sizeof(int32_t);
}

size_t mla_attention_workspace_bytes(int B, int rows, int n_heads, int kv_rank, int max_q_len,
                                     int n_groups) {
    if (plan_scalars("mla_attention_workspace_bytes", B, rows, n_heads, kv_rank, 1, max_q_len,
                     n_groups))
        return 0;
    return workspace_size(plan_shape(B, n_groups, rows, n_heads, kv_rank, max_q_len));
}

int mla_plan_attention(void* stream, int B, int rows, int n_heads, int kv_rank, int page_size,
                       int max_q_len, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                       const int32_t* info, int n_groups, const int32_t* cu_groups,
                       const int32_t* prefix_len, const int32_t* cu_prefix_pages,
                       const int32_t* prefix_page_ids, int n_prefix_pages, int num_pool_pages,
                       void* plan, size_t plan_bytes) {
    const char* fn = "mla_plan_attention";
    if (int st = plan_scalars(fn, B, rows, n_heads, kv_rank, page_size, max_q_len, n_groups))
        return st;
    if (n_prefix_pages < 0 || num_pool_pages < 0)
        return invalid(fn, "invalid argument");
    if (!cu_seqlens_q || !cu_seqlens_k || !info || !plan ||
        (n_groups > 0 && (!cu_groups || !prefix_len || !cu_prefix_pages ||
                          (n_prefix_pages > 0 && !prefix_page_ids))))
        return invalid(fn, "null buffer");
    PlanArgs a{};
    a.p = plan_shape(B, n_groups, rows, n_heads, kv_rank, max_q_len);
    a.p.tag = plan_tag(a.p, page_size, n_groups > 0 && prefix_page_ids);
    const size_t need = (size_t)a.p.words * sizeof(int32_t);
    if (plan_bytes < need || misaligned({plan}))
        return invalid(fn, "the plan needs " + std::to_string(need) +
                               " bytes at a multiple of 16");
    a.page_size = page_size;
    a.num_pool_pages = num_pool_pages;
    a.n_prefix_pages = n_prefix_pages;
    a.cu_q = cu_seqlens_q;
    a.cu_k = cu_seqlens_k;
    a.info = info;
    a.cu_groups = cu_groups;
    a.prefix_len = prefix_len;
    a.cu_prefix_pages = cu_prefix_pages;
    a.prefix_page_ids = prefix_page_ids;
    a.plan = static_cast<int32_t*>(plan);
    return gpu_status(launch_plan(a, static_cast<hipStream_t>(stream)), fn);
}

int mla_read_plan_info(void* stream, const void* plan, int32_t* host_info) {
    const char* fn = "mla_read_plan_info";
    if (!plan || !host_info)
        return invalid(fn, "null buffer");
    auto s = static_cast<hipStream_t>(stream);
    hipError_t e = hipMemcpyAsync(host_info, plan, MLA_PLAN_INFO_INTS * sizeof(int32_t),
                                  hipMemcpyDeviceToHost, s);
    if (e == hipSuccess)
        e = hipStreamSynchronize(s);
    if (int st = gpu_status(e, fn))
        return st;
    if (host_info[kPlanStatus] >= 0)
        return MLA_OK;
    const int bad = host_info[kPlanBad];
    return invalid(fn, bad == -1 ? "the batch's metadata build failed, or it has more rows than "
                                   "the plan"
                       : bad == -2 ? "the batch does not fit the plan's tables"
                                   : "entry " + std::to_string(bad) +
                                         " (the groups, then the sessions): a group's sessions, "
                                         "prefix length, page list or page id is out of range, or "
                                         "a session has more rows than max_q_len");
}

int mla_latent_attention(void* stream, int B, int rows, int n_heads, int kv_rank, int rope_dim,
                         int page_size, int max_q_len, int dtype, int cache_format, float scale,
                         const int32_t* page_table, int max_pages, int num_pool_pages,
                         const void* pages, const void* q_latent, const void* q_rope, int n_groups,
                         const int32_t* cu_prefix_pages, const int32_t* prefix_page_ids,
                         const void* plan, size_t plan_bytes, const int32_t* host_info, void* out,
                         float* lse, void* workspace, size_t workspace_bytes) {
    const char* fn = "mla_latent_attention";
    if (int st = plan_scalars(fn, B, rows, n_heads, kv_rank, page_size, max_q_len, n_groups))
        return st;
    if (max_pages < 0 || !(scale > 0.0f) || std::isinf(scale) ||
        (cache_format != MLA_CACHE_16BIT && cache_format != MLA_CACHE_Q8))
        return invalid(fn, "invalid argument");
    if (int st = q8_shape(fn, kv_rank, rope_dim, page_size, dtype, num_pool_pages))
        return st;
    if (B == 0 || rows == 0)
        return MLA_OK;
    if (!page_table || !pages || !q_latent || (rope_dim > 0 && !q_rope) || !plan || !out ||
        !workspace || (n_groups > 0 && !cu_prefix_pages))
        return invalid(fn, "null buffer");
    if (misaligned({pages, q_latent, q_rope, plan, out, workspace}))
        return invalid(fn, "pages, q_latent, q_rope, plan, out and workspace must lie at multiples "
                           "of 16 bytes");
    LatentArgs a{};
    a.p = plan_shape(B, n_groups, rows, n_heads, kv_rank, max_q_len);
    a.p.tag = plan_tag(a.p, page_size, n_groups > 0 && prefix_page_ids);
    if (plan_bytes < (size_t)a.p.words * sizeof(int32_t))
        return invalid(fn, "the plan was made for other sizes");
    a.jobs_k = a.p.max_jobs_k;
    a.jobs_r = a.p.max_jobs_r;
    a.parts = -1;
    if (host_info) {
        if (host_info[kPlanTag] != (int)a.p.tag || host_info[kPlanJobsK] < 0 ||
            host_info[kPlanJobsK] > a.jobs_k || host_info[kPlanJobsR] < 0 ||
            host_info[kPlanJobsR] > a.jobs_r || host_info[kPlanParts] < 0)
            return invalid(fn, "host_info is not that of a plan for these sizes");
        a.jobs_k = host_info[kPlanJobsK];
        a.jobs_r = host_info[kPlanJobsR];
        a.parts = host_info[kPlanParts];
    }
    if (workspace_bytes < workspace_size(a.p))
        return invalid(fn, "workspace needs " + std::to_string(workspace_size(a.p)) + " bytes");
    a.H = n_heads;
    a.kv_rank = kv_rank;
    a.rope_dim = rope_dim;
    a.page_size = page_size;
    a.max_pages = max_pages;
    a.num_pool_pages = num_pool_pages;
    auto inverse = [](int n) { return (uint32_t)std::min<uint64_t>((1ULL << 32) / n, 0xffffffffULL); };
    a.tpp_inverse = inverse(page_size / 16);
    a.h_inverse = inverse(n_heads);
    a.causal = max_q_len > 1;
    a.q8 = cache_format == MLA_CACHE_Q8;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.plan = static_cast<const int32_t*>(plan);
    a.page_table = page_table;
    a.cu_prefix_pages = cu_prefix_pages;
    a.prefix_page_ids = prefix_page_ids;
    a.pages = static_cast<const uint8_t*>(pages);
    a.q_latent = static_cast<const uint16_t*>(q_latent);
    a.q_rope = static_cast<const uint16_t*>(q_rope);
    a.out = static_cast<uint16_t*>(out);
    a.lse = lse;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + a.p.max_parts * kv_rank;
    return gpu_status(launch_latent_attention(a, dtype, static_cast<hipStream_t>(stream)), fn);
}

}  // extern "C"
