// C ABI of the paged key-value cache (include/mla_hip.h, section (f)): validation and launches.
#include "mla_capi_util.hpp"
#include "mla_hip.h"
#include "mla_kv.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
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

// Whether two stretches of bytes have one in common.
bool overlap(const void* a, long long a_bytes, const void* b, long long b_bytes) {
    const char *const x = static_cast<const char*>(a), *const y = static_cast<const char*>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

int invalid(const char* fn, const std::string& what) {
    return fail(MLA_ERR_INVALID_ARGUMENT, std::string(fn) + ": " + what);
}

// Shape of a cache; MLA_OK or an error status.
int cache_shape(const char* fn, int n_heads, int n_kv_heads, int head_dim, int v_dim,
                int page_size) {
    if (n_heads < 1 || n_kv_heads < 1 || head_dim < 1 || v_dim < 1 || page_size < 1)
        return invalid(fn, "invalid argument");
    if (!kv_supported(page_size, head_dim, v_dim))
        return fail(MLA_ERR_UNSUPPORTED,
                    std::string(fn) + ": page_size must be a multiple of 16 up to 65,536, head_dim "
                                      "and v_dim multiples of 16 up to 256");
    if (kv_record(n_kv_heads, page_size, head_dim, v_dim) > INT_MAX)
        return fail(MLA_ERR_UNSUPPORTED, std::string(fn) + ": a page record is larger than 4 GiB");
    return MLA_OK;
}

int plan_scalars(const char* fn, int B, int rows, int n_heads, int n_kv_heads, int head_dim,
                 int v_dim, int page_size, int max_q_len, int window, int sinks) {
    if (int st = cache_shape(fn, n_heads, n_kv_heads, head_dim, v_dim, page_size))
        return st;
    if (n_heads % n_kv_heads != 0)
        return invalid(fn, "n_heads must be a multiple of n_kv_heads");
    if (B < 0 || rows < 0 || max_q_len < 1 || window < 0 || sinks < 0 ||
        (long long)rows * n_heads > (1LL << 30) || B > (1 << 22))
        return invalid(fn, "invalid argument");
    if (sinks > 0 && window == 0)
        return invalid(fn, "sinks without a window");
    const KvShape p = kv_shape(B, rows, n_heads, n_kv_heads, head_dim, v_dim, page_size, max_q_len,
                               window ? window : INT_MAX, sinks);
    // (a launch has fewer than 2^32 threads; kv_many_kernel has twice as many at width 256)
    const int many_threads = p.width == 256 ? 2 * kKvThreads : kKvThreads;
    if (p.max_parts * n_kv_heads > INT_MAX || p.words > (1LL << 40) ||
        (long long)p.max_jobs_f * n_kv_heads * kKvThreads > 0xffffffffLL ||
        (long long)p.max_jobs_m * n_kv_heads * many_threads > 0xffffffffLL)
        return invalid(fn, "the batch is too large for one plan");
    return MLA_OK;
}

size_t workspace_size(const KvShape& p) {
    return (((size_t)p.max_parts * p.kv_heads * (p.v_dim + 2)) * sizeof(float) + 255) & ~(size_t)255;
}

}  // namespace

extern "C" {

size_t mla_kv_page_words(int n_kv_heads, int head_dim, int v_dim, int page_size) {
    if (cache_shape("mla_kv_page_words", n_kv_heads, n_kv_heads, head_dim, v_dim, page_size))
        return 0;
    return (size_t)kv_record(n_kv_heads, page_size, head_dim, v_dim);
}

int mla_append_kv(void* stream, int T, int n_heads, int n_kv_heads, int head_dim, int v_dim,
                  int page_size, int dtype, int row_dtype, const void* k, long long k_row,
                  long long k_head, const void* v, long long v_row, long long v_head, const void* q,
                  long long q_row, long long q_head, const int32_t* positions,
                  const double* frequencies, int pairs, int rotary_start, int adjacent,
                  const int32_t* slot_mapping, int num_pool_pages, void* pages, void* q_out) {
    const char* fn = "mla_append_kv";
    if (int st = cache_shape(fn, n_heads, n_kv_heads, head_dim, v_dim, page_size))
        return st;
    if (T < 0 || num_pool_pages < 0 || (dtype != MLA_DTYPE_F16 && dtype != MLA_DTYPE_BF16) ||
        (row_dtype != MLA_DTYPE_F16 && row_dtype != MLA_DTYPE_BF16 && row_dtype != MLA_DTYPE_F32) ||
        (adjacent != 0 && adjacent != 1))
        return invalid(fn, "invalid argument");
    if (pairs < 0 || rotary_start < 0 || rotary_start % 2 != 0 || pairs > head_dim / 2 ||
        rotary_start > head_dim - 2 * pairs)
        return invalid(fn, "the rotated columns, 2 pairs from an even rotary_start on, must lie "
                           "within head_dim");
    if (((long long)n_heads + n_kv_heads) * head_dim + (long long)n_kv_heads * v_dim > INT_MAX)
        return fail(MLA_ERR_UNSUPPORTED, std::string(fn) + ": a token's rows have more than 2^31 columns");
    if (T == 0)
        return MLA_OK;
    if (!k || !v || !slot_mapping || !pages || (q && !q_out) ||
        (pairs > 0 && (!positions || !frequencies)))
        return invalid(fn, "null buffer");
    if (misaligned({pages, q ? q_out : nullptr}))
        return invalid(fn, "pages and q_out must lie at multiples of 16 bytes");
    const int size = row_dtype == MLA_DTYPE_F32 ? 4 : 2;
    if (q) {  // workgroups write q_out while others still read their rows
        auto covers = [&](const void* rows, long long row, long long head, int heads, int columns) {
            const long long far[2] = {(T - 1LL) * row, (heads - 1LL) * head};
            const char* const from = static_cast<const char*>(rows);
            return overlap(q_out, 2LL * T * n_heads * head_dim,
                           from + (std::min(far[0], 0LL) + std::min(far[1], 0LL)) * size,
                           (std::abs(far[0]) + std::abs(far[1]) + columns) * size);
        };
        if (covers(q, q_row, q_head, n_heads, head_dim))
            return invalid(fn, "q_out overlaps q");
        if (covers(k, k_row, k_head, n_kv_heads, head_dim) || covers(v, v_row, v_head, n_kv_heads, v_dim))
            return invalid(fn, "q_out overlaps k or v");
        if (overlap(q_out, 2LL * T * n_heads * head_dim, pages,
                    2LL * num_pool_pages * kv_record(n_kv_heads, page_size, head_dim, v_dim)))
            return invalid(fn, "q_out overlaps the pages");
    }
    KvAppendArgs a{};
    a.T = T;
    a.heads = n_heads;
    a.kv_heads = n_kv_heads;
    a.dim = head_dim;
    a.v_dim = v_dim;
    a.page_size = page_size;
    a.num_pool_pages = num_pool_pages;
    a.k = k;
    a.v = v;
    a.q = q;
    a.k_row = k_row;
    a.k_head = k_head;
    a.v_row = v_row;
    a.v_head = v_head;
    a.q_row = q_row;
    a.q_head = q_head;
    a.positions = positions;
    a.slot_mapping = slot_mapping;
    a.frequencies = frequencies;
    a.pairs = pairs;
    a.start = rotary_start;
    a.adjacent = adjacent;
    // 16-byte loads: rows that start at multiples of 16 bytes, and for split halves chunks of 8
    // columns whose partners are one chunk.
    unsigned long long u = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                           reinterpret_cast<uintptr_t>(q);
    for (const long long s : {k_row, k_head, v_row, v_head, q ? q_row : 0, q ? q_head : 0})
        u |= (unsigned long long)s * size;
    a.wide = u % 16 == 0 && (adjacent || (pairs % 8 == 0 && rotary_start % 8 == 0));
    a.pages = static_cast<uint16_t*>(pages);
    a.q_out = static_cast<uint16_t*>(q_out);
    return gpu_status(launch_kv_append(a, dtype, row_dtype, static_cast<hipStream_t>(stream)), fn);
}

size_t mla_kv_plan_bytes(int B, int rows, int n_heads, int n_kv_heads, int head_dim, int v_dim,
                         int page_size, int max_q_len, int window, int sinks) {
    if (plan_scalars("mla_kv_plan_bytes", B, rows, n_heads, n_kv_heads, head_dim, v_dim, page_size,
                     max_q_len, window, sinks))
        return 0;
    return (size_t)kv_shape(B, rows, n_heads, n_kv_heads, head_dim, v_dim, page_size, max_q_len,
                            window ? window : INT_MAX, sinks)
               .words *
           sizeof(int32_t);
}

size_t mla_kv_workspace_bytes(int B, int rows, int n_heads, int n_kv_heads, int head_dim, int v_dim,
                              int page_size, int max_q_len, int window, int sinks) {
    if (plan_scalars("mla_kv_workspace_bytes", B, rows, n_heads, n_kv_heads, head_dim, v_dim,
                     page_size, max_q_len, window, sinks))
        return 0;
    return workspace_size(kv_shape(B, rows, n_heads, n_kv_heads, head_dim, v_dim, page_size,
                                   max_q_len, window ? window : INT_MAX, sinks));
}

int mla_plan_kv_attention(void* stream, int B, int rows, int n_heads, int n_kv_heads, int head_dim,
                          int v_dim, int page_size, int max_q_len, int window, int sinks,
                          const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                          const int32_t* info, void* plan, size_t plan_bytes) {
    const char* fn = "mla_plan_kv_attention";
    if (int st = plan_scalars(fn, B, rows, n_heads, n_kv_heads, head_dim, v_dim, page_size,
                              max_q_len, window, sinks))
        return st;
    if (!cu_seqlens_q || !cu_seqlens_k || !info || !plan)
        return invalid(fn, "null buffer");
    KvPlanArgs a{};
    a.p = kv_shape(B, rows, n_heads, n_kv_heads, head_dim, v_dim, page_size, max_q_len,
                   window ? window : INT_MAX, sinks);
    const size_t need = (size_t)a.p.words * sizeof(int32_t);
    if (plan_bytes < need || misaligned({plan}))
        return invalid(fn, "the plan needs " + std::to_string(need) +
                               " bytes at a multiple of 16");
    a.cu_q = cu_seqlens_q;
    a.cu_k = cu_seqlens_k;
    a.info = info;
    a.plan = static_cast<int32_t*>(plan);
    return gpu_status(launch_kv_plan(a, static_cast<hipStream_t>(stream)), fn);
}

int mla_read_kv_plan_info(void* stream, const void* plan, int32_t* host_info) {
    const char* fn = "mla_read_kv_plan_info";
    if (!plan || !host_info)
        return invalid(fn, "null buffer");
    auto s = static_cast<hipStream_t>(stream);
    hipError_t e = hipMemcpyAsync(host_info, plan, MLA_PLAN_INFO_INTS * sizeof(int32_t),
                                  hipMemcpyDeviceToHost, s);
    if (e == hipSuccess)
        e = hipStreamSynchronize(s);
    if (int st = gpu_status(e, fn))
        return st;
    if (host_info[kKvStatus] >= 0)
        return MLA_OK;
    const int bad = host_info[kKvBad];
    return invalid(fn, bad == -1 ? "the batch's metadata build failed, or it has more rows than "
                                   "the plan"
                       : bad == -2 ? "the batch does not fit the plan's tables"
                                   : "session " + std::to_string(bad) +
                                         " has more rows than max_q_len");
}

int mla_kv_attention(void* stream, int B, int rows, int n_heads, int n_kv_heads, int head_dim,
                     int v_dim, int page_size, int max_q_len, int window, int sinks, int dtype,
                     float scale, const int32_t* page_table, int max_pages, int num_pool_pages,
                     const void* pages, const void* q, const void* plan, size_t plan_bytes,
                     const int32_t* host_info, void* out, float* lse, void* workspace,
                     size_t workspace_bytes) {
    const char* fn = "mla_kv_attention";
    if (int st = plan_scalars(fn, B, rows, n_heads, n_kv_heads, head_dim, v_dim, page_size,
                              max_q_len, window, sinks))
        return st;
    if (max_pages < 0 || num_pool_pages < 0 || !(scale > 0.0f) || std::isinf(scale) ||
        (dtype != MLA_DTYPE_F16 && dtype != MLA_DTYPE_BF16))
        return invalid(fn, "invalid argument");
    if (B == 0 || rows == 0 || max_pages == 0 || num_pool_pages == 0)  // (no session has a key)
        return MLA_OK;
    if (!page_table || !pages || !q || !plan || !out || !workspace)
        return invalid(fn, "null buffer");
    if (misaligned({pages, q, plan, out, workspace}))
        return invalid(fn, "pages, q, plan, out and workspace must lie at multiples of 16 bytes");
    KvArgs a{};
    a.p = kv_shape(B, rows, n_heads, n_kv_heads, head_dim, v_dim, page_size, max_q_len,
                   window ? window : INT_MAX, sinks);
    if (plan_bytes < (size_t)a.p.words * sizeof(int32_t))
        return invalid(fn, "the plan was made for other sizes");
    a.jobs_f = a.p.max_jobs_f;
    a.jobs_m = a.p.max_jobs_m;
    a.parts = -1;
    if (host_info) {
        if (host_info[kKvTag] != (int)a.p.tag || host_info[kKvJobsF] < 0 ||
            host_info[kKvJobsF] > a.jobs_f || host_info[kKvJobsM] < 0 ||
            host_info[kKvJobsM] > a.jobs_m || host_info[kKvParts] < 0)
            return invalid(fn, "host_info is not that of a plan for these sizes");
        a.jobs_f = host_info[kKvJobsF];
        a.jobs_m = host_info[kKvJobsM];
        a.parts = host_info[kKvParts];
    }
    if (workspace_bytes < workspace_size(a.p))
        return invalid(fn, "workspace needs " + std::to_string(workspace_size(a.p)) + " bytes");
    // (a row of out may take the place of the row of q that it follows from: its job alone reads that)
    struct Stretch {
        const void* at;
        long long bytes;
    };
    const long long words = (long long)rows * n_heads;
    const long long record = kv_record(n_kv_heads, page_size, head_dim, v_dim);
    const Stretch own[] = {{out, 2 * words * v_dim},
                           {lse, lse ? 4 * words : 0},
                           {workspace, (long long)workspace_size(a.p)}};
    const Stretch read[] = {{q, 2 * words * head_dim}, {pages, 2 * num_pool_pages * record}};
    for (const Stretch& x : own) {
        bool apart = true;
        for (const Stretch& y : own)
            apart &= &x == &y || !overlap(x.at, x.bytes, y.at, y.bytes);
        for (const Stretch& y : read)
            apart &= (x.at == out && y.at == q && q == out && head_dim == v_dim) ||
                     !overlap(x.at, x.bytes, y.at, y.bytes);
        if (!apart)
            return invalid(fn, "out, lse and workspace must lie apart from each other, q (out may be q "
                               "itself where head_dim is v_dim) and the pages");
    }
    a.max_pages = max_pages;
    a.num_pool_pages = num_pool_pages;
    auto inverse = [](int n) { return (uint32_t)std::min<uint64_t>((1ULL << 32) / n, 0xffffffffULL); };
    a.tpp_inverse = inverse(page_size / 16);
    a.group_inverse = inverse(a.p.group);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.plan = static_cast<const int32_t*>(plan);
    a.page_table = page_table;
    a.pages = static_cast<const uint16_t*>(pages);
    a.q = static_cast<const uint16_t*>(q);
    a.out = static_cast<uint16_t*>(out);
    a.lse = lse;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + a.p.max_parts * n_kv_heads * v_dim;
    return gpu_status(launch_kv_attention(a, dtype, static_cast<hipStream_t>(stream)), fn);
}

}  // extern "C"
