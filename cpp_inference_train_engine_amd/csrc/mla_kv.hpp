// The paged key-value cache: its append (kv_append.hip), the plan of its attention (kv_plan.hip),
// the attention (kv_attend.hpp, kv_merge.hip) and the sizes that all derive from a call's scalars.
// Host-visible.
#pragma once

#include "mla_internal.hpp"

namespace mla {

// A page is one record of 16-bit words: keys [n_kv_heads][page_size][head_dim], then values
// [n_kv_heads][page_size][v_dim].
__host__ __device__ inline long long kv_record(int kv_heads, int page_size, int dim, int v_dim) {
    return (long long)kv_heads * page_size * (dim + v_dim);
}
inline bool kv_supported(int page_size, int dim, int v_dim) {
    return page_size >= 16 && page_size % 16 == 0 && page_size <= 65536 && dim >= 16 &&
           dim % 16 == 0 && dim <= 256 && v_dim >= 16 && v_dim % 16 == 0 && v_dim <= 256;
}

constexpr int kKvF32 = 2;  // MLA_DTYPE_F32: type of appended rows, beside the two 16-bit ones

struct KvAppendArgs {
    int T, heads, kv_heads, dim, v_dim, page_size, num_pool_pages;
    const void *k, *v, *q;  // rows; q may be null
    long long k_row, k_head, v_row, v_head, q_row, q_head;  // strides in elements
    const int32_t *positions, *slot_mapping;
    const double* frequencies;
    int pairs, start, adjacent;
    int wide;  // every row chunk of 8 elements lies at a multiple of its size, partners included
    uint16_t *pages, *q_out;
};
hipError_t launch_kv_append(const KvAppendArgs& a, int dtype, int row_dtype, hipStream_t stream);

// ---- attention ----
// The query rows of a session that read one kv head, (token, head of the group) one behind the
// other, are its flat rows.  A job is a block of flat rows over a range of the keys that they see.
// Sessions of few flat rows go to the list of blocks of 16 or 32 (few_rows), whose four waves split
// the keys; the others to the list of blocks of 128, whose waves split the rows.
constexpr int kKvThreads = 256;
constexpr int kKvManyRows = 128;
constexpr int kKvTile = 32;     // keys of a unit
// Widths of keys that kernels exist for; their values have the same, beside 192 128.  A shape takes
// the smallest that holds it.
__host__ __device__ inline int kv_width(int dim, int v_dim) {
    return dim <= 64 && v_dim <= 64     ? 64
           : dim <= 128 && v_dim <= 128 ? 128
           : dim <= 192 && v_dim <= 128 ? 192
                                        : 256;
}

constexpr int kKvJobInts = 8;  // session, its first query row, first flat row, rows, first and last
                               // unit (of those that the block sees) + 1, ctx, first partial row
constexpr int kKvRowInts = 4;  // partials of a flat row: first, how many (0: none), step
constexpr int kKvHead = 64;    // words
enum { kKvStatus, kKvBad, kKvJobsF, kKvJobsM, kKvParts, kKvRows, kKvTag, kKvSizes = 8 };
constexpr int kKvSizeInts = 10;  // what a plan's tables and jobs follow from, from kKvSizes on

struct KvShape {
    int B, rows, H, kv_heads, group, dim, v_dim, width, page_size, max_q_len;
    int window, sinks;           // window INT32_MAX: all earlier keys
    int few_rows, few;           // rows of a block of the first list; most flat rows of its sessions
    int slots_f, slots_m;        // workgroups of a list and kv head that the GPU holds at once
    int max_jobs_f, max_jobs_m;  // of a kv head; 0: no session of these sizes can be on the list
    int max_blocks;
    long long max_parts;         // partial rows of a kv head
    long long tables_at, rows_at, jobs_f_at, jobs_m_at, words;  // word offsets
    int sizes[kKvSizeInts];      // B .. sinks as they were given, as a plan's head holds them
    uint32_t tag;                // of them, for the host's copy of a plan's info
};
KvShape kv_shape(int B, int rows, int H, int kv_heads, int dim, int v_dim, int page_size,
                 int max_q_len, int window, int sinks);

// The keys that a block of rows at positions pa .. pb sees, in units of 32 keys: those of the
// sinks, then from the window's first on (skip units lie between), count in all.
struct KvUnits {
    int sink_units, skip, count;
};
__host__ __device__ inline KvUnits kv_units(int pa, int pb, int window, int sinks) {
    const int last = pb / kKvTile + 1;
    const int lo = pa >= window ? pa - window + 1 : 0;
    const int held = sinks < pb + 1 ? sinks : pb + 1;
    const int s = (int)(((unsigned)held + kKvTile - 1) / kKvTile), first = lo / kKvTile;
    if (first <= s)
        return {last, 0, last};
    return {s, first - s, s + last - first};
}

struct KvPlanArgs {
    KvShape p;
    const int32_t *cu_q, *cu_k, *info;
    int32_t* plan;
};
hipError_t launch_kv_plan(const KvPlanArgs& a, hipStream_t stream);

struct KvArgs {
    KvShape p;
    int max_pages, num_pool_pages;
    uint32_t tpp_inverse, group_inverse;  // floor(2^32 / n) of a page's 16-key tiles and of the
                                          // group (2^32 - 1 for 1)
    int jobs_f, jobs_m;  // of a kv head, to launch: the plan's, or as many as it could have
    int parts;           // the plan's partial rows, -1: not known
    float scale_log2;    // softmax scale * log2(e)
    const int32_t *plan, *page_table;
    const uint16_t *pages, *q;
    uint16_t* out;
    float *lse, *part_o, *part_ml;
};
// Tables that other kernels wrote are read through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t* table_ptr;
__device__ __forceinline__ table_ptr table(const int32_t* p) {
    return (table_ptr)reinterpret_cast<uintptr_t>(p);
}
// Whether the call is for the plan of this head: made for the same sizes (a failed one has none), and
// where the host knows its counts, with those.
__device__ __forceinline__ bool kv_plan_fits(const KvArgs& a, table_ptr head) {
    int differ = a.parts < 0 ? 0
                             : (head[kKvJobsF] ^ a.jobs_f) | (head[kKvJobsM] ^ a.jobs_m) |
                                   (head[kKvParts] ^ a.parts);
#pragma unroll
    for (int i = 0; i < kKvSizeInts; ++i)
        differ |= head[kKvSizes + i] ^ a.p.sizes[i];
    return differ == 0;
}
hipError_t launch_kv_attention(const KvArgs& a, int dtype, hipStream_t stream);
// The lists' kernels, one translation unit for each type (kv_attend_*.hip).
hipError_t launch_kv_attend_f16(const KvArgs& a, bool many, hipStream_t stream);
hipError_t launch_kv_attend_bf16(const KvArgs& a, bool many, hipStream_t stream);

}  // namespace mla
