// Planned attention over the paged latent cache (latent_attend.hpp, latent_merge.hip), its plan
// (attention_plan.hip) and the sizes both derive from a call's scalars.  Host-visible.
#pragma once

#include "mla_internal.hpp"

namespace mla {

// A segment is a run of keys that a set of consecutive query rows sees: a session's own pages
// with its rows, or a group's shared prefix with the rows of all of the group's sessions.  A job
// is one block of a segment's (query, head) rows over one range of its keys.  Segments with few
// rows go to list K (16 rows a job; its four waves split the keys), the others to list R (128 rows;
// its eight waves split them).
constexpr int kRowsK = 16, kRowsR = 128;  // rows of a block
constexpr int kThreadsK = 256, kThreadsR = 512;
constexpr int kTile = 32;    // keys of a unit
constexpr int kJobInts = 8;  // segment (>= 0 session, ~group), first flat row, rows, first row's
                             // index in the segment, first key, last key + 1, ctx, partial row
// A row's partials: how many of its prefix, of its own keys, the first of either (of its head 0), and
// from one to the next of either.
constexpr int kMergeInts = 8;
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
constexpr int kPlanHead = 64;  // words
enum { kPlanStatus, kPlanBad, kPlanJobsK, kPlanJobsR, kPlanParts, kPlanRows, kPlanTag };

// What a plan and the calls over it derive from the same scalars.
struct PlanShape {
    int B, groups, rows, H, kv_rank, max_q_len;
    int slots_k, slots_r;        // workgroups of a list that the GPU holds at once
    bool list_k_holds_all;       // list K has room for the segments of many rows, too
    int max_jobs_k, max_jobs_r;  // 0: no segment of these sizes can be on the list
    long long max_parts;         // (query, head) rows of partials
    long long seg_at, merge_at, jobs_k_at, jobs_r_at, words;  // word offsets
    uint32_t tag;  // plan_tag
};
PlanShape plan_shape(int B, int groups, int rows, int H, int kv_rank, int max_q_len);
// What a plan and its calls have to agree on: the sizes, the page size (page lists are indexed by
// it), and whether there is a list of prefix pages to index.
uint32_t plan_tag(const PlanShape& p, int page_size, bool prefix_pages);

struct PlanArgs {
    PlanShape p;
    int page_size, num_pool_pages, n_prefix_pages;
    const int32_t *cu_q, *cu_k, *info, *cu_groups, *prefix_len, *cu_prefix_pages,
        *prefix_page_ids;
    int32_t* plan;
};
hipError_t launch_plan(const PlanArgs& a, hipStream_t stream);

struct LatentArgs {
    PlanShape p;
    int H, kv_rank, rope_dim, page_size, max_pages, num_pool_pages;
    int causal;        // the rows of a block may see different keys
    int q8;
    uint32_t tpp_inverse, h_inverse;  // floor(2^32 / n) of a page's tiles and of H (2^32 - 1 for 1)
    int jobs_k, jobs_r;  // workgroups to launch: the plan's jobs, or as many as it could have
    int parts;           // the plan's partial rows, -1: not known (there may be some)
    float scale_log2;  // softmax scale * log2(e)
    const int32_t *plan, *page_table, *cu_prefix_pages, *prefix_page_ids;
    const uint8_t* pages;
    const uint16_t *q_latent, *q_rope;
    uint16_t* out;
    float *lse, *part_o, *part_ml;
};
// Whether the call is for this plan (its head): made for the same sizes, and where the host knows
// its counts, with those.
__host__ __device__ inline bool plan_fits(const LatentArgs& a, int tag, int jobs_k, int jobs_r,
                                          int parts) {
    return tag == (int)a.p.tag &&
           (a.parts < 0 || (jobs_k == a.jobs_k && jobs_r == a.jobs_r && parts == a.parts));
}
hipError_t launch_latent_attention(const LatentArgs& a, int dtype, hipStream_t stream);
hipError_t launch_latent_merge(const LatentArgs& a, int dtype, hipStream_t stream);
// The lists' kernels, one translation unit for each cache format (latent_attend_*.hip).
hipError_t launch_attend_16(const LatentArgs& a, int dtype, bool rows, hipStream_t stream);
hipError_t launch_attend_q8(const LatentArgs& a, int dtype, bool rows, hipStream_t stream);

}  // namespace mla
