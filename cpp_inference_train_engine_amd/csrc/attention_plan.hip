// The plan of mla_latent_attention: which workgroup takes which rows over which keys, built on
// the GPU once for a batch and used by every layer's call.  No reference counterpart.
//
// One workgroup.  For each segment (mla_latent.hpp) it takes the row blocks and the 32-key tiles,
// cuts the keys of all segments into ranges of one length per list, so that a list has about its
// target of jobs, and lays out jobs, partial rows and, per session, what the merge has to add up.
// Everything is scanned in one pass over the segments with a running carry, so any batch size
// works; the tables live in the plan itself.
#include "mla_latent.hpp"

#include <algorithm>

namespace mla {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

__device__ __forceinline__ long long wave_scan(long long v, int lane) {
    for (int d = 1; d < 64; d <<= 1) {
        const long long u = __shfl_up(v, d, 64);
        if (lane >= d)
            v += u;
    }
    return v;
}

// Inclusive scan over the workgroup; `total` receives the sum.  `tmp`: kWaves values in LDS.
__device__ long long block_scan(long long v, long long* tmp, long long& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v, lane);
    __syncthreads();
    if (lane == 63)
        tmp[wave] = v;
    __syncthreads();
    long long before = 0;
    total = 0;
    for (int w = 0; w < kWaves; ++w) {
        const long long x = tmp[w];
        before += w < wave ? x : 0;
        total += x;
    }
    return v + before;
}

struct Seg {
    long long n;  // (query, head) rows
    int tiles, keys, blocks, q0, q_len, few;
};

__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
    __shared__ long long tmp[kWaves];
    __shared__ int first_bad;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const PlanShape& p = a.p;
    const int B = p.B, G = p.groups, S = G + B, H = p.H;
    int32_t* head = a.plan;
    int32_t* segs = a.plan + p.seg_at;
    int32_t* merges = a.plan + p.merge_at;
    int32_t* session_of = a.plan + p.session_at;
    const int total_q = a.info[0] < 0 ? -1 : a.cu_q[B];

    // ---- checks: the metadata, the sessions' rows, the groups and their pages ----
    if (tid == 0)
        first_bad = 0x7fffffff;
    __syncthreads();
    if (total_q < 0 || total_q > p.rows) {
        if (tid == 0)
            first_bad = -1;  // a failed metadata build, or more rows than the call's
    } else {
        for (int s = tid; s < B; s += kThreads)
            if (a.cu_q[s + 1] - a.cu_q[s] > p.max_q_len)
                atomicMin(&first_bad, G + s);
        for (int g = tid; g < G; g += kThreads) {
            const int s0 = a.cu_groups[g], s1 = a.cu_groups[g + 1], len = a.prefix_len[g];
            const int c0 = a.cu_prefix_pages[g], c1 = a.cu_prefix_pages[g + 1];
            if (s0 < 0 || s1 < s0 || s1 > B || len < 0 || c0 < 0 || c1 < c0 ||
                c1 > a.n_prefix_pages || (long long)(c1 - c0) * a.page_size < len)
                atomicMin(&first_bad, g);
        }
        __syncthreads();
        for (int g = wave; g < G; g += kWaves) {  // a bad group's list may lie anywhere
            const int c0 = a.cu_prefix_pages[g], c1 = a.cu_prefix_pages[g + 1];
            if (c0 < 0 || c1 > a.n_prefix_pages)
                continue;
            for (int i = c0 + lane; i < c1; i += 64)
                if ((unsigned)a.prefix_page_ids[i] >= (unsigned)a.num_pool_pages)
                    atomicMin(&first_bad, g);
        }
    }
    __syncthreads();
    if (first_bad != 0x7fffffff) {
        if (tid < kPlanHead)
            head[tid] = tid == kPlanStatus ? -1 : tid == kPlanBad ? first_bad : 0;
        return;
    }

    // ---- which prefix a session has ----
    for (int s = tid; s < B; s += kThreads)
        for (int i = 0; i < kMergeInts; ++i)
            merges[(long long)s * kMergeInts + i] = 0;
    __syncthreads();
    for (int g = wave; g < G; g += kWaves)
        if (a.prefix_len[g] > 0)
            for (int s = a.cu_groups[g] + lane; s < a.cu_groups[g + 1]; s += 64)
                merges[(long long)s * kMergeInts] = 1;
    __syncthreads();

    auto segment = [&](int i) {
        Seg x{};
        if (i < G) {
            x.q0 = a.cu_q[a.cu_groups[i]];
            x.q_len = a.cu_q[a.cu_groups[i + 1]] - x.q0;
            x.keys = a.prefix_len[i];
        } else {
            x.q0 = a.cu_q[i - G];
            x.q_len = a.cu_q[i - G + 1] - x.q0;
            x.keys = a.cu_k[i - G + 1] - a.cu_k[i - G];
        }
        if (x.q_len <= 0 || x.keys <= 0)
            return x;
        x.n = (long long)x.q_len * H;
        x.few = x.n <= kFewRows;
        const int rows = x.few ? 16 * p.qt : kRowsR;
        x.blocks = (int)((x.n + rows - 1) / rows);
        x.tiles = (int)(((long long)x.keys + kTile - 1) / kTile);
        return x;
    };

    // ---- the length of a key range, per list: about target jobs in all ----
    long long cost_k = 0, cost_r = 0, all;
    for (int i = tid; i < S; i += kThreads) {
        const Seg x = segment(i);
        (x.few ? cost_k : cost_r) += (long long)x.blocks * x.tiles;
    }
    block_scan(cost_k, tmp, all);
    cost_k = all;
    block_scan(cost_r, tmp, all);
    cost_r = all;
    auto range = [](long long cost, int target, int least) {
        return std::max<long long>((cost + target - 1) / target, least);
    };
    const long long len_k = range(cost_k, p.target_k, p.least_k);
    const long long len_r = range(cost_r, p.target_r, p.least_r);

    // ---- jobs and partial rows of each segment ----
    long long at_k = 0, at_r = 0, at_part = 0;
    for (int i0 = 0; i0 < S; i0 += kThreads) {
        const int i = i0 + tid;
        Seg x{};
        if (i < S)
            x = segment(i);
        int splits = 0, len = 0;
        if (x.blocks > 0) {
            const long long most = x.few ? len_k : len_r;
            splits = (int)((x.tiles + most - 1) / most);
            len = (x.tiles + splits - 1) / splits;
            if (x.few)
                len = (len + 3) & ~3;  // the four waves of a list-K job take a tile each
            splits = (x.tiles + len - 1) / len;
        }
        const bool joined =
            x.blocks > 0 && (splits > 1 || i < G || merges[(long long)(i - G) * kMergeInts] != 0);
        const long long jobs = (long long)x.blocks * splits;
        const long long parts = joined ? x.n * splits : 0;
        long long sum;
        const long long jk = block_scan(x.few ? jobs : 0, tmp, sum) + at_k - (x.few ? jobs : 0);
        at_k += sum;
        const long long jr = block_scan(x.few ? 0 : jobs, tmp, sum) + at_r - (x.few ? 0 : jobs);
        at_r += sum;
        const long long pt = block_scan(parts, tmp, sum) + at_part - parts;
        at_part += sum;
        if (i < S) {
            int32_t* d = segs + (long long)i * kSegInts;
            d[0] = x.few;
            d[1] = (int)std::min<long long>(x.few ? jk : jr, 0x7fffffff);
            d[2] = splits;
            d[3] = len;
            d[4] = joined ? (int)std::min<long long>(pt, 0x7fffffff) : -1;
            d[5] = x.blocks;
        }
    }
    __syncthreads();
    const bool fits = at_k <= p.max_jobs_k && at_r <= p.max_jobs_r && at_part <= p.max_parts;
    if (tid < kPlanHead) {
        int v = 0;
        if (fits)
            v = tid == kPlanStatus ? (int)(at_k + at_r)
                : tid == kPlanJobsK ? (int)at_k
                : tid == kPlanJobsR ? (int)at_r
                : tid == kPlanParts ? (int)at_part
                : tid == kPlanRows  ? total_q
                : tid == kPlanTag   ? (int)p.tag
                                    : 0;
        else
            v = tid == kPlanStatus ? -1 : tid == kPlanBad ? -2 : 0;
        head[tid] = v;
    }
    if (!fits)
        return;

    // ---- the jobs; what the merge adds up for a session; the session of each row ----
    for (int i = wave; i < S; i += kWaves) {
        const Seg x = segment(i);
        const int32_t* d = segs + (long long)i * kSegInts;
        const int job0 = d[1], splits = d[2], len = d[3], part0 = d[4], blocks = d[5];
        if (i < G) {
            for (int s = a.cu_groups[i] + lane; s < a.cu_groups[i + 1]; s += 64) {
                int32_t* m = merges + (long long)s * kMergeInts;
                m[0] = blocks > 0 ? splits : 0;
                m[1] = part0;
                m[2] = (int)x.n;
                m[3] = (a.cu_q[s] - x.q0) * H;
            }
        } else {
            if (lane == 0) {
                int32_t* m = merges + (long long)(i - G) * kMergeInts;
                m[4] = part0 >= 0 ? splits : 0;
                m[5] = part0;
                m[6] = (int)x.n;
                m[7] = x.q0;
            }
            for (int r = lane; r < x.q_len; r += 64)
                session_of[x.q0 + r] = i - G;
        }
        const int rows = x.few ? 16 * p.qt : kRowsR;
        int32_t* list = a.plan + (x.few ? p.jobs_k_at : p.jobs_r_at);
        const int ctx = i < G ? x.keys : x.keys - x.q_len;
        for (int j = lane; j < blocks * splits; j += 64) {
            const int sp = j / blocks, rb = (j - sp * blocks) * rows;
            const int n = (int)std::min<long long>(rows, x.n - rb);
            const long long k0 = (long long)sp * len * kTile;
            // own keys: the block's last row sees keys up to its own token
            const int seen = i < G ? x.keys : ctx + (rb + n - 1) / H + 1;
            int32_t* o = list + (long long)(job0 + j) * kJobInts;
            o[0] = i < G ? ~i : i - G;
            o[1] = (int)((long long)x.q0 * H + rb);
            o[2] = n;
            o[3] = rb;
            o[4] = (int)k0;
            o[5] = (int)std::min<long long>(seen, k0 + (long long)len * kTile);
            o[6] = ctx;
            o[7] = part0 < 0 ? -1 : part0 + (int)(sp * x.n) + rb;
        }
    }
}

}  // namespace

PlanShape plan_shape(int B, int groups, int rows, int H, int kv_rank, int max_q_len) {
    PlanShape p{};
    p.B = B;
    p.groups = groups;
    p.rows = rows;
    p.H = H;
    p.kv_rank = kv_rank;
    p.max_q_len = max_q_len;
    const long long flat = (long long)rows * H;
    const long long own_most = std::min(flat, (long long)max_q_len * H);  // rows of a session
    const long long own = std::min<long long>(kFewRows, own_most);
    p.qt = kv_rank <= 128 && own > 16 ? 2 : 1;
    p.target_k = kv_rank <= 128 ? 768 : 256;
    p.target_r = kv_rank <= 128 ? 512 : 256;
    p.least_k = 4;
    p.least_r = 8;
    // a segment's jobs: blocks * ceil(tiles / len) <= cost / len + blocks
    const long long segs = (long long)B + groups, sides = groups > 0 ? 2 : 1;
    const long long blocks_k =
        std::min(segs * (kFewRows / (16 * p.qt)), sides * (flat / (16 * p.qt)) + segs);
    const long long blocks_r = sides * (flat / kRowsR) + std::min(segs, sides * (flat / (kFewRows + 1)));
    // a list that no segment of these sizes can be on is not launched
    const bool few = H <= kFewRows, many = own_most > kFewRows || (groups > 0 && flat > kFewRows);
    p.max_jobs_k = few ? (int)(p.target_k + blocks_k) : 0;
    p.max_jobs_r = many ? (int)(p.target_r + blocks_r) : 0;
    // rows of a segment cut into s >= 2 ranges: n s <= 2 (rows of a block) blocks tiles / len;
    // and one range each of the sessions behind a prefix, own keys and the prefix
    const long long cut = 2LL * 16 * p.qt * p.target_k + (p.max_jobs_r ? 2LL * kRowsR * p.target_r : 0);
    p.max_parts = std::min(cut + (groups > 0 ? 2 * flat : 0),
                           16LL * p.qt * p.max_jobs_k + (long long)kRowsR * p.max_jobs_r);
    p.seg_at = kPlanHead;
    p.merge_at = p.seg_at + segs * kSegInts;
    p.session_at = p.merge_at + (long long)B * kMergeInts;
    p.jobs_k_at = (p.session_at + rows + 7) & ~7LL;
    p.jobs_r_at = p.jobs_k_at + (long long)p.max_jobs_k * kJobInts;
    p.words = p.jobs_r_at + (long long)p.max_jobs_r * kJobInts;
    uint32_t h = 2166136261u;
    for (const int v : {B, groups, rows, H, kv_rank, max_q_len})
        h = (h ^ (uint32_t)v) * 16777619u;
    p.tag = h | 1u;
    return p;
}

hipError_t launch_plan(const PlanArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mla
