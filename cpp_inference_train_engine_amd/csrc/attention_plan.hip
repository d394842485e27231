// The plan of mla_latent_attention: which workgroup takes which rows over which keys, built on
// the GPU once for a batch and used by every layer's call.  No reference counterpart.
//
// One workgroup, everything in LDS tables (in the plan's own for very large batches).  A segment
// (mla_latent.hpp) has row blocks and 32-key tiles; the keys of all segments of a list are cut into
// ranges of one length.  A GPU that holds `slots` workgroups of the list at once takes
//     ceil(jobs / slots) * (length * time of a tile + time of a job's start and end)
//     + the time of writing and reading the jobs' partial rows, where there are any
// where a tile takes its full time with all slots taken and half of it with half of them or fewer
// (a wave alone is bound by its latencies).  So what counts is that the jobs fill one round or two
// and not a little more, and that small batches are not cut finer than pays for the partial rows:
// the length is the best of candidates between half and four times a slot's share.  (200 sessions
// behind 5 prefixes, 8 heads, kv 128: 470 jobs took 17.3 us, 801, a share each, 18.4.)
// Whether segments of many rows go to list R or are taken apart for list K is decided by the same
// estimate: list K costs more per row, but its jobs are small and there is one launch instead of
// two.  (4 chunks of 509 rows, 8 heads, kv 128: list K 26.8 us, list R 36.)
// The kernel is a chain of short phases of one workgroup: 10 us for one session, 24 for 200 with
// prefixes.  Two things cost it most and were taken out: 64-bit divisions, and sums across lanes
// for each candidate where a lane can have a candidate of its own (16-31 us).  512 threads: twice
// as many only wait longer at the barriers.
#include "mla_latent.hpp"

#include <algorithm>

namespace mla {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kLdsSegs = 3000;  // segments whose tables fit LDS (9 of 12 KB)
constexpr int kTables = 9;
constexpr int kUnits = 256;     // compute units
constexpr int kFewRows = 64;    // segments up to this go to list K in any case
constexpr int kRounds = 2, kSteps = 8, kTries = (kRounds + 1) * kSteps;

// Times in ns of a unit of 32 keys, by list, with all slots taken, and of a job's start and end:
// those of kv 128 (for up to 128) and 512 with fixed rope columns, and with the softmax weights in
// one part, as the other times of jobs here.  (In two parts a unit takes 13-18 % longer.  With that in the table,
// eleven batches at kv 128 to 512 got the same jobs.)
struct Cost {
    int tile_k, job_k, tile_r, job_r, launch;
};
__device__ __forceinline__ Cost cost_of(int kv_rank) {
    return kv_rank <= 128 ? Cost{1500, 3500, 1100, 4000, 3000} : Cost{6000, 6000, 2200, 8000, 3000};
}

// Inclusive scans of three counts over the workgroup; `total` receives the sums.  (Jobs and partial
// rows of a plan's sizes stay below 2^31, see plan_shape.)
__device__ void block_scan3(int (&v)[3], int (*tmp)[3], int (&total)[3]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d <<= 1)
        for (int k = 0; k < 3; ++k) {
            const int u = __shfl_up(v[k], d, 64);
            if (lane >= d)
                v[k] += u;
        }
    __syncthreads();
    if (lane == 63)
        for (int k = 0; k < 3; ++k)
            tmp[wave][k] = v[k];
    __syncthreads();
    for (int k = 0; k < 3; ++k) {
        int before = 0;
        total[k] = 0;
        for (int w = 0; w < kWaves; ++w) {
            const int x = tmp[w][k];
            before += w < wave ? x : 0;
            total[k] += x;
        }
        v[k] += before;
    }
}

__device__ __forceinline__ long long wave_total(long long v) {
    for (int d = 32; d > 0; d >>= 1)
        v += __shfl_xor(v, d, 64);
    return v;
}

__device__ __forceinline__ int ceil_div(int a, int b) { return (int)(((unsigned)a + b - 1) / (unsigned)b); }

// ON_CHIP: the tables lie in LDS (known to the compiler: generic loads take three times as long)
template <bool ON_CHIP>
__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
    __shared__ int32_t lds[ON_CHIP ? kTables * kLdsSegs : 1];
    __shared__ int tmp[kWaves][3];
    __shared__ unsigned long long best[3], tile_sum[3];
    __shared__ int listed[2];  // the prefix pages that groups list: first, behind the last
    __shared__ int first_bad, tries[3][3 * kTries];  // jobs, their partial rows' blocks, the longest
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const PlanShape& p = a.p;
    const int B = p.B, G = p.groups, S = G + B, H = p.H;
    int32_t* const head = a.plan;
    // tables of the segments: the groups' prefixes, then the sessions' own keys
    int32_t* t;
    if constexpr (ON_CHIP)
        t = lds;
    else
        t = a.plan + p.seg_at;
    int32_t *const q0 = t, *const ql = t + S, *const keys = t + 2LL * S, *const group = t + 3LL * S,
            *const job_k = t + 4LL * S, *const job_r = t + 5LL * S, *const part = t + 6LL * S,
            *const cuts = t + 7LL * S, *const len = t + 8LL * S;

    // ---- checks and the segments' sizes ----
    const int total_q = a.info[0] < 0 ? -1 : a.cu_q[B];
    if (tid < 2)
        listed[tid] = tid == 0 ? a.n_prefix_pages : 0;
    if (tid == 0)
        first_bad = total_q < 0 || total_q > p.rows ? -1 : 0x7fffffff;
    if (tid < 3) {
        best[tid] = ~0ull;
        tile_sum[tid] = 0;
    }
    if (tid < 3 * kTries)
        tries[0][tid] = tries[1][tid] = tries[2][tid] = 0;
    __syncthreads();
    if (first_bad != -1) {
        for (int i = tid; i < S; i += kThreads) {
            bool ok;
            int s0 = 0, s1 = 0, n = 0;
            if (i < G) {
                s0 = a.cu_groups[i];
                s1 = a.cu_groups[i + 1];
                n = a.prefix_len[i];
                const int c0 = a.cu_prefix_pages[i], c1 = a.cu_prefix_pages[i + 1];
                ok = s0 >= 0 && s1 >= s0 && s1 <= B && n >= 0 && c0 >= 0 && c1 >= c0 &&
                     c1 <= a.n_prefix_pages && (long long)(c1 - c0) * a.page_size >= n;
                if (ok && c1 > c0) {
                    atomicMin(&listed[0], c0);
                    atomicMax(&listed[1], c1);
                }
            } else {
                s0 = i - G;
                s1 = s0 + 1;
                n = a.cu_k[s1] - a.cu_k[s0];
                ok = a.cu_q[s1] - a.cu_q[s0] <= p.max_q_len;
            }
            if (!ok)
                atomicMin(&first_bad, i);
            q0[i] = ok ? a.cu_q[s0] : 0;
            ql[i] = ok ? a.cu_q[s1] - a.cu_q[s0] : 0;
            keys[i] = n;
            group[i] = -1;
        }
        // Only ids that some group lists count.  (Behind the lists there may be anything, -1 in a
        // buffer of fixed length: a bad id costs a pass over the groups, 2.4 ms for 65,536 behind
        // 200 groups.)
        __syncthreads();
        for (long long i = listed[0] + (long long)tid; i < listed[1]; i += kThreads)
            if ((unsigned)a.prefix_page_ids[i] >= (unsigned)a.num_pool_pages)
                for (int g = 0; g < G; ++g)
                    if (a.cu_prefix_pages[g] <= i && i < a.cu_prefix_pages[g + 1]) {
                        atomicMin(&first_bad, g);
                        break;
                    }
    }
    __syncthreads();
    if (first_bad != 0x7fffffff) {
        if (tid < kPlanHead)
            head[tid] = tid == kPlanStatus ? -1 : tid == kPlanBad ? first_bad : 0;
        return;
    }
    for (int g = wave; g < G; g += kWaves)  // which prefix a session has
        if (keys[g] > 0)
            for (int s = a.cu_groups[g] + lane; s < a.cu_groups[g + 1]; s += 64)
                group[G + s] = g;
    __syncthreads();

    auto flat = [&](int i) { return ql[i] > 0 && keys[i] > 0 ? ql[i] * H : 0; };  // its rows
    auto tiles = [&](int i) { return ceil_div(std::max(keys[i], 0), kTile); };
    const Cost cost = cost_of(p.kv_rank);
    // Lists to estimate: 0 list K of the few, 1 list R of the others, 2 list K of all.
    auto blocks_of = [&](int list, int n) {  // blocks of n rows
        const int k = ceil_div(n, kRowsK), r = ceil_div(n, kRowsR);
        return list == 2 ? k : list == 0 ? (n <= kFewRows ? k : 0) : (n > kFewRows ? r : 0);
    };

    // ---- the range lengths ----
    long long sums[3];
    {
        long long v[3] = {0, 0, 0};
        for (int i = tid; i < S; i += kThreads) {
            const int n = flat(i), t = tiles(i);
            for (int list = 0; list < 3; ++list)
                v[list] += (long long)blocks_of(list, n) * t;
            cuts[i] = n;  // for the estimates: rows, tiles, and whether there is more to join
            len[i] = i < G || group[i] >= 0 ? -1 - t : t;
        }
        for (int list = 0; list < 3; ++list) {
            v[list] = wave_total(v[list]);
            if (lane == 0 && v[list] != 0)
                atomicAdd(&tile_sum[list], (unsigned long long)v[list]);
        }
        __syncthreads();
        for (int list = 0; list < 3; ++list)
            sums[list] = (long long)tile_sum[list];
    }
    const int log_k = __builtin_ctz(p.slots_k), log_r = __builtin_ctz(p.slots_r);  // powers of two
    auto tried = [&](int list, int c) {  // length of candidate c, in tiles
        const int k = c / kSteps;  // 0: twice a slot's share or more, 1: its share, 2: half of it
        const long long share = (sums[list] * kRounds >> (k + (list == 1 ? log_r : log_k))) + 1;
        long long n = share + share * (c % kSteps) / kSteps;
        n = list == 1 ? (n + 1) & ~1LL : (n + 3) & ~3LL;  // a tile for each of the four waves
        return (int)std::min<long long>(n, 1 << 26);
    };
    // A lane estimates a candidate, over every kWaves-th segment in each wave.
    auto wanted = [&](int list) {  // (without segments of many rows lists 0 and 2 are the same)
        return sums[list] > 0 && !(list == 0 && sums[1] == 0) &&
               !(list == 2 && sums[1] > 0 && !p.list_k_holds_all);
    };
    for (int e = lane; e < 3 * kTries; e += 64) {
        const int list = e / kTries;
        if (!wanted(list))
            continue;
        const int n = tried(list, e % kTries);
        const float inv = 1.0f / (float)n;  // an estimate may be a range off where it just fits
        int jobs = 0, parts = 0, longest = 0;
#pragma unroll 4
        for (int i = wave; i < S; i += kWaves) {
            const int b = blocks_of(list, cuts[i]);
            const bool joined = len[i] < 0;
            const int t = joined ? -1 - len[i] : len[i];
            const int splits = (int)__builtin_ceilf((float)t * inv);
            jobs += b * splits;
            parts += splits > 1 || joined ? b * splits : 0;
            longest = b > 0 ? std::max(longest, std::min(n, t)) : longest;
        }
        atomicAdd(&tries[0][e], jobs);
        atomicAdd(&tries[1][e], parts);
        atomicMax(&tries[2][e], longest);
    }
    __syncthreads();
    if (const int list = tid / kTries; list < 3 && wanted(list)) {
        const int jobs = tries[0][tid], parts = tries[1][tid], longest = tries[2][tid];
        const int slots = list == 1 ? p.slots_r : p.slots_k, most = slots / kUnits;
        const float rounds = (float)ceil_div(jobs, slots);
        // workgroups that share a compute unit share its time, down to half of them
        const float share =
            std::max((float)std::min(most, ceil_div(jobs, kUnits)) / (float)most, 0.5f);
        const float each = list == 1
                               ? (float)longest * share * cost.tile_r + cost.job_r
                               : (float)((longest + 3) / 4) * share * cost.tile_k + cost.job_k;
        // fp32 rows written and read back, at about 4 TB/s
        const float rows =
            (float)parts * ((list == 1 ? kRowsR : kRowsK) * p.kv_rank) * (8.0f / 4000);
        const unsigned long long ns = (unsigned long long)std::min(rounds * each + rows, 4e9f);
        atomicMin(&best[list], ns << 32 | (unsigned)(tid - list * kTries));
    }
    __syncthreads();
    auto ns_of = [&](int list) { return sums[list] == 0 ? 0 : (long long)(best[list] >> 32); };
    const bool all_k = p.max_jobs_r == 0 || sums[1] == 0 ||
                       (p.list_k_holds_all &&
                        ns_of(2) < ns_of(0) + ns_of(1) + (sums[0] > 0 ? cost.launch : 0));
    auto few = [&](int i) { return all_k || flat(i) <= kFewRows; };
    const int list_k = all_k ? 2 : 0;
    const int len_k = sums[list_k] == 0 ? 4 : tried(list_k, (int)(best[list_k] & 0xffffffffu));
    const int len_r = all_k ? 1 : tried(1, (int)(best[1] & 0xffffffffu));

    // ---- jobs and partial rows of each segment ----
    int at[3] = {0, 0, 0};
    for (int i0 = 0; i0 < S; i0 += kThreads) {
        const int i = i0 + tid;
        int n = 0, splits = 0, range = 0, blocks = 0;
        bool f = false;
        if (i < S && (n = flat(i)) > 0) {
            f = few(i);
            blocks = ceil_div(n, f ? kRowsK : kRowsR);
            splits = ceil_div(tiles(i), f ? len_k : len_r);
            range = ceil_div(tiles(i), splits);  // the segment's ranges as even as they go
            range = f ? (range + 3) & ~3 : (range + 1) & ~1;  // (list R stages two units at once)
            splits = ceil_div(tiles(i), range);
        }
        const bool joined = n > 0 && (splits > 1 || i < G || group[i] >= 0);
        const int jobs = blocks * splits;
        const int mine[3] = {f ? jobs : 0, f ? 0 : jobs, joined ? n * splits : 0};
        int v[3] = {mine[0], mine[1], mine[2]}, sum[3];
        block_scan3(v, tmp, sum);
        if (i < S) {
            job_k[i] = at[0] + v[0] - mine[0];
            job_r[i] = at[1] + v[1] - mine[1];
            part[i] = joined ? at[2] + v[2] - mine[2] : -1;
            cuts[i] = splits;
            len[i] = range;
        }
        for (int k = 0; k < 3; ++k)
            at[k] += sum[k];
    }
    __syncthreads();
    const bool fits = at[0] <= p.max_jobs_k && at[1] <= p.max_jobs_r && at[2] <= p.max_parts;
    if (tid < kPlanHead) {
        int v = 0;
        if (fits)
            v = tid == kPlanStatus ? at[0] + at[1]
                : tid == kPlanJobsK ? at[0]
                : tid == kPlanJobsR ? at[1]
                : tid == kPlanParts ? at[2]
                : tid == kPlanRows  ? total_q
                : tid == kPlanTag   ? (int)p.tag
                                    : 0;
        else
            v = tid == kPlanStatus ? -1 : tid == kPlanBad ? -2 : 0;
        head[tid] = v;
    }
    if (!fits)
        return;

    // ---- the jobs ----
    for (int list = 0; list < 2; ++list) {
        const int32_t* first = list ? job_r : job_k;
        int32_t* out = a.plan + (list ? p.jobs_r_at : p.jobs_k_at);
        for (int j = tid; j < at[list]; j += kThreads) {
            int lo = 0, hi = S;  // the last segment that starts at or before the job
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (first[mid] <= j)
                    lo = mid;
                else
                    hi = mid;
            }
            const int i = lo, n = flat(i), rows = list ? kRowsR : kRowsK;
            const int blocks = ceil_div(n, rows), in = j - first[i];
            const int sp = in / blocks, rb = (in - sp * blocks) * rows;
            const int m = std::min(rows, n - rb), ctx = i < G ? keys[i] : keys[i] - ql[i];
            const long long k0 = (long long)sp * len[i] * kTile;
            // own keys: the block's last row sees keys up to its own token
            const int seen = i < G ? keys[i] : ctx + (rb + m - 1) / H + 1;
            int32_t* o = out + (long long)j * kJobInts;
            o[0] = i < G ? ~i : i - G;
            o[1] = q0[i] * H + rb;
            o[2] = m;
            o[3] = rb;
            o[4] = (int)k0;
            o[5] = (int)std::min<long long>(seen, k0 + (long long)len[i] * kTile);
            o[6] = ctx;
            o[7] = part[i] < 0 ? -1 : part[i] + sp * n + rb;
        }
    }
    // ---- what the merge adds up for each row ----
    if (at[2] == 0)
        return;
    for (int e = tid; e < 16 * B; e += kThreads) {  // 16 threads a session
        const int i = G + (e >> 4), g = group[i], rows = ql[i];
        const int pre = g >= 0 && flat(g) > 0 ? cuts[g] : 0, mine = part[i] >= 0 ? cuts[i] : 0;
        const int pre_n = pre > 0 ? flat(g) : 0;
        const int pre_at = pre > 0 ? part[g] + (q0[i] - q0[g]) * H : 0;
        for (int r = e & 15; r < rows; r += 16) {
            i32x4* m = reinterpret_cast<i32x4*>(a.plan + p.merge_at +
                                                (long long)(q0[i] + r) * kMergeInts);
            m[0] = i32x4{pre, mine, pre_at + r * H, part[i] + r * H};
            m[1] = i32x4{pre_n, flat(i), 0, 0};
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
    const long long own = std::min(flat, (long long)max_q_len * H);  // most rows of a session
    // Workgroups that 256 compute units hold: by registers and LDS of the two lists' kernels with
    // fixed rope columns.  (The others hold half as many at kv 128.)
    p.slots_k = kv_rank <= 128 ? 1024 : kv_rank <= 256 ? 512 : 256;
    p.slots_r = kv_rank <= 128 ? 512 : 256;
    const bool few = H <= kFewRows, many = own > kFewRows || (groups > 0 && flat > kFewRows);
    const long long segs = (long long)B + groups, sides = groups > 0 ? 2 : 1;
    // A list's ranges are at least sums / (kRounds slots) long (see tried), so a segment's jobs,
    // blocks * ceil(tiles / length) <= blocks * tiles / length + blocks, add up to at most
    // kRounds * slots + the blocks.
    const long long blocks_k = sides * (flat / kRowsK) + segs;
    const long long few_k = std::min(blocks_k, segs * (kFewRows / kRowsK));
    const long long blocks_r =
        sides * (flat / kRowsR) + std::min(segs, sides * (flat / (kFewRows + 1)));
    // List K takes segments of many rows only while its table stays small: where it would pay.
    p.list_k_holds_all = many && blocks_k <= 4LL * p.slots_k;
    const long long most_k = p.list_k_holds_all ? blocks_k : few_k;
    p.max_jobs_k = few || p.list_k_holds_all ? (int)(kRounds * p.slots_k + most_k) : 0;
    p.max_jobs_r = many ? (int)(kRounds * p.slots_r + blocks_r) : 0;
    // A segment of n rows cut into s >= 2 ranges has n s <= 2 (rows of a block) blocks tiles /
    // length partial rows, 2 (rows of a block) kRounds slots in all; the sessions behind a prefix
    // and the prefixes have n each even where they are not cut.
    const long long cut = 2LL * kRounds * (kRowsK * (p.max_jobs_k ? p.slots_k : 0) +
                                           kRowsR * (p.max_jobs_r ? p.slots_r : 0));
    p.max_parts = std::min(cut + (groups > 0 ? 2 * flat : 0),
                           (long long)kRowsK * p.max_jobs_k + (long long)kRowsR * p.max_jobs_r);
    p.seg_at = kPlanHead;
    p.merge_at = p.seg_at + (segs > kLdsSegs ? (segs * kTables + 7) & ~7LL : 0);
    p.jobs_k_at = p.merge_at + (long long)rows * kMergeInts;
    p.jobs_r_at = p.jobs_k_at + (long long)p.max_jobs_k * kJobInts;
    p.words = p.jobs_r_at + (long long)p.max_jobs_r * kJobInts;
    return p;
}

uint32_t plan_tag(const PlanShape& p, int page_size, bool prefix_pages) {
    uint32_t h = 2166136261u;
    for (const int v : {p.B, p.groups, p.rows, p.H, p.kv_rank, p.max_q_len, page_size, (int)prefix_pages})
        h = (h ^ (uint32_t)v) * 16777619u;
    return h | 1u;
}

hipError_t launch_plan(const PlanArgs& a, hipStream_t stream) {
    if (a.p.B + a.p.groups <= kLdsSegs)
        hipLaunchKernelGGL(plan_kernel<true>, dim3(1), dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL(plan_kernel<false>, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mla
