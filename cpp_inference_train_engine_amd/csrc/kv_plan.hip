// The plan of mla_kv_attention: which workgroup takes which query rows over which keys, built on
// the GPU once for a batch, a window and its sinks, and used by every such layer's call.  No
// reference counterpart.
//
// One workgroup, its tables in LDS (in the plan for large batches).  A session's flat rows
// (mla_kv.hpp) are cut into blocks, and the units of 32 keys that a block sees into ranges: of a
// length that gives every slot of the GPU one range (several where they are long, so that slots
// with short ones take more of them), or of twice a slot's share (so that only blocks well above it
// are cut) where there are more blocks than that.
// A chain of short phases of one workgroup: 6-10 us back to back, up to 14 alone.  (64 sessions of
// 128 .. 14,000 tokens, 32 heads on kv 8 x 128, attend in 302 us with up to four ranges a slot, in
// 313 with one.  Blocks of many rows keep their order, in which neighbours read the same keys at
// the same time: 4,000 rows take 204 us, and 212 with the longest blocks first.)
#include "mla_kv.hpp"

#include <algorithm>
#include <climits>

namespace mla {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kLdsBlocks = 2800, kLdsSessions = 1400;
constexpr int kTables = 4, kTries = 24, kEven = 2;
constexpr int kMinF = 4, kMinM = 8;  // least units of a range
// Blocks of the first list are left whole where the longest, taken by its four waves alone, takes no
// longer than the second launch, which joins what was cut, and a quarter of the time that memory
// needs for all of them: in ns.  (50 sessions of 900 to 1,100 tokens, 32 heads, kv 8 x 128: 42 us whole,
// 52 cut in two; 100 of 10 to 5,000: 200 and 183.)
constexpr int kJoin = 7000, kBytesPerNs = 6500;
__device__ __forceinline__ int unit_ns(int dim, int v_dim) { return 80 + 15 * (dim + v_dim) / 16; }
// Of the second list, blocks of up to so many units (2 x 300 rows: 17 us whole, 21 in ranges of 8).
constexpr int kWholeM = 16;
constexpr int kRounds = 4, kRoundUnits = 24;  // most ranges of a slot, and their least units

__device__ __forceinline__ int ceil_div(int a, int b) { return (int)(((unsigned)a + b - 1) / (unsigned)b); }

// Inclusive scans of two counts over the workgroup; `total` receives the sums.
__device__ void block_scan2(int (&v)[2], int (*tmp)[2], int (&total)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d <<= 1)
        for (int k = 0; k < 2; ++k) {
            const int u = __shfl_up(v[k], d, 64);
            if (lane >= d)
                v[k] += u;
        }
    __syncthreads();
    if (lane == 63)
        for (int k = 0; k < 2; ++k)
            tmp[wave][k] = v[k];
    __syncthreads();
    for (int k = 0; k < 2; ++k) {
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

// The last of n starts that lies at or before i.
__device__ __forceinline__ int find(const int32_t* starts, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= i)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

template <bool ON_CHIP>
__global__ __launch_bounds__(kThreads) void kv_plan_kernel(KvPlanArgs a) {
    __shared__ int32_t lds[ON_CHIP ? kTables * kLdsBlocks + 2 * kLdsSessions : 1];
    __shared__ int tmp[kWaves][2], tries[kEven + kTries], longest, first_bad;
    __shared__ unsigned long long sum;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const KvShape& p = a.p;
    const int B = p.B, G = p.group, NB = p.max_blocks;
    int32_t* const head = a.plan;
    int32_t* t;
    if constexpr (ON_CHIP)
        t = lds;
    else
        t = a.plan + p.tables_at;
    int32_t *const session = t, *const units = t + NB, *const job = t + 2LL * NB,
            *const part = t + 3LL * NB, *const start = t + (long long)kTables * NB;

    // ---- checks ----
    const int total_q = a.info[0] < 0 ? -1 : a.cu_q[B];
    if (tid == 0)
        first_bad = total_q < 0 || total_q > p.rows ? -1 : INT_MAX;
    __syncthreads();
    if (first_bad != -1)
        for (int s = tid; s < B; s += kThreads)
            if (a.cu_q[s + 1] - a.cu_q[s] > p.max_q_len)
                atomicMin(&first_bad, s);
    __syncthreads();
    if (first_bad != INT_MAX) {
        if (tid < kKvHead)
            head[tid] = tid == kKvStatus ? -1 : tid == kKvBad ? first_bad : 0;
        return;
    }

    int jobs[2] = {0, 0}, parts = 0;
    bool cut[2] = {false, false};  // whether the list has partial rows
    auto flat = [&](int s) { return (a.cu_q[s + 1] - a.cu_q[s]) * G; };
    for (int list = 0; list < 2; ++list) {
        const int per = list ? kKvManyRows : p.few_rows;
        const int slots = list ? p.slots_m : p.slots_f;
        const int most_jobs = list ? p.max_jobs_m : p.max_jobs_f;
        if (most_jobs == 0)
            continue;
        // ---- the sessions' blocks ----
        int blocks = 0;
        for (int s0 = 0; s0 < B; s0 += kThreads) {
            const int s = s0 + tid;
            const int n = s < B ? flat(s) : 0;
            const int mine = (n <= p.few) == (list == 0) ? ceil_div(n, per) : 0;
            int v[2] = {mine, 0}, total[2];
            block_scan2(v, tmp, total);
            if (s < B)
                start[s] = blocks + v[0] - mine;
            blocks += total[0];
        }
        if (tid < kEven + kTries)
            tries[tid] = 0;
        if (tid == 0) {
            sum = 0;
            longest = 0;
        }
        __syncthreads();
        // ---- the units that each sees ----
        unsigned long long mine = 0;
        int most = 0;
        for (int b = tid; b < blocks; b += kThreads) {
            const int s = find(start, B, b), f0 = (b - start[s]) * per, n = flat(s);
            const int keys = a.cu_k[s + 1] - a.cu_k[s], ctx = keys - n / G;
            const int last = std::min(f0 + per, n) - 1;
            session[b] = s;
            units[b] = kv_units(ctx + f0 / G, ctx + last / G, p.window, p.sinks).count;
            mine += units[b];
            most = std::max(most, units[b]);
        }
        for (int d = 32; d > 0; d >>= 1) {
            mine += __shfl_xor(mine, d, 64);
            most = std::max(most, __shfl_xor(most, d, 64));
        }
        if (lane == 0 && mine != 0) {
            atomicAdd(&sum, mine);
            atomicMax(&longest, most);
        }
        __syncthreads();
        // ---- the length of a range ----
        const unsigned long long whole = (sum + slots - 1) / slots;
        const int rounds =
            list ? 1 : (int)std::max<unsigned long long>(std::min<unsigned long long>(whole / kRoundUnits, kRounds), 1);
        const int goal = slots * rounds;
        const int least = list ? kMinM : kMinF;
        // Candidates: up to an eighth above a slot's share, then from a share of the goal on.
        auto length = [&](int c) {
            const int wanted = c < kEven ? slots : goal;
            const long long share = std::min<long long>((sum + wanted - 1) / wanted, 1 << 26);
            return (int)(std::max(share + share * (c < kEven ? c : c - kEven) / 8, (long long)least) + 3) & ~3;
        };
        int len = length(kEven + 8);
        const unsigned long long memory =
            sum * p.kv_heads * (kKvTile * 2 * (p.dim + p.v_dim)) / kBytesPerNs;
        if (list == 0 ? (unsigned long long)longest * unit_ns(p.dim, p.v_dim) <= kJoin + memory / 4
                      : longest <= kWholeM) {
            len = (longest + 3) & ~3;
        } else if (blocks <= goal) {
            if (lane < kEven + kTries) {
                const float inv = 1.0f / (float)length(lane);
                int n = 0;
                for (int b = wave; b < blocks; b += kWaves)
                    n += (int)__builtin_ceilf((float)units[b] * inv);
                atomicAdd(&tries[lane], n);
            }
            __syncthreads();
            // One even range for every slot, if there is such a length; else the shortest of those
            // that make no more ranges than wanted.
            int c = 0;
            while (c < kEven && tries[c] > slots)
                ++c;
            if (c == kEven)
                while (c < kEven + kTries - 1 && tries[c] > goal)
                    ++c;
            len = length(c);
            if (len > longest - longest / 4)  // (would shorten little)
                len = (longest + 3) & ~3;
        }
        // ---- jobs and partial rows of each block ----
        int at = 0;
        const int before = parts;
        for (int b0 = 0; b0 < blocks; b0 += kThreads) {
            const int b = b0 + tid;
            int n = 0, splits = 0, range = 0;
            if (b < blocks) {
                const int s = session[b];
                n = std::min(per, flat(s) - (b - start[s]) * per);
                splits = ceil_div(units[b], len);
                range = (ceil_div(units[b], splits) + 3) & ~3;  // a block's ranges as even as they go
                splits = ceil_div(units[b], range);
            }
            const int rows = splits > 1 ? n * splits : 0;
            int v[2] = {splits, rows}, total[2];
            block_scan2(v, tmp, total);
            if (b < blocks) {
                job[b] = at + v[0] - splits;
                part[b] = rows > 0 ? parts + v[1] - rows : -1;
                units[b] = range;  // (what a block sees is computed anew where it is needed)
            }
            at += total[0];
            parts += total[1];
        }
        __syncthreads();
        jobs[list] = at;
        cut[list] = parts > before;
        if (at > most_jobs || parts > p.max_parts)
            break;  // (the bounds hold for every batch of these sizes: never)
        // ---- the jobs, the last rows' first: a prompt's later blocks see more ----
        int32_t* out = a.plan + (list ? p.jobs_m_at : p.jobs_f_at);
        for (int j = tid; j < at; j += kThreads) {
            const int b = find(job, blocks, j), s = session[b], range = units[b];
            const int f0 = (b - start[s]) * per, n = flat(s), m = std::min(per, n - f0);
            const int ctx = a.cu_k[s + 1] - a.cu_k[s] - n / G, sp = j - job[b];
            const int seen = kv_units(ctx + f0 / G, ctx + (f0 + m - 1) / G, p.window, p.sinks).count;
            int32_t* o = out + (long long)(at - 1 - j) * kKvJobInts;
            o[0] = s;
            o[1] = a.cu_q[s];
            o[2] = f0;
            o[3] = m;
            o[4] = sp * range;
            o[5] = std::min(seen, (sp + 1) * range);
            o[6] = ctx;
            o[7] = part[b] < 0 ? -1 : part[b] + sp * m;
        }
        // ---- what the merge adds up for each row ----
        for (int e = tid >> 4; cut[list] && e < blocks; e += kThreads / 16) {
            const int s = session[e], f0 = (e - start[s]) * per, n = flat(s), m = std::min(per, n - f0);
            const int splits = part[e] < 0 ? 0 : (e + 1 < blocks ? job[e + 1] : at) - job[e];
            for (int r = tid & 15; r < m; r += 16) {
                int32_t* o = a.plan + p.rows_at +
                             ((long long)a.cu_q[s] * G + f0 + r) * kKvRowInts;
                o[0] = part[e] + r;
                o[1] = splits;
                o[2] = m;
            }
        }
        __syncthreads();
    }
    if (parts > 0 && cut[0] != cut[1])  // the rows of the list that has no partial ones
        for (int s = tid >> 4; s < B; s += kThreads / 16) {
            const int n = flat(s);
            if ((n <= p.few) == cut[1])
                for (int r = tid & 15; r < n; r += 16)
                    a.plan[p.rows_at + ((long long)a.cu_q[s] * G + r) * kKvRowInts + 1] = 0;
        }
    const bool fits = jobs[0] <= p.max_jobs_f && jobs[1] <= p.max_jobs_m && parts <= p.max_parts;
    if (tid < kKvHead) {
        int v = 0;
        if (fits) {
            v = tid == kKvStatus ? jobs[0] + jobs[1]
                : tid == kKvJobsF ? jobs[0]
                : tid == kKvJobsM ? jobs[1]
                : tid == kKvParts ? parts
                : tid == kKvRows  ? total_q
                : tid == kKvTag   ? (int)p.tag
                                  : 0;
#pragma unroll
            for (int i = 0; i < kKvSizeInts; ++i)
                v = tid == kKvSizes + i ? p.sizes[i] : v;
        } else
            v = tid == kKvStatus ? -1 : tid == kKvBad ? -2 : 0;
        head[tid] = v;
    }
}

}  // namespace

KvShape kv_shape(int B, int rows, int H, int kv_heads, int dim, int v_dim, int page_size,
                 int max_q_len, int window, int sinks) {
    KvShape p{};
    p.B = B;
    p.rows = rows;
    p.H = H;
    p.kv_heads = kv_heads;
    p.group = H / kv_heads;
    p.dim = dim;
    p.v_dim = v_dim;
    p.width = kv_width(dim, v_dim);
    p.page_size = page_size;
    p.max_q_len = max_q_len;
    p.window = window;
    p.sinks = sinks;
    const long long flat = (long long)rows * p.group;  // of one kv head
    const long long own = std::min(flat, (long long)max_q_len * p.group);
    // Where no session has more than 16 flat rows, blocks of 16; else of 32 (above width 192, whose
    // registers hold no more, 16 again), which read the keys half as often.
    p.few_rows = own <= 16 || p.width == 256 ? 16 : 32;
    p.few = own <= 16 ? 16 : p.width == 256 ? 32 : 64;
    // Workgroups of a list at once, which the ranges' lengths follow from.  256 compute units hold
    // as many, but for blocks of 16 at width 64 (1,024), of smaller heads in fp16 at width 128 (512)
    // and of width 256 (256): there an even range for each is one and a half or two rounds of them.
    const int at_once_f = p.width == 64    ? (p.few_rows == 16 ? 1536 : 768)
                          : p.width == 128 ? (p.few_rows == 16 ? 768 : 512)
                                           : 512;
    const int at_once_m = p.width == 256 ? 256 : 512;
    p.slots_f = std::max(1, at_once_f / kv_heads);
    p.slots_m = std::max(1, at_once_m / kv_heads);
    const int many = kKvManyRows;
    const long long blocks_f =
        p.group <= p.few ? std::min<long long>((long long)B * (p.few / p.few_rows), flat / p.few_rows + B) : 0;
    const long long blocks_m =
        own > p.few ? flat / many + std::min<long long>(B, flat / (p.few + 1)) : 0;
    // A range is at least a share of the goal long, so that a list's blocks have at most
    // units / share + blocks <= goal + blocks ranges; those that are cut have fewer than twice
    // units / share, of a block's rows each.
    const long long goal_f = (long long)kRounds * p.slots_f;
    p.max_jobs_f = (int)std::min<long long>(blocks_f ? blocks_f + goal_f : 0, INT_MAX);
    p.max_jobs_m = (int)std::min<long long>(blocks_m ? blocks_m + p.slots_m : 0, INT_MAX);
    p.max_blocks = (int)std::min<long long>(std::max(blocks_f, blocks_m), INT_MAX);
    p.max_parts = (p.max_jobs_f ? 2 * goal_f * std::min<long long>(p.few_rows, own) : 0) +
                  (p.max_jobs_m ? 2LL * p.slots_m * std::min<long long>(many, own) : 0);
    p.tables_at = kKvHead;
    const bool on_chip = p.max_blocks <= kLdsBlocks && B <= kLdsSessions;
    p.rows_at = p.tables_at +
                (on_chip ? 0 : (((long long)p.max_blocks * kTables + B + 7) & ~7LL));
    p.jobs_f_at = p.rows_at + flat * kKvRowInts;
    p.jobs_m_at = p.jobs_f_at + (long long)p.max_jobs_f * kKvJobInts;
    p.words = p.jobs_m_at + (long long)p.max_jobs_m * kKvJobInts;
    // (every bit of a size reaches every bit of the tag; kv_plan_fits compares the sizes themselves)
    const int sizes[kKvSizeInts] = {B, rows, H, kv_heads, dim, v_dim, page_size, max_q_len, window, sinks};
    uint32_t h = 2166136261u;
    for (int i = 0; i < kKvSizeInts; ++i) {
        p.sizes[i] = sizes[i];
        h = (h ^ (uint32_t)sizes[i]) * 0x9e3779b1u;
        h = (h ^ (h >> 15)) * 0x85ebca77u;
        h ^= h >> 13;
    }
    p.tag = h ? h : 1;
    return p;
}

hipError_t launch_kv_plan(const KvPlanArgs& a, hipStream_t stream) {
    if (a.p.rows_at == a.p.tables_at)
        hipLaunchKernelGGL(kv_plan_kernel<true>, dim3(1), dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL(kv_plan_kernel<false>, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mla
