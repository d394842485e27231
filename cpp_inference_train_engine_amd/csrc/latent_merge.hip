// Joins the partials of mla_latent_attention: a row's weighted sums over ranges of its shared
// prefix and of its own keys, each with its reference maximum and mass, become the final row.
//     M = max_i m_i,  L = sum_i l_i 2^(m_i - M),  row = sum_i o_i 2^(m_i - M) / L
// One thread per 4 columns of a row and each of GROUPS groups; the groups split the row's partials,
// each reads kFlight of them at once (a round trip to memory is what a row costs, a partial's bytes
// are few), and their states meet in LDS.
// Bound by the launch and two trips to memory (the plan's head with the row's ranges, the partials)
// where rows are few: 3.4-5.0 us for up to 6,400 partial rows of 128 columns; by its bytes where they
// are many: 32,512 partial rows of 512 columns into 8,192 rows 14.2 us, 5.3 TB/s.  (That is more
// than a copy from HBM reaches: the 67 MB were written just before and partly lie in the last
// cache.)
#include "mla_latent.hpp"
#include "mla_common.hpp"

#include <algorithm>
#include <cmath>

namespace mla {
namespace {

constexpr int kThreads = 256, kFlight = 4;
constexpr long long kFewElements = 1 << 20;
constexpr long long kBlocksX = 1 << 20;  // a grid's x: it has fewer than 2^32 threads there

template <typename T, int GROUPS>
__global__ __launch_bounds__(kThreads) void latent_merge_kernel(LatentArgs a) {
    constexpr int PER = kThreads / GROUPS;  // threads of a group
    __shared__ float so[GROUPS > 1 ? kThreads * 4 : 4], sml[GROUPS > 1 ? kThreads * 2 : 4];
    const int32_t* plan = a.plan;
    const int tid = threadIdx.x, group = tid / PER, me = tid % PER;
    const int per_row = a.kv_rank / 4, H = a.H;
    const long long block = blockIdx.y * (long long)gridDim.x + blockIdx.x, e = block * PER + me;
    const long long fr = e / per_row;
    const int c = (int)(e - fr * per_row) * 4;
    const int row = (int)(fr / H);  // (past the rows in the last blocks)
    // A row's entry is read with the plan's head, not behind it, and dropped if that does not fit.
    const i32x4* entry = reinterpret_cast<const i32x4*>(
        plan + a.p.merge_at + (long long)min(row, a.p.rows - 1) * kMergeInts);
    const i32x4 m0 = entry[0], m1 = entry[1];
    const int all = plan[kPlanParts], rows = plan[kPlanRows];
    const bool some = plan_fits(a, plan[kPlanTag], plan[kPlanJobsK], plan[kPlanJobsR], all) &&
                      all > 0 && row < rows;
    const int pre = some ? m0[0] : 0, mine = some ? m0[1] : 0, head = (int)(fr - (long long)row * H);
    const long long pre_at = m0[2] + head, own_at = m0[3] + head, pre_n = m1[0], own_n = m1[1];
    const int parts = pre + mine;  // 0: no such row, or one job wrote it itself
    float M = -INFINITY, L = 0.0f;
    floatx4 o = {0, 0, 0, 0};
    for (int i0 = group; i0 < parts; i0 += GROUPS * kFlight) {
        float m[kFlight], l[kFlight];
        floatx4 x[kFlight];
        float top = M;
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const int i = min(i0 + k * GROUPS, parts - 1);
            const long long p = i < pre ? pre_at + i * pre_n : own_at + (i - pre) * own_n;
            typedef float f2 __attribute__((ext_vector_type(2)));
            const f2 ml = *reinterpret_cast<const f2*>(a.part_ml + 2 * p);
            m[k] = ml[0];
            l[k] = ml[1];
            x[k] = *reinterpret_cast<const floatx4*>(a.part_o + p * a.kv_rank + c);
        }
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            if (i0 + k * GROUPS >= parts) {  // read twice: counts once
                m[k] = -INFINITY;
                l[k] = 0.0f;
                x[k] = floatx4{0, 0, 0, 0};
            }
            top = fmaxf(top, m[k]);
        }
        // A mass of NaN may come with a maximum of -inf (every score was NaN): weight 0 keeps it.
        const float f0 = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - top);
        L *= f0;
        o *= f0;
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const float f = m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - top);
            L += l[k] * f;
            o += x[k] * f;
        }
        M = top;
    }
    if constexpr (GROUPS > 1) {
        *reinterpret_cast<floatx4*>(so + 4 * tid) = o;
        sml[2 * tid] = M;
        sml[2 * tid + 1] = L;
        __syncthreads();
        if (group > 0)
            return;
#pragma unroll
        for (int v = 1; v < GROUPS; ++v)
            M = fmaxf(M, sml[2 * (tid + v * PER)]);
        const float f0 = sml[2 * tid] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sml[2 * tid] - M);
        L *= f0;
        o *= f0;
#pragma unroll
        for (int v = 1; v < GROUPS; ++v) {
            const int at = tid + v * PER;
            const float m = sml[2 * at];
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
            L += sml[2 * at + 1] * f;
            o += *reinterpret_cast<const floatx4*>(so + 4 * at) * f;
        }
    }
    if (parts == 0)
        return;
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    typedef typename T::scalar s4 __attribute__((ext_vector_type(4)));
    s4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = static_cast<typename T::scalar>(o[i] * inv);
    *reinterpret_cast<s4*>(a.out + fr * a.kv_rank + c) = y;
    if (a.lse && c == 0)
        a.lse[fr] = (M + __log2f(L)) * kLn2;
}

template <typename T, int GROUPS>
void launch_groups(const LatentArgs& a, hipStream_t stream) {
    constexpr int per = kThreads / GROUPS;
    const long long blocks = ((long long)a.p.rows * a.H * (a.kv_rank / 4) + per - 1) / per;
    const unsigned x = (unsigned)std::min(blocks, kBlocksX);
    hipLaunchKernelGGL((latent_merge_kernel<T, GROUPS>), dim3(x, (unsigned)((blocks + x - 1) / x)),
                       dim3(kThreads), 0, stream, a);
}

template <typename T>
hipError_t launch_merge_t(const LatentArgs& a, hipStream_t stream) {
    // few rows: eight groups, so that one round of reads covers 32 partials; many: as many threads
    // as columns already fill the GPU
    if ((long long)a.p.rows * a.H * a.kv_rank <= kFewElements)
        launch_groups<T, 8>(a, stream);
    else
        launch_groups<T, 1>(a, stream);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_latent_attention(const LatentArgs& a, int dtype, hipStream_t stream) {
    // List R first: its jobs are the longer ones.
    for (const bool rows : {true, false}) {
        if ((rows ? a.jobs_r : a.jobs_k) == 0)
            continue;
        const hipError_t e = a.q8 ? launch_attend_q8(a, dtype, rows, stream)
                                  : launch_attend_16(a, dtype, rows, stream);
        if (e != hipSuccess)
            return e;
    }
    return a.parts != 0 ? launch_latent_merge(a, dtype, stream) : hipSuccess;
}

hipError_t launch_latent_merge(const LatentArgs& a, int dtype, hipStream_t stream) {
    return dtype == 0 ? launch_merge_t<F16>(a, stream) : launch_merge_t<BF16>(a, stream);
}

}  // namespace mla
