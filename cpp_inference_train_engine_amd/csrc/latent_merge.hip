// Joins the partials of mla_latent_attention: a row's weighted sums over ranges of its shared
// prefix and of its own keys, each with its reference maximum and mass, become the final row.
//     M = max_i m_i,  L = sum_i l_i 2^(m_i - M),  row = sum_i o_i 2^(m_i - M) / L
// One thread per 4 columns of a row.  Bound by the partials' bytes, or by latency for few rows.
#include "mla_latent.hpp"
#include "mla_common.hpp"

#include <cmath>

namespace mla {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ __launch_bounds__(kThreads) void latent_merge_kernel(LatentArgs a) {
    const int32_t* plan = a.plan;
    if (plan[kPlanTag] != (int)a.p.tag || plan[kPlanParts] == 0)
        return;
    const int per_row = a.kv_rank / 4, H = a.H;
    const long long e = blockIdx.x * (long long)kThreads + threadIdx.x;
    const long long fr = e / per_row;
    const int c = (int)(e - fr * per_row) * 4;
    const int row = (int)(fr / H);
    if (row >= plan[kPlanRows])
        return;
    const int s = plan[a.p.session_at + row];
    const int32_t* m = plan + a.p.merge_at + (long long)s * kMergeInts;
    const int pre = m[0], mine = m[4];
    if (pre + mine == 0)
        return;  // one job wrote the row itself
    const long long own_at = m[5] + fr - (long long)m[7] * H;
    const long long pre_at = m[1] + m[3] + fr - (long long)m[7] * H;
    const long long own_n = m[6], pre_n = m[2];
    auto at = [&](int i) { return i < pre ? pre_at + i * pre_n : own_at + (i - pre) * own_n; };
    float M = -INFINITY;
    for (int i = 0; i < pre + mine; ++i)
        M = fmaxf(M, a.part_ml[2 * at(i)]);
    float L = 0.0f;
    floatx4 o = {0, 0, 0, 0};
    for (int i = 0; i < pre + mine; ++i) {
        const long long p = at(i);
        const float mi = a.part_ml[2 * p];
        if (mi == -INFINITY)
            continue;  // no key of the range is the row's
        const float f = __builtin_amdgcn_exp2f(mi - M);
        L += a.part_ml[2 * p + 1] * f;
        o += *reinterpret_cast<const floatx4*>(a.part_o + p * a.kv_rank + c) * f;
    }
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

}  // namespace

hipError_t launch_latent_attention(const LatentArgs& a, int dtype, hipStream_t stream) {
    // List R first: its jobs are the longer ones.
    for (const bool rows : {true, false}) {
        if ((rows ? a.p.max_jobs_r : a.p.max_jobs_k) == 0)
            continue;
        const hipError_t e = a.q8 ? launch_attend_q8(a, dtype, rows, stream)
                                  : launch_attend_16(a, dtype, rows, stream);
        if (e != hipSuccess)
            return e;
    }
    return launch_latent_merge(a, dtype, stream);
}

hipError_t launch_latent_merge(const LatentArgs& a, int dtype, hipStream_t stream) {
    const long long n = (long long)a.p.rows * a.H * (a.kv_rank / 4);
    const dim3 grid((unsigned)((n + kThreads - 1) / kThreads));
    if (dtype == 0)
        hipLaunchKernelGGL(latent_merge_kernel<F16>, grid, dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL(latent_merge_kernel<BF16>, grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mla
