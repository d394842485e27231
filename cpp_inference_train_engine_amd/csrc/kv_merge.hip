// Joins the partials of mla_kv_attention: a row's weighted sums over ranges of its keys, each with
// its reference maximum and mass, become the final row.
//     M = max_i m_i,  L = sum_i l_i 2^(m_i - M),  row = sum_i o_i 2^(m_i - M) / L
// One thread per 4 columns of a row and each of GROUPS groups, which split the row's partials; each
// reads kFlight of them at once, and their states meet in LDS.
// 7.4 us for 1,392 partial rows of 8 groups of heads, 10-11 for 3,557 of 16 heads of 128 columns: two
// trips to memory one after the other and the launch, then its bytes.
#include "mla_common.hpp"
#include "mla_kv.hpp"

#include <algorithm>
#include <cmath>

namespace mla {
namespace {

constexpr int kThreads = 256, kFlight = 4;
constexpr long long kThreadsAtOnce = 1 << 19;
constexpr long long kBlocksX = 1 << 20;  // a grid's x: it has fewer than 2^32 threads there
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

template <typename T, int GROUPS>
__global__ __launch_bounds__(kThreads) void kv_merge_kernel(KvArgs a) {
    constexpr int PER = kThreads / GROUPS;  // threads of a group
    __shared__ float so[GROUPS > 1 ? kThreads * 4 : 4], sml[GROUPS > 1 ? kThreads * 2 : 4];
    const table_ptr plan = table(a.plan);
    const int tid = threadIdx.x, group = tid / PER, me = tid % PER;
    const int DV = a.p.v_dim, per_row = DV / 4, H = a.p.H, G = a.p.group;
    const long long block = blockIdx.y * (long long)gridDim.x + blockIdx.x, e = block * PER + me;
    const long long fr = e / per_row;
    const int c = (int)(e - fr * per_row) * 4;
    const long long row = fr / H;  // (past the rows in the last blocks)
    const int h = (int)(fr - row * H), kh = h / G, in_group = h - kh * G;
    // A row's entry is read with the plan's head, not behind it, and dropped if that does not fit.
    const i32x4 entry = *reinterpret_cast<const i32x4*>(
        a.plan + a.p.rows_at + (min(row, (long long)a.p.rows - 1) * G + in_group) * kKvRowInts);
    const int all = plan[kKvParts], rows = plan[kKvRows];
    const bool some = kv_plan_fits(a, plan) && all > 0 && row < rows;
    const int parts = some ? entry[1] : 0;  // 0: no such row, or one job wrote it itself
    float M = -INFINITY, L = 0.0f;
    floatx4 o = {0, 0, 0, 0};
    for (int i0 = group; i0 < parts; i0 += GROUPS * kFlight) {
        float m[kFlight], l[kFlight];
        floatx4 x[kFlight];
        float top = M;
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const int i = min(i0 + k * GROUPS, parts - 1);
            const long long p = (entry[0] + (long long)i * entry[2]) * a.p.kv_heads + kh;
            typedef float f2 __attribute__((ext_vector_type(2)));
            const f2 ml = *reinterpret_cast<const f2*>(a.part_ml + 2 * p);
            m[k] = ml[0];
            l[k] = ml[1];
            x[k] = *reinterpret_cast<const floatx4*>(a.part_o + p * DV + c);
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
    const float inv = 1.0f / L;
    u32x2 y;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        y[i] = T::from_float(o[2 * i] * inv) | (uint32_t)T::from_float(o[2 * i + 1] * inv) << 16;
    *reinterpret_cast<u32x2*>(a.out + fr * DV + c) = y;
    if (a.lse && c == 0)
        a.lse[fr] = (M + __log2f(L)) * kLn2;
}

template <typename T, int GROUPS>
void launch_groups(const KvArgs& a, hipStream_t stream) {
    constexpr int per = kThreads / GROUPS;
    const long long blocks = ((long long)a.p.rows * a.p.H * (a.p.v_dim / 4) + per - 1) / per;
    const unsigned x = (unsigned)std::min(blocks, kBlocksX);
    hipLaunchKernelGGL((kv_merge_kernel<T, GROUPS>), dim3(x, (unsigned)((blocks + x - 1) / x)),
                       dim3(kThreads), 0, stream, a);
}

template <typename T>
hipError_t launch_merge_t(const KvArgs& a, hipStream_t stream) {
    // as many groups as the GPU holds threads for at once (eight: one round of reads covers 32 partials)
    const long long threads = (long long)a.p.rows * a.p.H * (a.p.v_dim / 4);
    if (threads * 8 <= kThreadsAtOnce)
        launch_groups<T, 8>(a, stream);
    else if (threads * 2 <= kThreadsAtOnce)
        launch_groups<T, 2>(a, stream);
    else
        launch_groups<T, 1>(a, stream);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_attention(const KvArgs& a, int dtype, hipStream_t stream) {
    // The list of many rows first: its jobs are the longer ones.
    for (const bool many : {true, false}) {
        if ((many ? a.jobs_m : a.jobs_f) == 0)
            continue;
        const hipError_t e = dtype == 0 ? launch_kv_attend_f16(a, many, stream)
                                        : launch_kv_attend_bf16(a, many, stream);
        if (e != hipSuccess)
            return e;
    }
    if (a.parts == 0)
        return hipSuccess;
    return dtype == 0 ? launch_merge_t<F16>(a, stream) : launch_merge_t<BF16>(a, stream);
}

}  // namespace mla
