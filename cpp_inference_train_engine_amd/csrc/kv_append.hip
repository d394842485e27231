// The paged key-value cache's append: new tokens' keys, rotated by their positions, and values,
// rounded to 16 bits, into their slots; the step's queries, rotated the same way, into rows of
// their own.  No reference counterpart (its caches hold latents); the rotation is that of
// src/model/ops.cpp:88-108, and with it the one over split halves.
//   (a, b) of pair i at position p:  (a cos t - b sin t, a sin t + b cos t),  t = p f_i
//
// append_kv_kernel -- a workgroup takes a token: its threads turn the positions into rotations
//   while the first rows are on their way, then each takes 8 columns of a head at a time.
//   t is taken in 64 bits, in revolutions, and only the rest of the last one rounded to 32: at
//   position 131,071 a 32-bit product would be off by up to 2^-8 rad.
// Every row is read and written once (of split halves that are no chunks of 8 columns, or not at
// multiples of 16 bytes, the turned columns are read twice).  Few tokens: a launch and three trips to
// memory one after the other (position, slot, rows), 3.5 us for 64 tokens of 8 heads, 4.6 for 200 of
// 48 (with one workgroup a token 6.9).  Many: memory, 8,009 tokens of 48 heads of 128 columns (197 MB)
// 43 us, 4.6 TB/s where a large copy reaches 4.8.
#include "mla_common.hpp"
#include "mla_kv.hpp"

#include <algorithm>
#include <cmath>

namespace mla {
namespace {

constexpr int kMaxPairs = 128;  // dim <= 256
constexpr int kThreads = 256, kFewTokens = 1024;
typedef float f8 __attribute__((ext_vector_type(8)));

struct F32Row {
    using scalar = float;
    __device__ static float to_float(float x) { return x; }
};
struct F16Row {
    using scalar = uint16_t;
    __device__ static float to_float(uint16_t x) { return F16::to_float(x); }
};
struct BF16Row {
    using scalar = uint16_t;
    __device__ static float to_float(uint16_t x) { return BF16::to_float(x); }
};

// Threads of a token's workgroup: 8,009 tokens of 48 heads of 128 columns 45.6 us with 128 and 47.6
// with 256 for 16-bit rows, 60.7 and 57.1 for fp32 ones.
template <typename R>
constexpr int threads_of = sizeof(typename R::scalar) == 4 ? kThreads : 128;

// Eight elements from p, 16-byte loads where WIDE.
template <typename R, bool WIDE>
__device__ __forceinline__ f8 load8(const typename R::scalar* p) {
    f8 x;
    if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = R::to_float(p[i]);
    } else if constexpr (sizeof(typename R::scalar) == 4) {
        const floatx4 lo = *reinterpret_cast<const floatx4*>(p);
        const floatx4 hi = *reinterpret_cast<const floatx4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = lo[i];
            x[4 + i] = hi[i];
        }
    } else {
        const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = R::to_float((uint16_t)v[i]);
            x[2 * i + 1] = R::to_float((uint16_t)(v[i] >> 16));
        }
    }
    return x;
}

template <typename T>
__device__ __forceinline__ u32x4 rounded(const f8& x) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = T::from_float(x[2 * i]) | (uint32_t)T::from_float(x[2 * i + 1]) << 16;
    return v;
}

// PAIRED (split halves whose chunks of 8 columns pair up): a thread takes a chunk of the first half
// and its partner together, so that each is read once.
template <typename T, typename R, bool WIDE, bool PAIRED>
__global__ __launch_bounds__(kThreads) void append_kv_kernel(KvAppendArgs a) {
    __shared__ float2 turn[kMaxPairs];
    const int tid = threadIdx.x + blockIdx.y * blockDim.x, step = gridDim.y * blockDim.x;
    const int P = a.pairs, first = a.start, behind = a.start + 2 * P;
    // a head's tasks: its chunks, less those that others take along
    const int per_k = a.dim / 8 - (PAIRED ? P / 8 : 0), per_v = a.v_dim / 8;
    const int qc = a.q ? a.heads * per_k : 0, kc = a.kv_heads * per_k;
    const int tasks = qc + kc + a.kv_heads * per_v;
    const long long rec = kv_record(a.kv_heads, a.page_size, a.dim, a.v_dim);

    for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
        if (P > 0) {
            const double p = (double)a.positions[t];
            __syncthreads();  // the token before has been turned
            for (int i = threadIdx.x; i < P; i += blockDim.x) {
                const double r = p * a.frequencies[i] * 0.15915494309189533577;  // 1 / (2 pi)
                float s, c;
                sincospif((float)(2.0 * (r - rint(r))), &s, &c);
                turn[i] = float2{c, s};
            }
            __syncthreads();
        }
        const int flat = a.slot_mapping[t];
        const int page = flat / a.page_size, slot = flat - page * a.page_size;
        const bool inside = flat >= 0 && page < a.num_pool_pages;
        uint16_t* const record = a.pages + (inside ? page : 0) * rec;
        for (int e = tid; e < tasks; e += step) {
            const bool is_q = e < qc, is_v = e >= qc + kc;
            const int f = is_q ? e : is_v ? e - qc - kc : e - qc;
            const int per = is_v ? per_v : per_k, width = is_v ? a.v_dim : a.dim;
            const int h = f / per;
            int c = (f - h * per) * 8;
            if (PAIRED && !is_v && c >= first + P)
                c += P;  // (the second half is taken along)
            const auto* src = static_cast<const typename R::scalar*>(is_q ? a.q : is_v ? a.v : a.k) +
                              t * (is_q ? a.q_row : is_v ? a.v_row : a.k_row) +
                              h * (is_q ? a.q_head : is_v ? a.v_head : a.k_head) + c;
            uint16_t* const dst =
                is_q ? a.q_out + ((long long)t * a.heads + h) * a.dim + c
                     : record + (is_v ? (long long)a.kv_heads * a.page_size * a.dim : 0) +
                           ((long long)h * a.page_size + slot) * width + c;
            const bool turned = !is_v && c + 8 > first && c < behind;
            f8 x = load8<R, WIDE>(src);
            if (PAIRED && turned) {
                f8 z = load8<R, true>(src + P);
                const float2* w = turn + (c - first);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = x[i];
                    x[i] = y * w[i].x - z[i] * w[i].y;
                    z[i] = y * w[i].y + z[i] * w[i].x;
                }
                if (is_q || inside)
                    *reinterpret_cast<u32x4*>(dst + P) = rounded<T>(z);
            } else if (turned && a.adjacent) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const int j = c + i - first;
                    if (j >= 0 && j < 2 * P) {
                        const float2 w = turn[j >> 1];
                        const float y = x[i], z = x[i + 1];
                        x[i] = y * w.x - z * w.y;
                        x[i + 1] = y * w.y + z * w.x;
                    }
                }
            } else if (turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int j = c + i - first;
                    if (j >= 0 && j < 2 * P) {
                        const bool low = j < P;
                        const float z = R::to_float(src[i + (low ? P : -P)]);
                        const float2 w = turn[low ? j : j - P];
                        x[i] = low ? x[i] * w.x - z * w.y : z * w.y + x[i] * w.x;
                    }
                }
            }
            if (is_q || inside)
                *reinterpret_cast<u32x4*>(dst) = rounded<T>(x);
        }
    }
}

template <typename T, typename R>
hipError_t launch_rows(const KvAppendArgs& a, hipStream_t stream) {
    const bool paired = a.wide && !a.adjacent && a.pairs > 0;
    const int per_k = a.dim / 8 - (paired ? a.pairs / 8 : 0);
    const int tasks = (a.q ? a.heads * per_k : 0) + a.kv_heads * (per_k + a.v_dim / 8);
    const int threads = std::min(threads_of<R>, (tasks + 63) / 64 * 64);
    // few tokens: as many workgroups a token as it has tasks for
    const int split = a.T <= kFewTokens ? std::min((tasks + threads - 1) / threads, 64) : 1;
    const dim3 grid(std::min(a.T, 1 << 20), split);
    if (paired)
        hipLaunchKernelGGL((append_kv_kernel<T, R, true, true>), grid, dim3(threads), 0, stream, a);
    else if (a.wide)
        hipLaunchKernelGGL((append_kv_kernel<T, R, true, false>), grid, dim3(threads), 0, stream, a);
    else
        hipLaunchKernelGGL((append_kv_kernel<T, R, false, false>), grid, dim3(threads), 0, stream, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const KvAppendArgs& a, int row_dtype, hipStream_t stream) {
    return row_dtype == kKvF32 ? launch_rows<T, F32Row>(a, stream)
           : row_dtype == 0     ? launch_rows<T, F16Row>(a, stream)
                                : launch_rows<T, BF16Row>(a, stream);
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& a, int dtype, int row_dtype, hipStream_t stream) {
    return dtype == 0 ? launch_type<F16>(a, row_dtype, stream) : launch_type<BF16>(a, row_dtype, stream);
}

}  // namespace mla
