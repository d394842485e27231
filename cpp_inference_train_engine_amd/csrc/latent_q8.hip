// The 8-bit latent cache's append and read-back (layout and rounding: mla_q8.hpp).
//
// append_q8_kernel -- one thread quantises 8 columns of a token: two 16-byte loads of fp32, the
//   block maximum over the 4 threads of a 32-column block (two quad permutes), one exact
//   multiplication by a power of two, v_cvt_pk_fp8_f32, one 8-byte store.  Rope keys: 8 columns a
//   thread, rounded to 16 bits.
// read_q8_kernel -- one thread turns 8 values of a token into 16 bits (v_cvt_scalef32_pk_*: one
//   instruction for two values, scale included) and stores 16 bytes.
// Both read and write every byte once and have nothing else to do: launch latency for a decode
// step's rows (64 tokens of kv 128: 2.7 us), memory for many: 60,013 tokens of kv 512 read back in
// 25.3 us, 4.3 TB/s, where a large copy reaches 4.8; 7,001 of them appended in 6.0 us, 3.5 TB/s.
// (A fixed group of threads for each token, without the divisions of an element's index: 24.9 and,
// with a block's threads not all taken, 8.2 us.)
#include "mla_internal.hpp"
#include "mla_q8.hpp"

#include <algorithm>

namespace mla {
namespace {

constexpr int kThreads = 256;
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows of any fp32 alignment

// Page and slot of a flat slot; false when it lies outside the pool.
__device__ __forceinline__ bool locate(int flat, int page_size, int num_pool_pages, int& page,
                                       int& slot) {
    page = flat / page_size;
    slot = flat - page * page_size;
    return flat >= 0 && page < num_pool_pages;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void append_q8_kernel(Q8Args a) {
    const int c8s = a.kv_rank / 8, r8s = a.rope_dim / 8;
    const long long lat = (long long)a.T * c8s, total = lat + (long long)a.T * r8s;
    const long long rec = q8_page_bytes(a.page_size, a.kv_rank, a.rope_dim);
    // lat is a multiple of 4 and so is the stride: the 4 threads of a block stay together
    for (long long e = blockIdx.x * (long long)kThreads + threadIdx.x; e < total;
         e += (long long)kThreads * gridDim.x) {
        const bool latent = e < lat;
        const long long f = latent ? e : e - lat;
        const int per = latent ? c8s : r8s;
        const int t = (int)(f / per), c8 = (int)(f - (long long)t * per);
        int page, slot;
        const bool inside = locate(a.slot_mapping[t], a.page_size, a.num_pool_pages, page, slot);
        const float* src = (latent ? a.ckv : a.krope) + f * 8;
        const f4 lo = *reinterpret_cast<const f4*>(src);
        const f4 hi = *reinterpret_cast<const f4*>(src + 4);
        const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        if (latent) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                m = fmaxf(m, finite_bits(x[i]) ? fabsf(x[i]) : 0.0f);
            m = fmaxf(m, __shfl_xor(m, 1, 4));
            m = fmaxf(m, __shfl_xor(m, 2, 4));
            const int k = q8_exponent<T>(m);
            const u32x2 v = q8_encode(x, k);
            if (inside) {
                uint8_t* base = a.pages + page * rec;
                *reinterpret_cast<u32x2*>(base + q8_latent_byte(slot, c8, a.kv_rank)) = v;
                if ((c8 & 3) == 0)
                    base[q8_scale_offset(a.page_size, a.kv_rank, a.rope_dim) +
                         (long long)slot * (a.kv_rank / 32) + c8 / 4] = (uint8_t)(k + 127);
            }
        } else if (inside) {
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = T::from_float(x[2 * i]) | (uint32_t)T::from_float(x[2 * i + 1]) << 16;
            uint8_t* base = a.pages + page * rec + q8_rope_offset(a.page_size, a.kv_rank);
            *reinterpret_cast<u32x4*>(base + ((long long)(slot >> 4) * r8s + c8) * 256 +
                                      (slot & 15) * 16) = v;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void read_q8_kernel(Q8Args a) {
    const int c8s = a.kv_rank / 8, r8s = a.rope_dim / 8;
    const long long lat = (long long)a.T * c8s, total = lat + (long long)a.T * r8s;
    const long long rec = q8_page_bytes(a.page_size, a.kv_rank, a.rope_dim);
    for (long long e = blockIdx.x * (long long)kThreads + threadIdx.x; e < total;
         e += (long long)kThreads * gridDim.x) {
        const bool latent = e < lat;
        const long long f = latent ? e : e - lat;
        const int per = latent ? c8s : r8s;
        const int t = (int)(f / per), c8 = (int)(f - (long long)t * per);
        int page, slot;
        if (!locate(a.slot_mapping[t], a.page_size, a.num_pool_pages, page, slot))
            continue;
        const uint8_t* base = a.pages + page * rec;
        u32x4 v;
        if (latent) {
            const u32x2 w =
                *reinterpret_cast<const u32x2*>(base + q8_latent_byte(slot, c8, a.kv_rank));
            const uint8_t k = base[q8_scale_offset(a.page_size, a.kv_rank, a.rope_dim) +
                                   (long long)slot * (a.kv_rank / 32) + c8 / 4];
            v = q8_decode8<T>(w[0], w[1], q8_scale(k));
        } else {
            v = *reinterpret_cast<const u32x4*>(base + q8_rope_offset(a.page_size, a.kv_rank) +
                                                ((long long)(slot >> 4) * r8s + c8) * 256 +
                                                (slot & 15) * 16);
        }
        *reinterpret_cast<u32x4*>((latent ? a.ckv16 : a.krope16) + f * 8) = v;
    }
}

int blocks_of(const Q8Args& a) {
    const long long n = (long long)a.T * (a.kv_rank + a.rope_dim) / 8;
    return (int)std::min<long long>((n + kThreads - 1) / kThreads, 16384);
}

}  // namespace

hipError_t launch_append_q8(const Q8Args& a, int dtype, hipStream_t stream) {
    if (a.T == 0)
        return hipSuccess;
    if (dtype == 0)
        hipLaunchKernelGGL(append_q8_kernel<F16>, dim3(blocks_of(a)), dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL(append_q8_kernel<BF16>, dim3(blocks_of(a)), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_read_q8(const Q8Args& a, int dtype, hipStream_t stream) {
    if (a.T == 0)
        return hipSuccess;
    if (dtype == 0)
        hipLaunchKernelGGL(read_q8_kernel<F16>, dim3(blocks_of(a)), dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL(read_q8_kernel<BF16>, dim3(blocks_of(a)), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mla
