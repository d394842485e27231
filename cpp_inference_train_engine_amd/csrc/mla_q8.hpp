// The 8-bit latent cache: record layout, and the conversions between its values and fp32 or the
// cache's 16-bit type.
//
// A page record holds page_size tokens: latents (kv_rank bytes a token), rope keys (16-bit words,
// in the order of the 16-bit records), scales (one byte for each 32-column block of a token).
// Shapes are those of the tiled 16-bit records, kv_rank up to 512 and rope_dim up to 64.
//   latent (slot, r): t = slot/16, n = slot%16, j = r/32, g = r%32/8, e = r%8
//     j in a pair (2i, 2i+1):   byte t*16*kv_rank + i*1024 + (16 g + n)*16 + (j%2)*8 + e
//     a last j without a pair:  byte t*16*kv_rank + j*512 + (16 g + n)*8 + e
//   so that lane (g, n) of a wave reads the MFMA operands of two k-steps in one 16-byte load.
//   rope (slot, c):  word (t*(rope_dim/8) + c/8)*128 + n*8 + c%8 of the rope section
//   scale (slot, j): byte slot*(kv_rank/32) + j of the scale section, k + 127
// A block's values are e4m3 (OCP) times 2^k, k the smallest with max|x| <= 448 * 2^k over its
// finite values, held to the range in which every value e4m3 * 2^k is one of the 16-bit type too:
// e4m3's multiples of 2^-9 up to 448 are fp16's for k in -15..7 and bf16's normal numbers for k in
// -117..119.  So rounding to e4m3 is the only rounding, and reading a value back into the 16-bit
// type is exact.  A power of two costs e4m3, a floating type, no precision but near the bottom of
// a block (2^-9 of 224..448), and makes division by the scale exact.
#pragma once

#include "mla_common.hpp"

namespace mla {

constexpr int kQ8MaxRank = 512, kQ8MaxRope = 64;
constexpr int kQ8MaxPage = 65536;  // offsets within a page's record stay below 2^31

__host__ __device__ inline bool q8_supported(int page_size, int kv_rank, int rope_dim) {
    return page_size >= 16 && page_size <= kQ8MaxPage && kv_rank >= 32 && rope_dim >= 0 &&
           page_tiled(page_size, kv_rank, rope_dim) && kv_rank <= kQ8MaxRank &&
           rope_dim <= kQ8MaxRope;
}
__host__ __device__ inline long long q8_rope_offset(int page_size, int kv_rank) {
    return (long long)page_size * kv_rank;
}
__host__ __device__ inline long long q8_scale_offset(int page_size, int kv_rank, int rope_dim) {
    return (long long)page_size * (kv_rank + 2 * rope_dim);
}
__host__ __device__ inline long long q8_page_bytes(int page_size, int kv_rank, int rope_dim) {
    return (long long)page_size * (kv_rank + 2 * rope_dim + kv_rank / 32);
}
// Byte of the 8 values (slot, 8 c8 .. 8 c8 + 7) in the record.
__host__ __device__ inline long long q8_latent_byte(int slot, int c8, int kv_rank) {
    const int t = slot >> 4, n = slot & 15, j = c8 >> 2, g = c8 & 3, ks = kv_rank >> 5;
    const bool paired = j < (ks & ~1);
    return (long long)t * 16 * kv_rank +
           (paired ? (j >> 1) * 1024 + (16 * g + n) * 16 + (j & 1) * 8
                   : j * 512 + (16 * g + n) * 8);
}

// Range of k, by the 16-bit type.
template <typename T> struct Q8Range;
template <> struct Q8Range<F16> { static constexpr int lo = -15, hi = 7; };
template <> struct Q8Range<BF16> { static constexpr int lo = -117, hi = 119; };

// k of a block from its largest finite magnitude m 2^e, 1 <= m < 2: 448 is 1.75 * 2^8.
template <typename T>
__device__ __forceinline__ int q8_exponent(float amax) {
    const uint32_t u = __builtin_bit_cast(uint32_t, amax);
    const int k = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(k, Q8Range<T>::lo), Q8Range<T>::hi);
}

__device__ __forceinline__ bool finite_bits(float x) {
    return (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) != 0x7f800000u;
}

// Eight values x / 2^k as e4m3 (round to nearest even, saturating; infinities and NaN as 0x7f).
__device__ __forceinline__ u32x2 q8_encode(const float (&x)[8], int k) {
    const float inv = __builtin_bit_cast(float, (uint32_t)(127 - k) << 23);
    float y[8];
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool ok = finite_bits(x[i]);
        bad |= ok ? 0u : 1u << i;
        y[i] = ok ? fminf(fmaxf(x[i] * inv, -448.0f), 448.0f) : 0.0f;
    }
    u32x2 r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
        r[h] = (uint32_t)w;
    }
    if (bad) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (bad >> i & 1)
                r[i / 4] |= 0x7fu << (8 * (i % 4));  // y was 0: the byte is 0x00
    }
    return r;
}

// Four e4m3 values of a word times scale (a power of two), as 16-bit values: exact, see above.
__device__ __forceinline__ u32x2 q8_decode4(uint32_t w, float scale, F16) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true);
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
__device__ __forceinline__ u32x2 q8_decode4(uint32_t w, float scale, BF16) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
// The scale of a scale byte (k + 127 >= 10 in a well-formed cache).
__device__ __forceinline__ float q8_scale(uint32_t byte) {
    return __builtin_bit_cast(float, byte << 23);
}
template <typename T>
__device__ __forceinline__ u32x4 q8_decode8(uint32_t w0, uint32_t w1, float scale) {
    const u32x2 a = q8_decode4(w0, scale, T{}), b = q8_decode4(w1, scale, T{});
    return u32x4{a[0], a[1], b[0], b[1]};
}

// Bit 7 of each byte that holds e4m3's NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t q8_nan_bits(uint32_t w) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

}  // namespace mla
