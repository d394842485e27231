// Attention of a batch's query rows over the paged key-value cache by a plan's jobs, gfx950: the
// kernels of both lists (the units kv_attend_*.hip instantiate them).
//
// For a (query, head) row with query q at position p, and keys k_j with values v_j of its kv head,
// j <= p and (p - j < window or j < sinks):
//     s_j = q . k_j scale,   o = sum_j softmax(s)_j v_j,   lse = ln sum_j exp(s_j)
//
// Both kernels take 32 keys (a unit: two 16-token tiles, which may lie on different pages) at a
// time, 16 rows to an MFMA tile:
//     S^T = K . Q^T       v_mfma_f32_16x16x32; a lane then holds, for one row, the scores of keys
//                         4g .. 4g+3 of each tile (g = lane / 16)
//     online softmax      log2 domain in 32 bits, the reference maximum raised lazily
//     O^T += V^T . P^T    the product's key order is free as long as both operands have the same:
//                         taken as the lanes hold the scores, P^T needs no exchange between lanes.
//                         V^T: a lane takes some columns of its eight keys' rows and transposes
//                         them in registers (v_perm_b32).
// P^T enters in 16-bit parts: only the row is rounded.  bf16: two, e = hi + lo, off by 2^-17 of it at
// most.  fp16: two, off by 2^-23 of it or 2^-25, and in units where that is more than 2^-15 of some
// weight a third, of what they leave, off by 2^-47 (a row's largest weight is 2^11 at least).
//
// kv_few_kernel -- a job of at most 16 or 32 rows: each of four waves holds all of them and takes
//   every 4th unit, straight from memory into the operands' registers; the waves' states meet in LDS
//   at the end.
// kv_many_kernel -- a job of 128 rows: each of four waves holds 32 (of eight 16 above width 192).
//   They stage 32 keys (64 at width 64) together in LDS, in operand order, into one of three
//   buffers: one barrier a stage, and every LDS access is 16 bytes a lane in a row.
//
// What bounds them, and what was measured (MI355X, on which a 2 GiB copy reaches 4.8 TB/s and an
// 8,192-cubed bf16 product 1,200 TFLOP/s; operations are the formula's, the second part of P^T not
// counted):
//   few rows: memory.  Traced: 64 rows, 32 heads on kv 8 x 128, contexts of 128 .. 14,000 tokens
//     (1.69 GB) 298 us, 5.7 TB/s; two rows on 100,000 .. 131,072 tokens (0.90 GB) 154 us, 5.8; 64
//     rows, kv 8 x 64, contexts of 128 .. 4,096 (0.29 GB) 56 us, 5.1 (46 where the last cache holds
//     part of them).  One row on 1,040 tokens, kv 8 x 64: 10 us, eight workgroups with 9 units a
//     wave, one behind the other.  There a compute unit's own rate decides: 600 tokens more of
//     kv x 128 (307 KB) take it 5.4 us, and eight waves in place of four are no faster (700 tokens
//     12.5 us against 11.1).
//   many rows: both pipes of a SIMD, one after the other.  A prompt of 8,191 rows, 32 heads on kv
//     8 x 128 (550 GFLOP) 735 us, 0.75 PFLOP/s (1.1 with the second part); 4,093 rows twice through
//     a window of 1,024 (138 GFLOP) 238 us, 0.58.  A SIMD takes 1,590 cycles for a wave's stage:
//     768 are those of its 48 MFMAs (the matrix cores are busy 49 % of the time), and its 150 other
//     vector instructions, exponentials among them, take about the rest, so that its two waves
//     hardly ever use both pipes at once.  LDS is busy 25 %, the L2 holds 95 % of what is read.
//     Then at 742 us: without the staging 680, without the exponentials 697, the products and LDS
//     reads alone 536, P^T in one part 597.
//   Measured and not kept for many rows (prompt and window; each against its own time then): four
//     waves a SIMD of 16 rows 840 and 268 us (730, 240); the 32 x 32 products 780 and 250 (724, 240);
//     64 keys a stage in two buffers 758 and 247 (740, 239); vector instructions spread among the
//     MFMAs 758 and 248 (746, 245); raised priority for the products 768 and 249 (747, 245); stages
//     fetched two ahead 722 and 237 (715, 236).
//
// A key past a row's position, or between its sinks and its window, adds nothing to the row,
// whatever it holds: its score is replaced, and its value is taken as zero where no row of the
// block sees it.  Where some rows of a block see a key, non-finite values are taken out of the
// product and added to those rows alone.
#pragma once

#include "mla_common.hpp"
#include "mla_kv.hpp"

#include <climits>
#include <cmath>

namespace mla {
namespace {

// The reference maximum sits HEAD below the row's when it is set, and is raised again when a score
// passes it by more than RISE: weights stay within fp16.
// A row can be made of small weights alone, where the values of the tokens far above the others are
// zero, and a part in fp16 is a multiple of 2^-24.  So where a unit has weights below SMALL, what two
// parts leave of its weights is multiplied, too, LIFT times as large.  (SMALL is 14.5 nats below the
// row's largest at least; 2^-15 is about what scores that far apart are off by themselves.)  bf16 has
// fp32's range.  The check takes 3 % of a prompt's time (4,000 rows, 32 heads on kv 8 x 128: 216 us,
// 211 without), the third part up to half as much again (216 us with scores spread by 1 nat, 244 by
// 2, 317 by 4, where every unit needs it); decode rows wait for memory all the same.
template <typename T>
struct Weights {
    static constexpr bool REST = false;
    static constexpr float HEAD = 6.0f, RISE = 14.0f;
};
template <>
struct Weights<F16> {
    static constexpr bool REST = true;
    static constexpr float HEAD = 11.0f, RISE = 15.0f, SMALL = 0x1p-10f, LIFT = 0x1p22f;
    static constexpr uint16_t SMALL_HALF = 0x1400;  // SMALL in fp16
};

// n / d and the rest by a product with floor(2^32 / d) (2^32 - 1 for d = 1): one too small at most
// for n < 2^32.
__device__ __forceinline__ int quotient(int n, int d, uint32_t inverse, int& rest) {
    int q = (int)(((unsigned long long)(unsigned)n * inverse) >> 32);
    rest = n - q * d;
    if (rest >= d) {
        ++q;
        rest -= d;
    }
    return q;
}

// Two values rounded to 16 bits (to nearest even) in one word: one instruction.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef typename T::scalar s2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), s2));
}

template <typename T>
__device__ __forceinline__ bool nonfinite(uint32_t half) {
    return (half & T::exp_mask) == T::exp_mask;
}
// Halves of v whose exponent is all ones become 0; true if there was one.
template <typename T>
__device__ __forceinline__ bool drop_nonfinite(uint32_t& v) {
    const bool lo = nonfinite<T>(v), hi = nonfinite<T>(v >> 16);
    v &= (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
    return lo || hi;
}

// A job, and what its rows see.
struct Job {
    int session, q0, f0, rows, u0, u1, ctx, part;
    int pa, pb;      // positions of its first and last row
    int lo_a, lo_b;  // first keys of their windows
    KvUnits units;
};
__device__ __forceinline__ bool take_job(const KvArgs& a, bool many, int index, Job& j) {
    const table_ptr plan = table(a.plan);
    const table_ptr d = plan + (many ? a.p.jobs_m_at : a.p.jobs_f_at) + (long long)index * kKvJobInts;
    j.session = d[0];
    j.q0 = d[1];
    j.f0 = d[2];
    j.rows = d[3];
    j.u0 = d[4];
    j.u1 = d[5];
    j.ctx = d[6];
    j.part = d[7];
    // no such job; or a plan for other sizes, or a failed one, or not the build that the host knows
    if (index >= plan[many ? kKvJobsM : kKvJobsF] || !kv_plan_fits(a, plan))
        return false;
    int r;
    j.pa = j.ctx + quotient(j.f0, a.p.group, a.group_inverse, r);
    j.pb = j.ctx + quotient(j.f0 + j.rows - 1, a.p.group, a.group_inverse, r);
    const int W = a.p.window;
    j.lo_a = j.pa >= W ? j.pa - W + 1 : 0;
    j.lo_b = j.pb >= W ? j.pb - W + 1 : 0;
    j.units = kv_units(j.pa, j.pb, W, a.p.sinks);
    return true;
}
// First key of the u-th unit that the block sees.
__device__ __forceinline__ int first_key(const Job& j, int u) {
    return (u < j.units.sink_units ? u : u + j.units.skip) * kKvTile;
}

// The units that rows at positions from `first` on, the last of them with a window from `lo` on, all
// see in full: some of the sinks', some of the window's.
struct Full {
    int sinks, from, to;
    __device__ __forceinline__ Full(const Job& j, int first, int lo, int held) {
        const int behind = (first + 1) / kKvTile;
        sinks = min(min(held / kKvTile, behind), j.units.sink_units);
        from = (int)(((unsigned)lo + kKvTile - 1) / kKvTile) - j.units.skip;
        to = behind - j.units.skip;
    }
    __device__ __forceinline__ bool has(int u) const { return u < sinks || (u >= from && u < to); }
};

// An element at a uniform address and the lane's 32-bit distance in bytes.
template <typename E>
__device__ __forceinline__ E fetch(const uint16_t* base, uint32_t bytes) {
    return *reinterpret_cast<const E*>(reinterpret_cast<const char*>(base) + bytes);
}

// Page ids of a unit's two tiles, and their places there.
struct Pages {
    int id0, id1, in0, in1;
    __device__ __forceinline__ int id(int tt) const { return tt ? id1 : id0; }
    __device__ __forceinline__ int in(int tt) const { return tt ? in1 : in0; }
};

// What both kernels share: T 16-bit type, HK and HV widths of keys and values (the head's sizes in
// EXACT instantiations, at least those in the others), CW consecutive columns of V that a lane
// transposes (a tile of O^T holds every CW-th), N tiles of 16 rows a wave.
template <typename T, int HK, int HV, bool EXACT, int CW, int N>
struct Attend {
    static constexpr int KS = HK / 32, NT = HV / 16, NC = NT / CW;
    using V8 = typename T::vec8;

    const KvArgs& a;
    const Job& job;
    const int D, DV, lane, g, n, head;
    const table_ptr ptab;
    const uint16_t *keys_of_head, *values_of_head;  // of page 0
    const long long record;
    V8 q[N][KS];
    int pos[N], lo[N];  // of the lane's row in each tile
    float m[N], l[N];
    floatx4 acc[N][NT];

    __device__ __forceinline__ Attend(const KvArgs& a_, const Job& j, int lane_, int head_, int row0)
        : a(a_), job(j), D(EXACT ? HK : a_.p.dim), DV(EXACT ? HV : a_.p.v_dim), lane(lane_),
          g(lane_ >> 4), n(lane_ & 15), head(head_),
          ptab(table(a_.page_table + (long long)j.session * a_.max_pages)),
          keys_of_head(a_.pages + (long long)head_ * a_.p.page_size * D),
          values_of_head(a_.pages + (long long)a_.p.kv_heads * a_.p.page_size * D +
                         (long long)head_ * a_.p.page_size * DV),
          record(kv_record(a_.p.kv_heads, a_.p.page_size, D, DV)) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const int r = min(row0 + 16 * t + n, j.rows - 1);  // rows past the block repeat its last
            int in_group;
            const int i = quotient(j.f0 + r, a.p.group, a.group_inverse, in_group);
            pos[t] = j.ctx + i;
            lo[t] = pos[t] >= a.p.window ? pos[t] - a.p.window + 1 : 0;
            const uint16_t* src =
                a.q + (((long long)j.q0 + i) * a.p.H + head * a.p.group + in_group) * D;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int c = 32 * s + 8 * g;
                V8 v = {};
                if (EXACT || c < D)
                    v = *reinterpret_cast<const V8*>(src + c);
                q[t][s] = v;
            }
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int i2 = 0; i2 < NT; ++i2)
                acc[t][i2] = floatx4{0, 0, 0, 0};
        }
    }

    // Units past the last are read as if they were the last (and not used).
    __device__ __forceinline__ Pages find_pages(int u) const {
        Pages p;
        const int t = first_key(job, min(u, job.u1 - 1)) >> 4, tpp = a.p.page_size >> 4;
        p.id0 = ptab[quotient(t, tpp, a.tpp_inverse, p.in0)];
        // a tile behind the last key is not on a page: the one before it is read again
        const int t1 = min(t + 1, job.pb >> 4);
        p.id1 = ptab[quotient(t1, tpp, a.tpp_inverse, p.in1)];
        return p;
    }
    // (Ids were checked by the metadata's build; the bound is for memory's sake.)
    __device__ __forceinline__ long long page_at(int id) const {
        return (long long)min((unsigned)id, (unsigned)a.num_pool_pages - 1) * record;
    }
    __device__ __forceinline__ const uint16_t* keys_at(const Pages& p, int tt) const {
        return keys_of_head + page_at(p.id(tt)) + (long long)p.in(tt) * 16 * D;
    }
    __device__ __forceinline__ const uint16_t* values_at(const Pages& p, int tt) const {
        return values_of_head + page_at(p.id(tt)) + (long long)p.in(tt) * 16 * DV;
    }
    // Key operand of a tile's step s: columns 32s + 8g .. of key n.
    __device__ __forceinline__ u32x4 load_key(const uint16_t* tile, int s) const {
        const int c = 32 * s + 8 * g;
        if constexpr (EXACT)
            return fetch<u32x4>(tile + 32 * s, (uint32_t)(n * HK + 8 * g) * 2);
        const u32x4 v = fetch<u32x4>(tile, (uint32_t)(n * D + min(c, D - 8)) * 2);
        return c < D ? v : u32x4{0, 0, 0, 0};
    }
    // The lane's columns of chunk c of a tile's row 4g + i.
    struct Row {
        uint32_t w[CW / 2];
    };
    __device__ __forceinline__ Row load_value(const uint16_t* tile, int c, int i) const {
        typedef uint32_t words __attribute__((ext_vector_type(CW / 2)));
        const int col = 16 * CW * c + CW * n;
        Row r;
        words v;
        if constexpr (EXACT)
            v = fetch<words>(tile + 16 * CW * c + i * HV, (uint32_t)(4 * g * HV + CW * n) * 2);
        else
            v = fetch<words>(tile + i * DV, (uint32_t)(4 * g * DV + min(col, DV - CW)) * 2);
#pragma unroll
        for (int k = 0; k < CW / 2; ++k)
            r.w[k] = v[k];  // (columns past the head's are computed and not stored)
        return r;
    }
    // Operand e of eight rows: their columns e, two keys a word.
    __device__ __forceinline__ static u32x4 transposed(const Row (&x)[8], int e) {
        u32x4 v;
        const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            v[k] = __builtin_amdgcn_perm(x[2 * k + 1].w[e >> 1], x[2 * k].w[e >> 1], sel);
        return v;
    }
    // Whether some row of the block sees the key.
    __device__ __forceinline__ bool some_row_sees(int key) const {
        return key <= job.pb && (key >= job.lo_a || key < a.p.sinks);
    }
    // The lane's rows (tile r / 4, row 4g + r % 4) of a unit that not every row of the block sees:
    // values that no row sees become zero.  With several positions in the block non-finite ones
    // become zero, too; true if this lane had one.
    __device__ __forceinline__ bool clean(Row (&x)[8], int key0) const {
        bool bad = false;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const bool keep = some_row_sees(key0 + 16 * (r >> 2) + 4 * g + (r & 3));
#pragma unroll
            for (int k = 0; k < CW / 2; ++k) {
                x[r].w[k] = keep ? x[r].w[k] : 0;
                if (job.pa != job.pb)
                    bad |= drop_nonfinite<T>(x[r].w[k]);
            }
        }
        return bad;
    }

    // Scores of keys that a row does not see are replaced.
    __device__ __forceinline__ void mask(floatx4 (&sc)[N][2], int key0) const {
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 16 * tt + 4 * g + i;
                    const bool sees = (key <= pos[t]) & ((key >= lo[t]) | (key < a.p.sinks));
                    sc[t][tt][i] = sees ? sc[t][tt][i] : -INFINITY;
                }
    }
    // The rows' reference maxima, and what was summed under lower ones, follow the scores of U units.
    template <int U>
    __device__ __forceinline__ void raise(const floatx4 (&sc)[U][N][2]) {
        using W = Weights<T>;
        float mp[N];
        bool above = false;
#pragma unroll
        for (int t = 0; t < N; ++t) {
            mp[t] = -INFINITY;  // of the lane's scores (NaN is passed over)
#pragma unroll
            for (int x = 0; x < U; ++x)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mp[t] = fmaxf(mp[t], sc[x][t][tt][i]);
            mp[t] *= a.scale_log2;
            above |= mp[t] > m[t] + W::RISE;
        }
        if (__builtin_amdgcn_ballot_w64(above) == 0)
            return;
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const float top = rows_max(mp[t]) - W::HEAD;
            // (with less room above, all rows at once: one raise in place of several; 4,093 rows
            // twice through a window then took 250 us in place of 261, and 245 now)
            const float m_new = top > m[t] + (W::REST ? 0.0f : W::RISE - W::HEAD) ? top : m[t];
            const bool had = m[t] != -INFINITY;  // the row has accumulated state
            if (__builtin_amdgcn_ballot_w64(had && m_new > m[t])) {
                const float alpha = had ? __builtin_amdgcn_exp2f(m[t] - m_new) : 1.0f;
                l[t] *= alpha;
#pragma unroll
                for (int k = 0; k < NT; ++k)
                    acc[t][k] *= alpha;
            }
            m[t] = m_new;
        }
    }
    // The least of some weights' high parts, by their bits: these are ordered as the weights are.
    struct Least {
        typedef uint16_t u2 __attribute__((ext_vector_type(2)));
        u2 x = {0xffff, 0xffff};
        __device__ __forceinline__ void add(uint32_t word) {
            x = __builtin_elementwise_min(x, __builtin_bit_cast(u2, word));
        }
        // Whether a lane has a weight below SMALL (a zero counts, too).
        __device__ __forceinline__ bool small() const {
            const int a = x[0], b = x[1];
            return __builtin_amdgcn_ballot_w64(min(a, b) < Weights<T>::SMALL_HALF) != 0;
        }
    };
    // Scores become weights, also in two parts, and are summed.
    __device__ __forceinline__ void weights(floatx4 (&sc)[N][2], V8 (&hi)[N], V8 (&lw)[N], Least& least) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const float ref = m[t] == -INFINITY ? 0.0f : m[t];
            float sum = 0.0f;
            u32x4 h, w;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const floatx4 y = sc[t][x >> 1];
                const float e0 = __builtin_amdgcn_exp2f(fmaf(y[2 * (x & 1)], a.scale_log2, -ref));
                const float e1 = __builtin_amdgcn_exp2f(fmaf(y[2 * (x & 1) + 1], a.scale_log2, -ref));
                sum += e0 + e1;
                h[x] = pack2<T>(e0, e1);
                w[x] = pack2<T>(e0 - T::to_float((uint16_t)h[x]), e1 - T::to_float((uint16_t)(h[x] >> 16)));
                least.add(h[x]);
                sc[t][x >> 1][2 * (x & 1)] = e0;
                sc[t][x >> 1][2 * (x & 1) + 1] = e1;
            }
            hi[t] = __builtin_bit_cast(V8, h);
            lw[t] = __builtin_bit_cast(V8, w);
            l[t] += sum;
        }
    }

    // Adds what is left of a unit's weights, if some are below SMALL.  `operand`: tile i of its V^T.
    template <typename F>
    __device__ __forceinline__ void add_rest(const floatx4 (&e)[N][2], const V8 (&hi)[N], const V8 (&lw)[N],
                                             F&& operand) {
        using W = Weights<T>;
        uint32_t least = ~0u;  // of the weights' bits less one: those of zero are the largest
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = e[t][i >> 2][i & 3];  // (an element itself is not cast right)
                least = min(least, __builtin_bit_cast(uint32_t, y) - 1);
            }
        if (__builtin_amdgcn_ballot_w64(least < __builtin_bit_cast(uint32_t, W::SMALL) - 1) == 0)
            return;
        V8 rest[N];
#pragma unroll
        for (int t = 0; t < N; ++t) {
            u32x4 r;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                float y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    y[i] = (e[t][x >> 1][2 * (x & 1) + i] - static_cast<float>(hi[t][2 * x + i]) -
                            static_cast<float>(lw[t][2 * x + i])) * W::LIFT;
                r[x] = pack2<T>(y[0], y[1]);
            }
            rest[t] = __builtin_bit_cast(V8, r);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const V8 x = operand(i);
#pragma unroll
            for (int t = 0; t < N; ++t)
                acc[t][i] += T::mma32(x, rest[t], floatx4{0, 0, 0, 0}) * (1.0f / W::LIFT);
        }
    }

    // Adds what clean() took out, to the rows that see it: values read again from memory.
    __device__ __forceinline__ void add_nonfinite(const Pages& p, int key0,
                                                            const V8 (&hi)[N], const V8 (&lw)[N]) {
#pragma unroll 1
        for (int k = 0; k < kKvTile; ++k) {
            const int tt = k >> 4, gg = (k >> 2) & 3, i = k & 3, key = key0 + k;
            if (!some_row_sees(key))
                continue;
            const uint16_t* row = values_at(p, tt) + (4 * gg + i) * DV;
            float w[N];
            bool sees[N];
#pragma unroll
            for (int t = 0; t < N; ++t) {
                float e = 0.0f;
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (x == 4 * tt + i)
                        e = static_cast<float>(hi[t][x]) + static_cast<float>(lw[t][x]);
                w[t] = __shfl(e, 16 * gg + n, 64);
                sees[t] = key <= pos[t] && (key >= lo[t] || key < a.p.sinks);
            }
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int col = column(x, y);
                    const uint16_t v = EXACT || col < DV ? row[col] : 0;
                    if (nonfinite<T>(v))
#pragma unroll
                        for (int t = 0; t < N; ++t)
                            if (sees[t])
                                acc[t][x][y] += w[t] * T::to_float(v);
                }
        }
    }

    // Column of a row that element y of tile x of O^T holds in this lane.
    __device__ __forceinline__ int column(int x, int y) const {
        return 16 * CW * (x / CW) + CW * (4 * g + y) + x % CW;
    }
};

// Waves a SIMD: as many as hold a unit, the rows and O^T without spilling, where there is such a
// number.  (64 decode rows, kv 4 x 256: 168 us at one wave, 195 at two, which spill; kv 8 x 96 in the
// kernel of width 128: 131 at two, 154 at three.)  At two waves some registers spill in three
// instances: 192 on 128 in blocks of 32 rows 4 (fp16: 25), the same for smaller heads 25 (66), and
// width 256 for smaller heads 59 (61).
constexpr int few_occupancy(int width, int tiles, bool exact) {
    return width == 64                ? 5 - tiles
           : width == 128 && exact    ? 4 - tiles
           : width == 256 && exact    ? 1
                                      : 2;
}

template <typename T, int HK, int HV, int N, bool EXACT>
__global__ __launch_bounds__(kKvThreads) __attribute__((
    amdgpu_waves_per_eu(few_occupancy(HK, N, EXACT), 8))) void kv_few_kernel(KvArgs a) {
    constexpr int CW = HV >= 128 ? 8 : 4, PITCH = HV + 4;
    using A = Attend<T, HK, HV, EXACT, CW, N>;
    using V8 = typename T::vec8;
    __shared__ __attribute__((aligned(16))) float smem[4][16 * PITCH + 32];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int index = (int)(blockIdx.x / (unsigned)a.p.kv_heads);
    const int head = (int)(blockIdx.x - (unsigned)index * a.p.kv_heads);
    Job job;
    if (!take_job(a, false, index, job))
        return;
    A s(a, job, tid & 63, head, 0);

    u32x4 k[2][A::KS];
    typename A::Row v[A::NC][8];
    auto load_keys = [&](const Pages& p) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int st = 0; st < A::KS; ++st)
                k[tt][st] = s.load_key(s.keys_at(p, tt), st);
    };
    auto load_values = [&](const Pages& p) {
#pragma unroll
        for (int c = 0; c < A::NC; ++c)
#pragma unroll
            for (int r = 0; r < 8; ++r)
                v[c][r] = s.load_value(s.values_at(p, r >> 2), c, r & 3);
    };
    const Full full_units(job, job.pa, job.lo_b, a.p.sinks);
    int u = job.u0 + wave;
    Pages now{}, next{};
    if (u < job.u1) {
        now = s.find_pages(u);
        load_keys(now);
        load_values(now);
        next = s.find_pages(u + 4);
    }
    for (; u < job.u1; u += 4) {
        const int key0 = first_key(job, u);
        floatx4 sc[1][N][2];
#pragma unroll
        for (int t = 0; t < N; ++t)
            sc[0][t][0] = sc[0][t][1] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < A::KS; ++st)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int t = 0; t < N; ++t)
                    sc[0][t][tt] = T::mma32(__builtin_bit_cast(V8, k[tt][st]), s.q[t][st], sc[0][t][tt]);
        load_keys(next);
        const bool full = full_units.has(u);
        if (!full)
            s.mask(sc[0], key0);
        s.raise(sc);
        V8 hi[N], lw[N];
        typename A::Least least;
        s.weights(sc[0], hi, lw, least);
        bool bad = false;
        if (!full)
#pragma unroll
            for (int c = 0; c < A::NC; ++c)
                bad |= s.clean(v[c], key0);
        if constexpr (Weights<T>::REST)
            if (least.small())
                s.add_rest(sc[0], hi, lw, [&](int i) {
                    return __builtin_bit_cast(V8, A::transposed(v[i / CW], i % CW));
                });
#pragma unroll
        for (int c = 0; c < A::NC; ++c)
#pragma unroll
            for (int e = 0; e < CW; ++e) {
                const V8 x = __builtin_bit_cast(V8, A::transposed(v[c], e));
#pragma unroll
                for (int t = 0; t < N; ++t)
                    s.acc[t][c * CW + e] = T::mma32(x, hi[t], s.acc[t][c * CW + e]);
#pragma unroll
                for (int t = 0; t < N; ++t)
                    s.acc[t][c * CW + e] = T::mma32(x, lw[t], s.acc[t][c * CW + e]);
            }
        if (__builtin_amdgcn_ballot_w64(bad))
            s.add_nonfinite(now, key0, hi, lw);
        load_values(next);
        now = next;
        next = s.find_pages(u + 8);
    }

    // ---- the waves' states become rows, or partials ----
    const int DV = s.DV, per_row = DV / 4;
#pragma unroll
    for (int t = 0; t < N; ++t) {
        if (16 * t >= job.rows)
            break;
        const float l = rows_sum(s.l[t]);
        float* mine = smem[wave];
        if (t > 0)
            __syncthreads();  // the rows before have been read
#pragma unroll
        for (int c = 0; c < A::NC; ++c)
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int e = 0; e < CW; e += 4) {
                    const int x = c * CW + e;
                    *reinterpret_cast<floatx4*>(mine + s.n * PITCH + s.column(x, y)) = floatx4{
                        s.acc[t][x][y], s.acc[t][x + 1][y], s.acc[t][x + 2][y], s.acc[t][x + 3][y]};
                }
        if (s.g == 0) {
            mine[16 * PITCH + s.n] = s.m[t];
            mine[16 * PITCH + 16 + s.n] = l;
        }
        __syncthreads();
        for (int e = tid; e < min(job.rows - 16 * t, 16) * per_row; e += kKvThreads) {
            const int r = e / per_row, c = (e - r * per_row) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w)
                M = fmaxf(M, smem[w][16 * PITCH + r]);
            float L = 0.0f;
            floatx4 o = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float mv = smem[w][16 * PITCH + r];
                // A sum of NaN may come with a maximum of -inf (all scores NaN): weight 0 keeps it.
                const float f = mv == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mv - M);
                L += smem[w][16 * PITCH + 16 + r] * f;
                o += *reinterpret_cast<const floatx4*>(&smem[w][r * PITCH + c]) * f;
            }
            if (job.part < 0) {
                int in_group;
                const int i = quotient(job.f0 + 16 * t + r, a.p.group, a.group_inverse, in_group);
                const long long row = ((long long)job.q0 + i) * a.p.H + head * a.p.group + in_group;
                const float inv = 1.0f / L;
                *reinterpret_cast<u32x2*>(a.out + row * DV + c) =
                    u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
                if (a.lse && c == 0)
                    a.lse[row] = (M + __log2f(L)) * kLn2;
            } else {
                const long long row = ((long long)job.part + 16 * t + r) * a.p.kv_heads + head;
                *reinterpret_cast<floatx4*>(a.part_o + row * DV + c) = o;
                if (c == 0) {
                    a.part_ml[2 * row] = M;
                    a.part_ml[2 * row + 1] = L;
                }
            }
        }
    }
}

constexpr int many_waves(int width) { return width == 256 ? 8 : 4; }

template <typename T, int HK, int HV, bool EXACT>
__global__ __launch_bounds__(64 * many_waves(HK)) __attribute__((
    amdgpu_waves_per_eu(2, 8))) void kv_many_kernel(KvArgs a) {
    constexpr int NW = many_waves(HK), N = kKvManyRows / (16 * NW), CW = 2;
    constexpr int U = HK == 64 ? 2 : 1;  // units of a stage
    using A = Attend<T, HK, HV, EXACT, CW, N>;
    using V8 = typename T::vec8;
    // a stage in operand order, 1 KB each: keys [unit][tile][step], values [unit][tile of O^T]
    constexpr int KW = U * 2 * A::KS * 512, STAGE = KW + U * A::NT * 512;
    constexpr int KO = U * 2 * A::KS / NW;  // key operands that a wave stages
    static_assert(KO * NW == U * 2 * A::KS && A::KS % KO == 0 && U * A::NC == NW,
                  "a wave's share of a stage");
    __shared__ __attribute__((aligned(16))) uint16_t smem[3][STAGE];
    __shared__ int marks[3][NW];  // whether a wave took non-finite values out of the stage
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int index = (int)(blockIdx.x / (unsigned)a.p.kv_heads);
    const int head = (int)(blockIdx.x - (unsigned)index * a.p.kv_heads);
    Job job;
    if (!take_job(a, true, index, job))
        return;
    const int row0 = wave * 16 * N;
    A s(a, job, tid & 63, head, row0);

    // the first and last window, and the first position, of the wave's rows
    int r;
    const int wa = job.ctx + quotient(job.f0 + min(row0, job.rows - 1), a.p.group, a.group_inverse, r);
    const int wb = job.ctx + quotient(job.f0 + min(row0 + 16 * N, job.rows) - 1, a.p.group, a.group_inverse, r);
    const int lo_wb = wb >= a.p.window ? wb - a.p.window + 1 : 0;

    const Full full_wave(job, wa, lo_wb, a.p.sinks), full_block(job, job.pa, job.lo_b, a.p.sinks);

    // ---- what the wave stages: key operands of one tile and 32 columns of the values of one unit ----
    const int su = wave / A::NC, vc = wave % A::NC, o0 = KO * wave % (2 * A::KS);
    // Where a stage's tiles lie (bytes from the head's first page): lane i of these holds the places
    // of stage (group of 64) + i.
    long long key_at = 0, value_at0 = 0, value_at1 = 0;
    auto find_tiles = [&](int st) {
        const int t = first_key(job, min(job.u0 + (st + s.lane) * U + su, job.u1 - 1)) >> 4;
        const int tpp = a.p.page_size >> 4, t1 = min(t + 1, job.pb >> 4);
        int in0, in1;
        const int32_t* ids = a.page_table + (long long)job.session * a.max_pages;
        const int id0 = ids[quotient(t, tpp, a.tpp_inverse, in0)];
        const int id1 = ids[quotient(t1, tpp, a.tpp_inverse, in1)];
        const long long p0 = s.page_at(id0), p1 = s.page_at(id1);
        key_at = 2 * (o0 / A::KS ? p1 + (long long)in1 * 16 * s.D : p0 + (long long)in0 * 16 * s.D);
        value_at0 = 2 * (p0 + (long long)in0 * 16 * s.DV);
        value_at1 = 2 * (p1 + (long long)in1 * 16 * s.DV);
    };
    auto of_lane = [&](long long x, int i) {
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, i);
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((unsigned long long)x >> 32), i);
        return (long long)((unsigned long long)hi << 32 | lo);
    };
    auto at = [](const uint16_t* p, long long bytes) {
        return reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(p) + bytes);
    };
    struct Loaded {
        u32x4 k[KO];
        typename A::Row v[8];
    };
    auto load = [&](Loaded& x, int st) {
        const int i = st & 63;
        const uint16_t* kt = at(s.keys_of_head, of_lane(key_at, i));
        const uint16_t* v0 = at(s.values_of_head, of_lane(value_at0, i));
        const uint16_t* v1 = at(s.values_of_head, of_lane(value_at1, i));
#pragma unroll
        for (int i2 = 0; i2 < KO; ++i2)
            x.k[i2] = s.load_key(kt, o0 % A::KS + i2);
#pragma unroll
        for (int i2 = 0; i2 < 8; ++i2)
            x.v[i2] = s.load_value(i2 < 4 ? v0 : v1, vc, i2 & 3);
    };
    auto clean = [&](Loaded& x, int st, int b) {
        const int u = min(job.u0 + st * U + su, job.u1 - 1);
        if (!full_block.has(u)) {
            const bool bad = __builtin_amdgcn_ballot_w64(s.clean(x.v, first_key(job, u))) != 0;
            if (s.lane == 0)
                marks[b][wave] = bad;
        }
    };
    auto store = [&](const Loaded& x, int b) {
        uint16_t* const buf = smem[b] + s.lane * 8;
#pragma unroll
        for (int i = 0; i < KO; ++i)
            *reinterpret_cast<u32x4*>(buf + (su * 2 * A::KS + o0 + i) * 512) = x.k[i];
#pragma unroll
        for (int e = 0; e < CW; ++e)
            *reinterpret_cast<u32x4*>(buf + KW + (su * A::NT + vc * CW + e) * 512) = A::transposed(x.v, e);
    };
    constexpr int NK = U * 2 * A::KS, NV = U * A::NT, AHEAD = 4;
    auto read = [&](const uint16_t* p, int slot) {
        return *reinterpret_cast<const V8*>(p + s.lane * 8 + slot * 512);
    };
    const int stages = (job.u1 - job.u0 + U - 1) / U;
    Loaded x;
    find_tiles(0);
    {
        Loaded first;
        load(first, 0);
        load(x, 1);
        clean(first, 0, 0);
        store(first, 0);
        clean(x, 1, 1);
        store(x, 1);
        load(x, 2);
    }
    // Stage st lies in buffer b, stage st + 1 in b1; b2, free since the last barrier, takes stage
    // st + 2.  (Units behind the last are staged as the last and not used.)
    int b = 0, b1 = 1, b2 = 2;
    __syncthreads();
    // The first operands of a stage's scores are read behind the weights of the one before it.
    constexpr int EARLY = A::KS <= 4 ? NK : 4;
    V8 ko[NK];
#pragma unroll
    for (int i = 0; i < EARLY; ++i)
        ko[i] = read(smem[b], i);
    for (int st = 0; st < stages; ++st) {
        clean(x, st + 2, b2);
        if (((st + 3) & 63) == 0)
            find_tiles(st + 3);
        // ---- scores; beside them stage st + 2 goes to LDS, and stage st + 3 is sent for ----
#pragma unroll
        for (int i = EARLY; i < NK; ++i)
            ko[i] = read(smem[b], i);
        store(x, b2);
        load(x, st + 3);
        floatx4 sc[U][N][2];
#pragma unroll
        for (int x = 0; x < U; ++x) {
#pragma unroll
            for (int t = 0; t < N; ++t)
                sc[x][t][0] = sc[x][t][1] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < A::KS; ++i)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int t = 0; t < N; ++t)
                        sc[x][t][tt] = T::mma32(ko[(x * 2 + tt) * A::KS + i], s.q[t][i], sc[x][t][tt]);
        }
        V8 ring[AHEAD];
        // the first of the values' operands on their way while the weights are computed
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            ring[i] = read(smem[b] + KW, i);
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const int u = job.u0 + st * U + x;
            if (!full_wave.has(u) || u >= job.u1)
                s.mask(sc[x], u < job.u1 ? first_key(job, u) : INT_MAX - 31);
        }
        s.raise(sc);
        V8 hi[U][N], lw[U][N];
        typename A::Least least;
#pragma unroll
        for (int x = 0; x < U; ++x)
            s.weights(sc[x], hi[x], lw[x], least);
        if constexpr (Weights<T>::REST)
            if (least.small())
#pragma unroll
                for (int x = 0; x < U; ++x)
                    s.add_rest(sc[x], hi[x], lw[x], [&](int i) { return read(smem[b] + KW, x * A::NT + i); });
#pragma unroll
        for (int i = 0; i < EARLY; ++i)
            ko[i] = read(smem[b1], i);
#pragma unroll
        for (int i = 0; i < NV; i += 2) {  // (two tiles at a time: a sum is added to every 4th product)
            const V8 y[2] = {ring[i % AHEAD], ring[(i + 1) % AHEAD]};
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (i + j + AHEAD < NV)
                    ring[(i + j) % AHEAD] = read(smem[b] + KW, i + j + AHEAD);
            const int x = i / A::NT, tile = i % A::NT;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int t = 0; t < N; ++t)
                    s.acc[t][tile + j] = T::mma32(y[j], hi[x][t], s.acc[t][tile + j]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int t = 0; t < N; ++t)
                    s.acc[t][tile + j] = T::mma32(y[j], lw[x][t], s.acc[t][tile + j]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const int u = job.u0 + st * U + x;
            if (u < job.u1 && !full_block.has(u)) {
                bool bad = false;
#pragma unroll
                for (int w = 0; w < A::NC; ++w)
                    bad |= marks[b][x * A::NC + w] != 0;
                if (__builtin_amdgcn_readfirstlane(bad))
                    s.add_nonfinite(s.find_pages(u), first_key(job, u), hi[x], lw[x]);
            }
        }
        __syncthreads();
        const int b0 = b;
        b = b1;
        b1 = b2;
        b2 = b0;
    }

    // ---- rows, or partials ----
#pragma unroll
    for (int t = 0; t < N; ++t) {
        const float l = rows_sum(s.l[t]);
        const int row = row0 + 16 * t + s.n;
        if (row >= job.rows)
            continue;
        int in_group;
        const int i = quotient(job.f0 + row, a.p.group, a.group_inverse, in_group);
        const long long at = job.part < 0
                                 ? ((long long)job.q0 + i) * a.p.H + head * a.p.group + in_group
                                 : ((long long)job.part + row) * a.p.kv_heads + head;
        const float inv = 1.0f / l;
#pragma unroll
        for (int x = 0; x < A::NT; x += 2) {  // eight columns a lane of two tiles
            const int col = s.column(x, 0);
            if (!EXACT && col >= s.DV)
                continue;
            if (job.part < 0) {
                u32x4 o;
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    o[y] = pack2<T>(s.acc[t][x][y] * inv, s.acc[t][x + 1][y] * inv);
                *reinterpret_cast<u32x4*>(a.out + at * s.DV + col) = o;
            } else {
#pragma unroll
                for (int y = 0; y < 4; y += 2)
                    *reinterpret_cast<floatx4*>(a.part_o + at * s.DV + col + 2 * y) =
                        floatx4{s.acc[t][x][y], s.acc[t][x + 1][y], s.acc[t][x][y + 1],
                                s.acc[t][x + 1][y + 1]};
            }
        }
        if (s.g == 0) {
            if (job.part < 0) {
                if (a.lse)
                    a.lse[at] = (s.m[t] + __log2f(l)) * kLn2;
            } else {
                a.part_ml[2 * at] = s.m[t];
                a.part_ml[2 * at + 1] = l;
            }
        }
    }
}

template <typename T, int HK, int HV, bool EXACT>
hipError_t launch_one(const KvArgs& a, bool many, hipStream_t stream) {
    const dim3 grid((unsigned)((many ? a.jobs_m : a.jobs_f) * a.p.kv_heads));
    if (many)
        hipLaunchKernelGGL((kv_many_kernel<T, HK, HV, EXACT>), grid, dim3(64 * many_waves(HK)), 0,
                           stream, a);
    else if (HK == 256 || a.p.few_rows == 16)
        hipLaunchKernelGGL((kv_few_kernel<T, HK, HV, 1, EXACT>), grid, dim3(kKvThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((kv_few_kernel<T, HK, HV, HK == 256 ? 1 : 2, EXACT>), grid, dim3(kKvThreads),
                           0, stream, a);
    return hipGetLastError();
}

template <typename T, int HK, int HV>
hipError_t launch_width(const KvArgs& a, bool many, hipStream_t stream) {
    return a.p.dim == HK && a.p.v_dim == HV ? launch_one<T, HK, HV, true>(a, many, stream)
                                            : launch_one<T, HK, HV, false>(a, many, stream);
}

template <typename T>
hipError_t launch_list(const KvArgs& a, bool many, hipStream_t stream) {
    return a.p.width == 64    ? launch_width<T, 64, 64>(a, many, stream)
           : a.p.width == 128 ? launch_width<T, 128, 128>(a, many, stream)
           : a.p.width == 192 ? launch_width<T, 192, 128>(a, many, stream)
                              : launch_width<T, 256, 256>(a, many, stream);
}

}  // namespace
}  // namespace mla
