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
// P^T enters in two 16-bit parts, e = hi + lo, off by 2^-17 of it (bf16) or 2^-23 (fp16) at most:
// only the row is rounded to 16 bits.
//
// kv_few_kernel -- a job of at most 16 rows: each of four waves holds all of them and takes every
//   4th unit, straight from memory into the operands' registers; the waves' states meet in LDS at
//   the end.
// kv_many_kernel -- a job of 128 rows (64 above width 128): each of four waves holds 32 (16).  They
//   stage 64 keys (128 at width 64, 32 at 256) together in LDS, in operand order, into one of two
//   buffers: one barrier a stage, and every LDS access is 16 bytes a lane in a row.
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

// The reference maximum sits kHead below the row's when it is set, and is raised again when a
// score passes it by more than kRise: probabilities stay within fp16, and those near the maximum
// clear of its subnormals.
constexpr float kHead = 6.0f, kRise = 14.0f;

// Tables that other kernels wrote are read through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t* table_ptr;
__device__ __forceinline__ table_ptr table(const int32_t* p) {
    return (table_ptr)reinterpret_cast<uintptr_t>(p);
}

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
    const int jobs_f = plan[kKvJobsF], jobs_m = plan[kKvJobsM], parts = plan[kKvParts],
              tag = plan[kKvTag];
    j.session = d[0];
    j.q0 = d[1];
    j.f0 = d[2];
    j.rows = d[3];
    j.u0 = d[4];
    j.u1 = d[5];
    j.ctx = d[6];
    j.part = d[7];
    // no such job; or a plan for other sizes, or a failed one, or not the build that the host knows
    if (index >= (many ? jobs_m : jobs_f) || !kv_plan_fits(a, tag, jobs_f, jobs_m, parts))
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

// Page ids of a unit's two tiles, and their places there.
struct Pages {
    int id[2], in[2];
};

// What both kernels share: T 16-bit type, HD width (head sizes are HD in EXACT instantiations, at
// most HD in the others), CW consecutive columns of V that a lane transposes (a tile of O^T holds
// every CW-th), N tiles of 16 rows a wave.
template <typename T, int HD, bool EXACT, int CW, int N>
struct Attend {
    static constexpr int KS = HD / 32, NT = HD / 16, NC = NT / CW;
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
        : a(a_), job(j), D(EXACT ? HD : a_.p.dim), DV(EXACT ? HD : a_.p.v_dim), lane(lane_),
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
        p.id[0] = ptab[quotient(t, tpp, a.tpp_inverse, p.in[0])];
        // a tile behind the last key is not on a page: the one before it is read again
        const int t1 = min(t + 1, job.pb >> 4);
        p.id[1] = ptab[quotient(t1, tpp, a.tpp_inverse, p.in[1])];
        return p;
    }
    // (Ids were checked by the metadata's build; the bound is for memory's sake.)
    __device__ __forceinline__ long long page_at(int id) const {
        return (long long)min((unsigned)id, (unsigned)a.num_pool_pages - 1) * record;
    }
    __device__ __forceinline__ const uint16_t* keys_at(const Pages& p, int tt) const {
        return keys_of_head + page_at(p.id[tt]) + (long long)p.in[tt] * 16 * D;
    }
    __device__ __forceinline__ const uint16_t* values_at(const Pages& p, int tt) const {
        return values_of_head + page_at(p.id[tt]) + (long long)p.in[tt] * 16 * DV;
    }
    // Key operand of a tile's step s: columns 32s + 8g .. of key n.
    __device__ __forceinline__ u32x4 load_key(const uint16_t* tile, int s) const {
        const int c = 32 * s + 8 * g;
        const u32x4 v = *reinterpret_cast<const u32x4*>(tile + n * D + (EXACT ? c : min(c, D - 8)));
        return EXACT || c < D ? v : u32x4{0, 0, 0, 0};
    }
    // The lane's columns of chunk c of a tile's row 4g + i.
    struct Row {
        uint32_t w[CW / 2];
    };
    __device__ __forceinline__ Row load_value(const uint16_t* tile, int c, int i) const {
        const int col = 16 * CW * c + CW * n;
        const uint16_t* p = tile + (4 * g + i) * DV + (EXACT ? col : min(col, DV - CW));
        Row r;
        if constexpr (CW == 8) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                r.w[k] = EXACT || col < DV ? v[k] : 0;
        } else {
            const u32x2 v = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                r.w[k] = EXACT || col < DV ? v[k] : 0;
        }
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
    // Whether every row of the block sees the unit's keys.
    __device__ __forceinline__ bool all_rows_see(int key0) const {
        return key0 + kKvTile - 1 <= job.pa &&
               (key0 >= job.lo_b || key0 + kKvTile - 1 < a.p.sinks);
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

    // Scores become weights: masks, maximum, exponentials and their sum, in two parts.
    __device__ __forceinline__ void weights(floatx4 (&sc)[N][2], int key0, bool full, V8 (&hi)[N],
                                            V8 (&lw)[N]) {
        float mp[N];
#pragma unroll
        for (int t = 0; t < N; ++t) {
            if (!full)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + 16 * tt + 4 * g + i;
                        if (key > pos[t] || (key < lo[t] && key >= a.p.sinks))
                            sc[t][tt][i] = -INFINITY;
                    }
            mp[t] = -INFINITY;  // of the lane's eight scores (NaN is passed over)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mp[t] = fmaxf(mp[t], sc[t][tt][i]);
            mp[t] *= a.scale_log2;
        }
        bool raise = false;
#pragma unroll
        for (int t = 0; t < N; ++t)
            raise |= mp[t] > m[t] + kRise;
        if (__builtin_amdgcn_ballot_w64(raise)) {
#pragma unroll
            for (int t = 0; t < N; ++t) {
                const float top = rows_max(mp[t]) - kHead;
                const float m_new = top > m[t] + (kRise - kHead) ? top : m[t];
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
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const float ref = m[t] == -INFINITY ? 0.0f : m[t];
            float sum = 0.0f;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(sc[t][tt][i], a.scale_log2, -ref));
                    sum += e;
                    const auto h = static_cast<typename T::scalar>(e);
                    hi[t][4 * tt + i] = h;
                    lw[t][4 * tt + i] = static_cast<typename T::scalar>(e - static_cast<float>(h));
                }
            l[t] += sum;
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

template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    return T::from_float(x) | (uint32_t)T::from_float(y) << 16;
}

template <typename T, int HD, bool EXACT>
__global__ __launch_bounds__(kKvThreads) __attribute__((
    amdgpu_waves_per_eu(HD == 64 ? 4 : HD == 128 ? 3 : 2, 8))) void kv_few_kernel(KvArgs a) {
    constexpr int CW = HD >= 128 ? 8 : 4, PITCH = HD + 4;
    using A = Attend<T, HD, EXACT, CW, 1>;
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
        floatx4 sc[1][2] = {{{0, 0, 0, 0}, {0, 0, 0, 0}}};
#pragma unroll
        for (int st = 0; st < A::KS; ++st)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
                sc[0][tt] = T::mma32(__builtin_bit_cast(V8, k[tt][st]), s.q[0][st], sc[0][tt]);
        load_keys(next);
        const bool full = s.all_rows_see(key0);
        V8 hi[1], lw[1];
        s.weights(sc, key0, full, hi, lw);
        bool bad = false;
        if (!full)
#pragma unroll
            for (int c = 0; c < A::NC; ++c)
                bad |= s.clean(v[c], key0);
#pragma unroll
        for (int c = 0; c < A::NC; ++c)
#pragma unroll
            for (int e = 0; e < CW; ++e) {
                const V8 x = __builtin_bit_cast(V8, A::transposed(v[c], e));
                s.acc[0][c * CW + e] = T::mma32(x, hi[0], s.acc[0][c * CW + e]);
                s.acc[0][c * CW + e] = T::mma32(x, lw[0], s.acc[0][c * CW + e]);
            }
        if (__builtin_amdgcn_ballot_w64(bad))
            s.add_nonfinite(now, key0, hi, lw);
        load_values(next);
        now = next;
        next = s.find_pages(u + 8);
    }

    // ---- the waves' states become rows, or partials ----
    const float l = rows_sum(s.l[0]);
    float* mine = smem[wave];
#pragma unroll
    for (int c = 0; c < A::NC; ++c)
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int e = 0; e < CW; e += 4) {
                const int x = c * CW + e;
                *reinterpret_cast<floatx4*>(mine + s.n * PITCH + s.column(x, y)) =
                    floatx4{s.acc[0][x][y], s.acc[0][x + 1][y], s.acc[0][x + 2][y], s.acc[0][x + 3][y]};
            }
    if (s.g == 0) {
        mine[16 * PITCH + s.n] = s.m[0];
        mine[16 * PITCH + 16 + s.n] = l;
    }
    __syncthreads();
    const int DV = s.DV, per_row = DV / 4;
    for (int e = tid; e < job.rows * per_row; e += kKvThreads) {
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
            const int i = quotient(job.f0 + r, a.p.group, a.group_inverse, in_group);
            const long long row = ((long long)job.q0 + i) * a.p.H + head * a.p.group + in_group;
            const float inv = 1.0f / L;
            *reinterpret_cast<u32x2*>(a.out + row * DV + c) =
                u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
            if (a.lse && c == 0)
                a.lse[row] = (M + __log2f(L)) * kLn2;
        } else {
            const long long row = ((long long)job.part + r) * a.p.kv_heads + head;
            *reinterpret_cast<floatx4*>(a.part_o + row * DV + c) = o;
            if (c == 0) {
                a.part_ml[2 * row] = M;
                a.part_ml[2 * row + 1] = L;
            }
        }
    }
}

template <typename T, int HD, bool EXACT>
__global__ __launch_bounds__(kKvThreads) __attribute__((
    amdgpu_waves_per_eu(2, 8))) void kv_many_kernel(KvArgs a) {
    constexpr int N = HD == 256 ? 1 : 2, CW = 4;
    constexpr int SU = HD == 64 ? 4 : HD == 128 ? 2 : 1;  // units of a stage
    using A = Attend<T, HD, EXACT, CW, N>;
    using V8 = typename T::vec8;
    // a stage in operand order, 1 KB each: keys [unit][tile][step], values [unit][tile of O^T]
    constexpr int KW = SU * 2 * A::KS * 512, STAGE = KW + SU * A::NT * 512;
    __shared__ __attribute__((aligned(16))) uint16_t smem[2][STAGE];
    __shared__ int marks[3][SU];  // units whose non-finite values were taken out
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int index = (int)(blockIdx.x / (unsigned)a.p.kv_heads);
    const int head = (int)(blockIdx.x - (unsigned)index * a.p.kv_heads);
    Job job;
    if (!take_job(a, true, index, job))
        return;
    const int row0 = wave * 16 * N;
    A s(a, job, tid & 63, head, row0);

    // positions of the wave's first and last row (none: it takes no units)
    int r;
    const int w_last = min(job.rows, row0 + 16 * N) - 1;
    const int wa = job.ctx + quotient(job.f0 + min(row0, job.rows - 1), a.p.group, a.group_inverse, r);
    const int wb = w_last < row0 ? -1 : job.ctx + quotient(job.f0 + w_last, a.p.group, a.group_inverse, r);
    const int lo_wa = wa >= a.p.window ? wa - a.p.window + 1 : 0;
    const int lo_wb = wb >= a.p.window ? wb - a.p.window + 1 : 0;

    // ---- what the wave stages: a quarter of the stage, all of it of one unit ----
    const int su = wave * SU / 4;                 // the unit
    const int o0 = wave * 4 % (2 * A::KS);        // its first of four key operands there
    const int vc = wave % A::NC;                  // its chunk of the values
    u32x4 k[4];
    typename A::Row v[8];
    auto load = [&](const Pages& p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int o = o0 + i;
            k[i] = s.load_key(s.keys_at(p, o / A::KS), o % A::KS);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = s.load_value(s.values_at(p, i >> 2), vc, i & 3);
    };
    const int stages = (job.u1 - job.u0 + SU - 1) / SU;
    if (tid < 3 * SU)
        marks[tid / SU][tid % SU] = 0;
    __syncthreads();
    Pages pages = s.find_pages(job.u0 + su);
    load(pages);
    for (int st = 0; st < stages; ++st) {
        uint16_t* const buf = smem[st & 1];
        const int u0 = job.u0 + st * SU, mine = first_key(job, min(u0 + su, job.u1 - 1));
        if (!s.all_rows_see(mine)) {
            const bool bad = s.clean(v, mine);
            if (__builtin_amdgcn_ballot_w64(bad) && s.lane == 0)
                marks[st % 3][su] = 1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x4*>(buf + (su * 2 * A::KS + o0 + i) * 512 + s.lane * 8) = k[i];
#pragma unroll
        for (int e = 0; e < CW; ++e)
            *reinterpret_cast<u32x4*>(buf + KW + (su * A::NT + vc * CW + e) * 512 + s.lane * 8) =
                A::transposed(v, e);
        pages = s.find_pages(u0 + SU + su);
        load(pages);  // (the last one once more, at the end)
        // The other buffer is free: every wave that passed the barrier before this one has finished
        // with it.  Likewise the marks: stage st + 2's, last read in stage st - 1, are cleared behind
        // this barrier and set again behind the next.
        __syncthreads();
        if (tid < SU)
            marks[(st + 2) % 3][tid] = 0;
#pragma unroll 1
        for (int x = 0; x < SU; ++x) {
            if (u0 + x >= job.u1)
                break;
            const int key0 = first_key(job, u0 + x);
            if (key0 > wb || (key0 + kKvTile <= lo_wa && key0 >= a.p.sinks))
                continue;
            const uint16_t* const kb = buf + x * 2 * A::KS * 512 + s.lane * 8;
            const uint16_t* const vb = buf + KW + x * A::NT * 512 + s.lane * 8;
            floatx4 sc[N][2];
#pragma unroll
            for (int t = 0; t < N; ++t)
                sc[t][0] = sc[t][1] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < A::KS; ++i)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const V8 y = *reinterpret_cast<const V8*>(kb + (tt * A::KS + i) * 512);
#pragma unroll
                    for (int t = 0; t < N; ++t)
                        sc[t][tt] = T::mma32(y, s.q[t][i], sc[t][tt]);
                }
            const bool full = key0 + kKvTile - 1 <= wa &&
                              (key0 >= lo_wb || key0 + kKvTile - 1 < a.p.sinks);
            V8 hi[N], lw[N];
            s.weights(sc, key0, full, hi, lw);
#pragma unroll
            for (int i = 0; i < A::NT; ++i) {
                const V8 y = *reinterpret_cast<const V8*>(vb + i * 512);
#pragma unroll
                for (int t = 0; t < N; ++t) {
                    s.acc[t][i] = T::mma32(y, hi[t], s.acc[t][i]);
                    s.acc[t][i] = T::mma32(y, lw[t], s.acc[t][i]);
                }
            }
            if (marks[st % 3][x])
                s.add_nonfinite(s.find_pages(u0 + x), key0, hi, lw);
        }
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
        for (int x = 0; x < A::NT; x += CW)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int col = s.column(x, y);
                if (!EXACT && col >= s.DV)
                    continue;
                const floatx4 o = {s.acc[t][x][y], s.acc[t][x + 1][y], s.acc[t][x + 2][y],
                                   s.acc[t][x + 3][y]};
                if (job.part < 0)
                    *reinterpret_cast<u32x2*>(a.out + at * s.DV + col) =
                        u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
                else
                    *reinterpret_cast<floatx4*>(a.part_o + at * s.DV + col) = o;
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

template <typename T, int HD, bool EXACT>
hipError_t launch_one(const KvArgs& a, bool many, hipStream_t stream) {
    if (many)
        hipLaunchKernelGGL((kv_many_kernel<T, HD, EXACT>), dim3((unsigned)(a.jobs_m * a.p.kv_heads)),
                           dim3(kKvThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((kv_few_kernel<T, HD, EXACT>), dim3((unsigned)(a.jobs_f * a.p.kv_heads)),
                           dim3(kKvThreads), 0, stream, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_list(const KvArgs& a, bool many, hipStream_t stream) {
    const int w = a.p.width;
    const bool exact = a.p.dim == w && a.p.v_dim == w;
    if (w == 64)
        return exact ? launch_one<T, 64, true>(a, many, stream) : launch_one<T, 64, false>(a, many, stream);
    if (w == 128)
        return exact ? launch_one<T, 128, true>(a, many, stream) : launch_one<T, 128, false>(a, many, stream);
    return exact ? launch_one<T, 256, true>(a, many, stream) : launch_one<T, 256, false>(a, many, stream);
}

}  // namespace
}  // namespace mla
