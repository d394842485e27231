// Attention of a batch's query rows over the paged latent cache by a plan's jobs, gfx950: the
// kernel of both lists and both cache formats (the units latent_attend_*.hip instantiate it).
//
// For a (query, head) row with query (q, qr) and keys i = (latent c_i, rope key k_i) that it sees
//     s_i = (q . c_i + qr . k_i) scale,   o = sum_i softmax(s)_i c_i,   lse = ln sum_i exp(s_i)
// as the framework's other attention kernels (src/infer/inference.cpp:116-153 in the reference,
// causal rows src/model/ops.cpp:109-142).
//
// latent_attend_kernel -- a workgroup takes a job: rows of a segment over a range of its keys, 32
//   keys (a unit: two 16-token tiles, which may lie on different pages) at a time, a wave 16 rows.
//   List K, 16 rows: each of four waves holds all of them and takes every 4th unit, whose
//   latents pass through a slot of its own; the waves' states meet in LDS at the end.  List R, 128
//   rows: each of eight waves holds 16, they stage a unit together into one of two buffers (one
//   barrier a unit), and no state is exchanged: a key is fetched and converted once for 128 rows.
//   A unit goes from memory to registers while the unit before it is computed, and from there to
//   LDS as 16-bit words in MFMA-operand order (8-bit latents: v_cvt_scalef32_pk_*, exact, see
//   mla_q8.hpp), so that both formats share everything behind it:
//     S^T = K . Q^T     v_mfma_f32_16x16x32, Q^T in registers for the whole job; list K's keys
//                       come from the registers that they were loaded into, list R's from LDS
//     online softmax    log2 domain in 32 bits, the reference maximum raised lazily
//     O^T += C^T . P^T  C^T by transpose reads (ds_read_b64_tr_b16); P^T in two 16-bit parts
//                       (see finish_unit)
//
// What bounds it, and what was measured (MI355X, kernels in a trace; a large copy reaches 4.8 TB/s
// there, a large bf16 product 1,350 TFLOP/s; operations of the formula, the second part of P^T not
// counted):
//   kv 128, 8 heads, 64 sessions of 128 .. 4,096 tokens in 8 bits (23.7 MB): 9.4 us: the launch,
//     three dependent trips to memory (job, page ids, unit), the chain of the 3 or 4 units that a
//     wave gets, the waves' merge.  Latency: half of the waves' time is waiting for memory.  10.6 us
//     for 64 sessions behind one 4,000-token prefix, 16 bits.
//   kv 128, chunks of 509 rows: 30 us, 0.29 PFLOP/s.  List K fetches and converts every key for 16
//     rows: 191 vector and 122 scalar instructions for a unit's 26 MFMAs.  37 % of the waves' time
//     waits for issue, 29 % for memory.
//   kv 512, 128 heads, list R: 64 decode rows over 534,000 8-bit tokens (149 GFLOP) 232-238 us with
//     the merge, 0.63 PFLOP/s; 48 sessions behind an 8,191-token prefix, 16 bits (117 GFLOP),
//     192-195 us, 0.60.  Over the whole dispatch the matrix cores are busy 42 and 38 % of the time,
//     LDS 36 and 33 % (eight waves read each unit twice, for the scores and for the weighted sum):
//     neither is full, a unit's phases follow one another in a wave, and with two waves a SIMD
//     little else is there to run.  The longest job is 13-17 % above the mean.  32 rows a wave
//     would halve the LDS reads, and take 256 registers for O^T alone: at one wave a SIMD it spilled
//     210 registers (940 us).
//   With P^T in one part (in error, see finish_unit): 8.2 us, 10.2, 26.7, 202 and 168.
// Registers: of the instantiations for one shape, those over the 16-bit cache spill 3 to 35 (list K
// at kv 512 the most); of the others, 8-bit list K 97-104 above kv 256 and 16 at kv 256, the rest
// above kv 256 12 to 28.
// A key past a row's position adds nothing to the row, whatever it holds: its rope key only enters
// the score, which is replaced, and a non-finite latent is staged as zero with the key marked, and
// makes the scores of the rows that see it NaN.  (Where every row of a job sees the key, such a
// latent spreads to them by itself, and is not looked for.)
#pragma once

#include "mla_latent.hpp"
#include "mla_q8.hpp"

#include <cmath>
#include <type_traits>

namespace mla {
namespace {

// Rows of odd 256-byte sub-chunks of a latent block sit at slot row ^ kRot in LDS, so that the
// transpose reads of a sub-chunk pair fall in disjoint banks.
constexpr int kRot = 12;
// The reference maximum sits kHead below the row's when it is set, and is raised again when a
// score passes it by more than kRise: probabilities stay within fp16, and those near the maximum
// clear of its subnormals.
constexpr float kHead = 6.0f, kRise = 14.0f;

// Tables that other kernels wrote are read through the scalar cache: a vector load of a page id
// would be waited for together with the unit that was just sent for.
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

__device__ __forceinline__ u32x2 read_tr16(const uint16_t* p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    const auto v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (s4 __attribute__((address_space(3)))*)((__attribute__((address_space(3))) char*)p));
    return __builtin_bit_cast(u32x2, v);
}

// The 16-bit words of v whose exponent is all ones become 0; true if there was one.
template <typename T>
__device__ __forceinline__ bool drop_nonfinite16(u32x4& v) {
    constexpr uint32_t e = T::exp_mask, both = e | e << 16;
    constexpr uint32_t step = (e & -e) | (e & -e) << 16;  // the exponent's lowest bit
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        any |= ((v[i] & both) + step) & 0x80008000u;
    if (!any)
        return false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((v[i] & e) == e)
            v[i] &= 0xffff0000u;
        if ((v[i] >> 16 & e) == e)
            v[i] &= 0x0000ffffu;
    }
    return true;
}
// The NaN bytes of v become 0; true if there was one.
__device__ __forceinline__ bool drop_nan8(u32x4& v) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        any |= q8_nan_bits(v[i]);
    if (!any)
        return false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] &= ~((q8_nan_bits(v[i]) >> 7) * 0xffu);
    return true;
}

// T: 16-bit type of the queries, rope keys, 16-bit latents and rows; Q8: 8-bit latents; KSM: latent
// k-steps (kv_rank / 32 <= KSM); ROWS: list R; RP_: the rope columns of an instantiation for one
// shape (kv_rank = 32 KSM, rope_dim = RP_), -1 for any.
template <typename T, bool Q8, int KSM, bool ROWS, int RP_ = -1>
__global__ __launch_bounds__(ROWS ? kThreadsR : kThreadsK) __attribute__((
    amdgpu_waves_per_eu(KSM >= 16 && !ROWS ? 1 : RP_ == 16 ? 4 : 2, 8))) void latent_attend_kernel(LatentArgs a) {
    constexpr int NW = (ROWS ? kThreadsR : kThreadsK) / 64;  // waves
    constexpr bool ONE = RP_ >= 0;
    constexpr int RSM = ONE ? (RP_ + 31) / 32 : 2;      // rope k-steps (rope_dim <= 64)
    constexpr int RTM = 2 * KSM;                        // 16-row tiles of O^T
    // 32-key units that are fetched and staged together: two on list R where LDS has room, which
    // halves the barriers and what else a unit costs besides its products
    constexpr int SUB = ROWS && KSM <= 8 ? 2 : 1;
    constexpr int NT = 2 * SUB, KEYS = 32 * SUB;
    // Words of a unit in LDS: 32 keys' latents, on list R (whose waves take each other's keys) their
    // rope keys too, on list K (see the end) room for 16 rows of O^T in fp32 and their m and l.
    constexpr int SLOT = ROWS ? 32 * 32 * (KSM + RSM) : 2 * (16 * (32 * KSM + 4) + 32);
    constexpr int UPT = Q8 ? (KSM + 1) / 2 : KSM;       // 16-byte loads of a lane per tile
    constexpr int NL = ROWS ? (NT * UPT + NW - 1) / NW : NT * UPT;
    constexpr int RCS = ONE ? RP_ / 8 : 8;              // 8-column rope chunks of a tile, at most
    constexpr int NR = ROWS ? (NT * RCS + 4 * NW - 1) / (4 * NW) : 2 * RSM;  // rope loads of a lane
    constexpr int SLOTS = ROWS ? 2 * SUB : 4;
    // Q^T k-steps that stay in LDS, lane by lane, where the registers would spill (a reload waits
    // for every load in flight): at kv 512 O^T takes 128 of a wave's 256 registers, Q^T 72.
    constexpr int AHEAD = ONE && KSM >= 16 ? 2 : 1;  // steps that LDS reads run ahead of their use
    constexpr int QL = KSM >= 16 && ROWS ? (ONE ? (Q8 ? 8 : 10) : 8) : 0;
    using V8 = typename T::vec8;
    __shared__ __attribute__((aligned(16))) uint16_t smem[SLOTS][SLOT];
    __shared__ __attribute__((aligned(16))) uint16_t q_lds[QL > 0 ? NW * QL * 512 : 8];
    __shared__ uint32_t marks[3 * SUB];  // list R: keys of a unit with a non-finite latent

    const table_ptr plan = table(a.plan);
    const table_ptr d = plan + (ROWS ? a.p.jobs_r_at : a.p.jobs_k_at) + (long long)blockIdx.x * kJobInts;
    const int jobs_k = plan[kPlanJobsK], jobs_r = plan[kPlanJobsR], parts = plan[kPlanParts],
              tag = plan[kPlanTag];
    const int seg = d[0], f0 = d[1], n_rows = d[2], rb = d[3], key0 = d[4], key_end = d[5],
              ctx = d[6], part = d[7];
    // no such job; or a plan for other sizes, or a failed one, or not the build that the host knows
    if ((int)blockIdx.x >= (ROWS ? jobs_r : jobs_k) || !plan_fits(a, tag, jobs_k, jobs_r, parts))
        return;

    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int H = a.H, PS = a.page_size;
    const int KV = ONE ? 32 * KSM : a.kv_rank, RP = ONE ? RP_ : a.rope_dim;
    const int ks = KV >> 5, rs = (RP + 31) >> 5, tpp = PS >> 4;
    const long long rec = Q8 ? q8_page_bytes(PS, KV, RP) : 2LL * PS * (KV + RP);
    const table_ptr ptab = table(seg >= 0 ? a.page_table + (long long)seg * a.max_pages
                                          : a.prefix_page_ids + table(a.cu_prefix_pages)[~seg]);
    const int n_units = key_end > key0 && a.num_pool_pages > 0 ? (key_end - key0 + KEYS - 1) / KEYS : 0;
    const int row0 = ROWS ? 16 * wave : 0;  // the wave's first row of the block

    // ---- Q^T operands: row n, latent columns 32j + 8g .., then the rope key's; the rows' limits ----
    V8 qv[KSM + RSM - QL];
    uint16_t* const my_q = q_lds + wave * QL * 512 + lane * 8;
    const bool causal_seg = a.causal && seg >= 0;
    int lim, lim_wave = -1, lim_all = key_end - 1;  // lane's row n sees keys [0, lim] of the segment
    // The last key that every row of the block sees: from there on a non-finite latent has to be
    // kept from the rows before it.
    auto token_of = [&](int row) {  // row / H
        int r;
        return quotient(row, H, a.h_inverse, r);
    };
    const int seen_by_all = causal_seg ? ctx + token_of(rb) : 0x7fffffff;
    {
        const int r = min(row0 + n, n_rows - 1);  // rows past the block repeat its last
        const long long fr = (long long)f0 + r;
        lim = causal_seg ? ctx + token_of(rb + r) : key_end - 1;
        const uint16_t* ql = a.q_latent + fr * KV + 8 * g;
        const uint16_t* qr = a.q_rope + fr * RP;
#pragma unroll
        for (int j = 0; j < KSM + RSM; ++j) {
            V8 v = {};
            if (j < KSM) {
                if (j < ks)
                    v = *reinterpret_cast<const V8*>(ql + 32 * j);
            } else if (j - KSM < rs) {
                const int c = 32 * (j - KSM) + 8 * g;
                v = *reinterpret_cast<const V8*>(qr + min(c, RP - 8));
                v = c < RP ? v : V8{};
            }
            if (j < KSM + RSM - QL)
                qv[j] = v;
            else
                *reinterpret_cast<V8*>(my_q + (j - (KSM + RSM - QL)) * 512) = v;
        }
        // the last key that any of the wave's rows sees (-1: it has no rows), and that all see
        const int last = min(n_rows, row0 + 16) - 1;
        if (last >= row0)
            lim_wave = causal_seg ? ctx + token_of(rb + last) : key_end - 1;
        if (causal_seg)
            lim_all = ctx + token_of(rb + row0);
    }
    auto q_operand = [&](int j) {
        return j < KSM + RSM - QL
                   ? qv[j]
                   : *reinterpret_cast<const V8*>(my_q + (j - (KSM + RSM - QL)) * 512);
    };

    // ---- a unit's way into LDS ----
    const int s_lane = g * 128 + (n ^ ((g & 1) * kRot)) * 8;
    // Nothing is done to what was loaded before it is staged (taking a scale's byte out of its word
    // would wait for the load): scales stay as they lie in memory, the words of a tile's token
    // (WORDS), or those of a load's two k-steps in one word or in two.
    constexpr bool WORDS = Q8 && ONE && !ROWS;
    struct Loaded {
        u32x4 st[NL], sr[NR];
        uint32_t sk[WORDS ? KSM / 2 : Q8 ? (ONE ? NL : 2 * NL) : 1];
    };
    auto scale_of = [](const Loaded& x, int i, int half) {  // of k-step `half` of load i
        if constexpr (WORDS) {
            const int b = 2 * (i % UPT) + half;
            return q8_scale(x.sk[i / UPT * (KSM / 4) + b / 4] >> (8 * (b % 4)) & 0xff);
        } else if constexpr (ONE) {
            return q8_scale(half ? x.sk[i] >> 8 : x.sk[i] & 0xff);
        } else {
            return q8_scale(x.sk[2 * i + half]);
        }
    };
    const int upt = Q8 ? (ks + 1) >> 1 : ks;
    const int lat_tile = (Q8 ? 16 : 32) * KV, key_tile = 32 * RP, sc_tile = 16 * ks;  // bytes
    const long long key_at = (long long)PS * (Q8 ? 1 : 2) * KV, sc_at = (long long)PS * (KV + 2 * RP);
    // This lane's rope chunks: tile, and bytes from the unit's first keys (-1: none).  List K: the
    // operands of (tile, k-step) i; lanes past the rope columns take a valid chunk (their Q^T is 0).
    const int rcs = RP >> 3;
    int rope_tt[NR], rope_in[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        if constexpr (ROWS) {
            const int c = (tid >> 4) + 4 * NW * i;
            const int tt = ONE ? c / (RCS > 0 ? RCS : 1) : (rcs > 0 ? c / rcs : 0);
            const bool some = tt < NT && rcs > 0;
            rope_tt[i] = some ? tt : 0;
            rope_in[i] = some ? tt * key_tile + (c - tt * rcs) * 256 + n * 16 : -1;
        } else {
            const int tt = i / RSM, j = i % RSM;
            rope_tt[i] = tt;
            rope_in[i] = tt * key_tile + (32 * j + 8 * g < RP ? 4 * j + g : 0) * 256 + n * 16;
        }
    }
    // A tile's page (number in the list) and place there.
    auto page_of = [&](int t, int& in) { return quotient(t, tpp, a.tpp_inverse, in); };
    const int last_tile = (key_end - 1) >> 4;
    const bool one_page = PS % KEYS == 0;  // a unit lies on one page
    // Page ids of the unit at tile t, and the places of its tiles there.  Tiles past the keys take
    // the last one's: they are read, so that no load hangs on a branch (the compiler would load
    // into other registers, and wait to move), and dropped when they are staged.
    struct Pages {
        int id[NT], in[NT];
    };
    auto find_pages = [&](int t) {
        Pages p;
        if (one_page) {
            const int id = ptab[page_of(min(t, last_tile), p.in[0])];
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                p.id[k] = id;
                p.in[k] = p.in[0] + (t + k <= last_tile ? k : 0);
            }
        } else {
#pragma unroll
            for (int k = 0; k < NT; ++k)
                p.id[k] = ptab[page_of(min(t + k, last_tile), p.in[k])];
        }
        return p;
    };
    // (Ids were checked by the builds of the metadata and the plan; the bound is for memory's sake.)
    auto page_base = [&](int id) {
        return a.pages + (long long)min((unsigned)id, (unsigned)a.num_pool_pages - 1) * rec;
    };
    auto load_unit = [&](Loaded& x, const Pages& p) {
        const uint8_t* base[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
            base[t] = one_page && t > 0 ? base[0] : page_base(p.id[t]);
        auto base_of = [&](int tt, int& in) {
            const uint8_t* b = base[0];
            in = p.in[0];
#pragma unroll
            for (int t = 1; t < NT; ++t) {
                b = tt == t ? base[t] : b;
                in = tt == t ? p.in[t] : in;
            }
            return b;
        };
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            // (indexes past the unit's loads, in shapes that do not fill them, read its first again)
            int u = ROWS ? wave + NW * i : i, tt = u / UPT, k = u % UPT;
            if (!ONE || ROWS) {
                const bool some = u < NT * UPT && k < upt;
                tt = some ? tt : 0;
                k = some ? k : 0;
            }
            int in;
            const uint8_t* b = base_of(tt, in);
            if constexpr (Q8) {
                const uint8_t* lat = b + in * lat_tile + k * 1024;
                const uint8_t* sc = b + sc_at + in * sc_tile + 2 * k + n * ks;
                if constexpr (ONE) {
                    x.st[i] = *reinterpret_cast<const u32x4*>(lat + lane * 16);
                    if constexpr (!WORDS)
                        x.sk[i] = *reinterpret_cast<const uint16_t*>(sc);
                } else {
                    // an odd last k-step has 8 bytes a lane, and one scale: read twice
                    const bool pair = 2 * k + 1 < ks;
                    const u32x2 lo = *reinterpret_cast<const u32x2*>(lat + lane * (pair ? 16 : 8));
                    const u32x2 hi =
                        *reinterpret_cast<const u32x2*>(lat + (pair ? lane * 16 + 8 : lane * 8));
                    x.st[i] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                    x.sk[2 * i] = sc[0];
                    x.sk[2 * i + 1] = sc[pair ? 1 : 0];
                }
            } else {
                x.st[i] = *reinterpret_cast<const u32x4*>(b + in * lat_tile + k * 1024 + lane * 16);
            }
        }
        if constexpr (WORDS)
#pragma unroll
            for (int i = 0; i < KSM / 2; ++i) {
                int in;
                const uint8_t* b = base_of(i / (KSM / 4), in);
                x.sk[i] = reinterpret_cast<const uint32_t*>(b + sc_at + in * sc_tile +
                                                            n * ks)[i % (KSM / 4)];
            }
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            int in;
            const uint8_t* b = base_of(rope_tt[i], in);
            if (ROWS || RP > 0)
                x.sr[i] = *reinterpret_cast<const u32x4*>(b + (RP > 0 ? key_at : 0) +
                                                          (in - rope_tt[i]) * key_tile +
                                                          max(rope_in[i], rope_tt[i] * key_tile));
        }
    };
    // The keys of 32-key part `sub` of the unit at tile t0 that exist.
    auto keys_of = [&](int t0, int sub) {
        const int valid = key_end - 16 * t0 - 32 * sub;
        return valid >= 32 ? 0xffffffffu : valid <= 0 ? 0u : (1u << valid) - 1u;
    };
    // Keys of the loaded unit outside `ok` become 0 (their slots, scales included, may hold
    // anything).  look: non-finite latents become 0 as well, and the wave's `mark` names their keys.
    auto clean_unit = [&](Loaded& x, const uint32_t (&ok)[SUB], uint32_t (&mark)[SUB], bool look) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int u = ROWS ? wave + NW * i : i, tt = u / UPT;
            const uint32_t of = SUB == 1 || tt < 2 ? ok[0] : ok[SUB - 1];
            const uint32_t keep = -(of >> (16 * (tt & 1) + n) & 1);
            x.st[i] &= keep;
            if constexpr (Q8 && !ONE)
                x.sk[2 * i + 1] &= keep;
            if constexpr (Q8 && !WORDS)
                x.sk[ONE ? i : 2 * i] &= keep;
            if (look) {
                bool bad;
                if constexpr (Q8)
                    bad = drop_nan8(x.st[i]);
                else
                    bad = drop_nonfinite16<T>(x.st[i]);
                const uint64_t b = __builtin_amdgcn_ballot_w64(bad);
                const uint32_t m = (uint32_t)((b | b >> 16 | b >> 32 | b >> 48) & 0xffff)
                                   << (16 * (tt & 1));
                if (u < NT * UPT && u % UPT < upt) {
                    if (SUB == 1 || tt < 2)
                        mark[0] |= m;
                    else
                        mark[SUB - 1] |= m;
                }
            }
        }
        if constexpr (WORDS)
#pragma unroll
            for (int i = 0; i < KSM / 2; ++i)
                x.sk[i] &= -(ok[0] >> (16 * (i / (KSM / 4)) + n) & 1);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int tt = rope_tt[i];
            const uint32_t of = SUB == 1 || tt < 2 ? ok[0] : ok[SUB - 1];
            x.sr[i] &= -(of >> (16 * (tt & 1) + n) & 1);
        }
    };
    // List R: writes the loaded unit to `sp` and behind.
    auto stage_unit = [&](const Loaded& x, uint16_t* sp) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int u = wave + NW * i, tt = u / UPT, k = u % UPT;
            if (u >= NT * UPT || k >= upt)
                continue;
            uint16_t* dst = sp + (tt >> 1) * SLOT + (tt & 1) * 16 * KV + s_lane;
            const u32x4 v = x.st[i];
            if constexpr (Q8) {
                *reinterpret_cast<u32x4*>(dst + 2 * k * 512) =
                    q8_decode8<T>(v[0], v[1], scale_of(x, i, 0));
                if (2 * k + 1 < ks)
                    *reinterpret_cast<u32x4*>(dst + (2 * k + 1) * 512) =
                        q8_decode8<T>(v[2], v[3], scale_of(x, i, 1));
            } else {
                *reinterpret_cast<u32x4*>(dst + k * 512) = v;
            }
        }
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (rope_in[i] >= 0) {
                const int tt = rope_tt[i];
                // (a tile's key rows take as many bytes here as in the record)
                *reinterpret_cast<u32x4*>(sp + (tt >> 1) * SLOT + 32 * KV +
                                          (rope_in[i] - (tt >> 1) * 2 * key_tile) / 2) = x.sr[i];
            }
    };
    // List K: a wave loads its units in the order of the score product's operands, and so takes
    // the scores from its registers; the latents go to `sp` for the second product.
    auto stage_scores = [&](Loaded& x, uint16_t* sp, floatx4 (&sc)[2]) {
        if constexpr (WORDS)
#pragma unroll
            for (int i = 0; i < KSM / 2; ++i)
                asm volatile("" : "+v"(x.sk[i]));  // (bytes are taken from here on)
        auto step = [&](int tt, int j, u32x4 v) {
            sc[tt] = T::mma32(__builtin_bit_cast(V8, v), qv[j], sc[tt]);
            *reinterpret_cast<u32x4*>(sp + tt * 16 * KV + j * 512 + s_lane) = v;
        };
#pragma unroll
        for (int k = 0; k < UPT; ++k)
            if (k < upt)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const int i = tt * UPT + k;
                    const u32x4 v = x.st[i];
                    if constexpr (Q8) {
                        step(tt, 2 * k, q8_decode8<T>(v[0], v[1], scale_of(x, i, 0)));
                        if (2 * k + 1 < ks)
                            step(tt, 2 * k + 1 < KSM ? 2 * k + 1 : 0,
                                 q8_decode8<T>(v[2], v[3], scale_of(x, i, 1)));
                    } else {
                        step(tt, k, v);
                    }
                }
#pragma unroll
        for (int j = 0; j < RSM; ++j)
            if (j < rs)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
                    sc[tt] = T::mma32(__builtin_bit_cast(V8, x.sr[tt * RSM + j]), qv[KSM + j], sc[tt]);
    };

    const int tr_par = (n & 3) >> 1;
    const int tr_lane = tr_par * 128 + ((4 * g + (n >> 2)) ^ (tr_par * kRot)) * 8 + 4 * (n & 1);
    int rope_off[RSM];  // lanes past the rope columns read a valid chunk (their Q^T is zero)
#pragma unroll
    for (int j = 0; j < RSM; ++j)
        rope_off[j] = (32 * j + 8 * g < RP ? 4 * j + g : 0) * 128 + n * 8;

    float m_run = -INFINITY, l_run = 0.0f;
    floatx4 acc[RTM];
#pragma unroll
    for (int rt = 0; rt < RTM; ++rt)
        acc[rt] = floatx4{0, 0, 0, 0};

    // ---- list R: scores of the unit at `sp` ----
    auto take_scores = [&](const uint16_t* sp, floatx4 (&sc)[2]) {
        // One k-step's operands are read while the step before it multiplies; the scheduler is held
        // to that (it would read all of them ahead, and spill).
        auto k_operand = [&](int tt, int j) {
            return j < KSM ? *reinterpret_cast<const V8*>(sp + tt * 16 * KV + j * 512 + s_lane)
                           : *reinterpret_cast<const V8*>(sp + 32 * KV + tt * 16 * RP +
                                                          rope_off[j - KSM]);
        };
        if constexpr (ONE) {
            // Step j's operands are read AHEAD steps before (an LDS read takes about as long as
            // that many steps' products); the first of the second product before the softmax.
            V8 ring[AHEAD][2], q_ring[AHEAD];
#pragma unroll
            for (int j = 0; j < KSM + RSM + AHEAD; ++j) {
                if (j >= AHEAD) {
                    const int i = j - AHEAD;
                    const V8 q_now = i < KSM + RSM - QL ? qv[i < KSM + RSM - QL ? i : 0] : q_ring[i % AHEAD];
                    sc[0] = T::mma32(ring[i % AHEAD][0], q_now, sc[0]);
                    sc[1] = T::mma32(ring[i % AHEAD][1], q_now, sc[1]);
                }
                if (j < KSM + RSM) {
                    ring[j % AHEAD][0] = k_operand(0, j);
                    ring[j % AHEAD][1] = k_operand(1, j);
                    if (j >= KSM + RSM - QL)
                        q_ring[j % AHEAD] = q_operand(j);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            V8 next[2] = {k_operand(0, 0), k_operand(1, 0)};
#pragma unroll
            for (int j = 0; j < KSM + RSM; ++j)
                if (j < KSM ? j < ks : j - KSM < rs) {
                    const V8 now[2] = {next[0], next[1]}, q_now = q_operand(j);
                    const int after = j + 1 < ks ? j + 1 : (j < KSM ? KSM : j + 1);
                    if (after < KSM + rs) {
                        next[0] = k_operand(0, after);
                        next[1] = k_operand(1, after);
                    }
                    sc[0] = T::mma32(now[0], q_now, sc[0]);
                    sc[1] = T::mma32(now[1], q_now, sc[1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    };
    // ---- softmax and product of the unit at `sp`, whose first tile is t0; `ok`: keys of the unit
    // that exist, `mark`: those with a non-finite latent ----
    auto finish_unit = [&](floatx4 (&sc)[2], const uint16_t* sp, int t0, uint32_t ok, uint32_t mark) {
        auto c_operand = [&](int rt) {  // latent columns 16rt.. of the unit's 32 keys
            const int blk = ((rt >> 1) * 4 + 2 * (rt & 1)) * 128;
            const u32x2 lo = read_tr16(sp + blk + tr_lane);
            const u32x2 hi = read_tr16(sp + 16 * KV + blk + tr_lane);
            return __builtin_bit_cast(V8, u32x4{lo[0], lo[1], hi[0], hi[1]});
        };
        V8 cring[AHEAD][2];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (2 * k < 2 * ks) {
                cring[k][0] = c_operand(2 * k);
                cring[k][1] = c_operand(2 * k + 1);
            }

        float mp = -INFINITY;  // of the lane's eight scores (NaN is passed over)
        auto take_max = [&]() {
            mp = -INFINITY;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mp = fmaxf(mp, sc[tt][i]);
        };
        take_max();
        if constexpr (!Q8) {
            // An infinite latent that every row sees has not been looked for, and a score of -inf
            // would give it the weight 0: such keys are marked now.  (NaN scores need no mark.)
            float mn = INFINITY;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mn = fminf(mn, sc[tt][i]);
            if (__builtin_amdgcn_ballot_w64(mp == INFINITY || mn == -INFINITY)) {
#pragma unroll 1
                for (int j = 0; j < 2 * ks; ++j) {
                    const int tt = j >= ks;
                    u32x4 v = *reinterpret_cast<const u32x4*>(sp + j * 512 + s_lane);
                    const uint64_t b = __builtin_amdgcn_ballot_w64(drop_nonfinite16<T>(v));
                    mark |= (uint32_t)((b | b >> 16 | b >> 32 | b >> 48) & 0xffff) << (16 * tt);
                }
            }
        }
        // Units that some row does not see in full: their scores are replaced.
        if (ok != 0xffffffffu || mark != 0 || 16 * t0 + 31 > lim_all) {
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = 16 * tt + 4 * g + i;
                    if (mark >> key & 1)
                        sc[tt][i] = NAN;
                    if (!(ok >> key & 1) || 16 * t0 + key > lim)
                        sc[tt][i] = -INFINITY;
                }
            take_max();
        }
        mp *= a.scale_log2;
        if (__builtin_amdgcn_ballot_w64(mp > m_run + kRise)) {
            const float m_new = fmaxf(m_run, rows_max(mp) - kHead);
            const bool had = m_run != -INFINITY;  // the row has accumulated state
            if (__builtin_amdgcn_ballot_w64(had && m_new > m_run)) {
                const float alpha = had ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
                l_run *= alpha;
#pragma unroll
                for (int rt = 0; rt < RTM; ++rt)
                    acc[rt] *= alpha;
            }
            m_run = m_new;
        }
        const float m_ref = m_run == -INFINITY ? 0.0f : m_run;
        // A weight enters the product as two parts of the 16-bit type, e = hi + lo, off by 2^-17 of
        // it (bf16), or 2^-23 of it or 2^-25 (fp16; a row's largest is 2^kHead at least, so that a
        // row made of weights 17 nats below a token with a latent of zero is off by 1 %): as one
        // part it would be off by up to 2^-8 or 2^-11, all weights of keys of one score the same
        // way, while the mass sums them in 32 bits.
        float psum = 0.0f;
        V8 pb, pl;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(sc[tt][i], a.scale_log2, -m_ref));
                psum += e;
                const auto hi = static_cast<typename T::scalar>(e);
                pb[4 * tt + i] = hi;
                pl[4 * tt + i] = static_cast<typename T::scalar>(e - static_cast<float>(hi));
            }
        l_run += psum;
#pragma unroll
        for (int k = 0; k < KSM; ++k)
            if (k < ks) {
                acc[2 * k] = T::mma32(cring[k % AHEAD][0], pb, acc[2 * k]);
                acc[2 * k + 1] = T::mma32(cring[k % AHEAD][1], pb, acc[2 * k + 1]);
                acc[2 * k] = T::mma32(cring[k % AHEAD][0], pl, acc[2 * k]);
                acc[2 * k + 1] = T::mma32(cring[k % AHEAD][1], pl, acc[2 * k + 1]);
                if (k + AHEAD < ks) {
                    cring[k % AHEAD][0] = c_operand(2 * (k + AHEAD));
                    cring[k % AHEAD][1] = c_operand(2 * (k + AHEAD) + 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
    };

    // ---- the units: loaded one ahead, page ids two ahead ----
    constexpr int STEP = ROWS ? 1 : 4;
    const int first = ROWS ? 0 : wave, tile0 = key0 >> 4;
    if constexpr (ROWS) {
        if (tid < 3 * SUB)
            marks[tid] = 0;
        __syncthreads();
    }
    Loaded x;
    Pages pages{};
    if (first < n_units) {
        pages = find_pages(tile0 + NT * first);
        load_unit(x, pages);
        pages = find_pages(tile0 + NT * (first + STEP));
    }
    for (int u = first; u < n_units; u += STEP) {
        const int t0 = tile0 + NT * u;
        uint16_t* sp = smem[ROWS ? (u & 1) * SUB : wave];
        const bool look = 16 * t0 + KEYS - 1 > seen_by_all;
        uint32_t ok[SUB], mark[SUB] = {};
#pragma unroll
        for (int k = 0; k < SUB; ++k)
            ok[k] = keys_of(t0, k);
        if ((ok[0] & ok[SUB - 1]) != 0xffffffffu || look)
            clean_unit(x, ok, mark, look);
        if constexpr (ROWS) {
            if (look && lane == 0)
#pragma unroll
                for (int k = 0; k < SUB; ++k)
                    if (mark[k])
                        atomicOr(&marks[u % 3 * SUB + k], mark[k]);
            stage_unit(x, sp);
            load_unit(x, pages);  // (the last one once more, at the end)
            pages = find_pages(t0 + 2 * NT * STEP);
            // The other buffer is free: every wave that passed the barrier before this one has
            // finished with it.  Likewise marks: unit u + 2's words, last read in unit u - 1, are
            // cleared behind this barrier and set again behind the next.
            __syncthreads();
            if (look) {
#pragma unroll
                for (int k = 0; k < SUB; ++k)
                    mark[k] = __builtin_amdgcn_readfirstlane(marks[u % 3 * SUB + k]);
            }
            if (causal_seg && tid < SUB)
                marks[(u + 2) % 3 * SUB + tid] = 0;
#pragma unroll
            for (int k = 0; k < SUB; ++k)
                if (16 * t0 + 32 * k <= lim_wave) {
                    floatx4 sc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                    take_scores(sp + k * SLOT, sc);
                    finish_unit(sc, sp + k * SLOT, t0 + 2 * k, ok[k], mark[k]);
                }
        } else {
            floatx4 sc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            stage_scores(x, sp, sc);
            load_unit(x, pages);
            pages = find_pages(t0 + 2 * NT * STEP);
            wave_lds_fence();
            finish_unit(sc, sp, t0, ok[0], mark[0]);
            wave_lds_fence();  // the slot's reads are done before the next unit's writes
        }
    }

    // ---- final rows, or partials ----
    typedef typename T::scalar s4 __attribute__((ext_vector_type(4)));
    auto rounded = [](floatx4 v) {
        s4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = static_cast<typename T::scalar>(v[i]);
        return x;
    };
    const float l = rows_sum(l_run);
    if constexpr (ROWS) {
        const int r = row0 + n;
        if (r >= n_rows)
            return;
        if (part < 0) {
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            uint16_t* o = a.out + ((long long)f0 + r) * KV;
#pragma unroll
            for (int rt = 0; rt < RTM; ++rt)
                if (rt < 2 * ks)
                    *reinterpret_cast<s4*>(o + 16 * rt + 4 * g) = rounded(acc[rt] * inv);
            if (a.lse && g == 0)
                a.lse[(long long)f0 + r] = (m_run + __log2f(l)) * kLn2;
        } else {
            float* o = a.part_o + ((long long)part + r) * KV;
#pragma unroll
            for (int rt = 0; rt < RTM; ++rt)
                if (rt < 2 * ks)
                    *reinterpret_cast<floatx4*>(o + 16 * rt + 4 * g) = acc[rt];
            if (g == 0) {
                a.part_ml[2 * ((long long)part + r)] = m_run;
                a.part_ml[2 * ((long long)part + r) + 1] = l;
            }
        }
    } else {
        // A wave parks its rows in its own slot: 16 rows of KV + 4 floats, then m and l.
        const int pitch = KV + 4;
        float* mine = reinterpret_cast<float*>(smem[wave]);
#pragma unroll
        for (int rt = 0; rt < RTM; ++rt)
            if (rt < 2 * ks)
                *reinterpret_cast<floatx4*>(mine + n * pitch + 16 * rt + 4 * g) = acc[rt];
        if (g == 0) {
            mine[16 * pitch + n] = m_run;
            mine[16 * pitch + 16 + n] = l;
        }
        __syncthreads();
        const int per_row = KV / 4;
        for (int e = tid; e < n_rows * per_row; e += kThreadsK) {
            const int r = e / per_row, c = (e % per_row) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int v = 0; v < 4; ++v)
                M = fmaxf(M, reinterpret_cast<const float*>(smem[v])[16 * pitch + r]);
            float L = 0.0f;
            floatx4 o = {0, 0, 0, 0};
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float* w = reinterpret_cast<const float*>(smem[v]);
                const float mv = w[16 * pitch + r];
                // A sum of NaN may come with a maximum of -inf (all scores NaN): weight 0 keeps it.
                const float f = mv == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mv - M);
                L += w[16 * pitch + 16 + r] * f;
                o += *reinterpret_cast<const floatx4*>(w + r * pitch + c) * f;
            }
            if (part < 0) {
                const float inv = L > 0.0f ? 1.0f / L : 0.0f;
                *reinterpret_cast<s4*>(a.out + ((long long)f0 + r) * KV + c) = rounded(o * inv);
                if (a.lse && c == 0)
                    a.lse[(long long)f0 + r] = (M + __log2f(L)) * kLn2;
            } else {
                *reinterpret_cast<floatx4*>(a.part_o + ((long long)part + r) * KV + c) = o;
                if (c == 0) {
                    a.part_ml[2 * ((long long)part + r)] = M;
                    a.part_ml[2 * ((long long)part + r) + 1] = L;
                }
            }
        }
    }
}

template <typename T, bool Q8, int KSM, bool ROWS, int RP = -1>
hipError_t launch_one(const LatentArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((latent_attend_kernel<T, Q8, KSM, ROWS, RP>),
                       dim3(ROWS ? a.jobs_r : a.jobs_k), dim3(ROWS ? kThreadsR : kThreadsK), 0,
                       stream, a);
    return hipGetLastError();
}

template <typename T, bool Q8, bool ROWS>
hipError_t launch_shape(const LatentArgs& a, hipStream_t stream) {
    const int ks = a.kv_rank / 32;
    if (ks == 4 && a.rope_dim == 16)
        return launch_one<T, Q8, 4, ROWS, 16>(a, stream);
    if (ks == 16 && a.rope_dim == 64)
        return launch_one<T, Q8, 16, ROWS, 64>(a, stream);
    return ks <= 4   ? launch_one<T, Q8, 4, ROWS>(a, stream)
           : ks <= 8 ? launch_one<T, Q8, 8, ROWS>(a, stream)
                     : launch_one<T, Q8, 16, ROWS>(a, stream);
}

template <typename T, bool Q8>
hipError_t launch_list(const LatentArgs& a, bool rows, hipStream_t stream) {
    return rows ? launch_shape<T, Q8, true>(a, stream) : launch_shape<T, Q8, false>(a, stream);
}

}  // namespace
}  // namespace mla
