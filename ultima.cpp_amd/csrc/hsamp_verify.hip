// Verification of drafted tokens by the rejection rule: on logits
// (ultima_hsamp_verify_draft) and on kept sets (ultima_hsamp_verify_sets). The
// formulas stand at their declarations.
//
// On logits, three kernels:
//   k_draft_start    clears the call's counters
//   k_draft_stats    a wave per slice of a row (16 KB of logits): its maximum m_s
//                    and sum of exp((x - m_s) / T) in double, a greedy row's lowest
//                    id of the maximum. Positions first, sequences second: the wave
//                    that completes a position's rows decides its draft, and waves
//                    of later positions find the rejection and read nothing. What
//                    they skip is never used, whether they see it or not.
//   k_draft_draw     a wave per slice of each sequence's emitting row: the slice's
//                    sum of max(p - q, 0); the wave that completes a sequence finds
//                    the slice where the running sum reaches u_draw, then the id.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "ultima_hsamp.h"

namespace hsamp {
namespace {

using u64 = unsigned long long;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kChunks = 16;                  // 16-byte loads of a lane per slice
constexpr float kNegInf = -__builtin_inff();
constexpr float kFltMax = 3.402823466e38f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// exp(d) in double for d <= 0 by Tang's table method: d = (k + f) ln 2 / 32, |f| <=
// 1/2, exp(d) = 2^(k >> 5) 2^((k & 31) / 32) exp(f ln 2 / 32), the last by its series
// to the fifth power (the sixth is below 3e-15). The 32 doubles of the table fill
// the 64 LDS banks once, so its reads never conflict. Fourteen double operations;
// the library's exp takes three times as long.
__device__ const double kPow[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

__device__ __forceinline__ void load_table(double* t) {
    if (threadIdx.x < 32) t[threadIdx.x] = kPow[threadIdx.x];
    __syncthreads();
}

// t = d 32 / ln 2, at most 0; below -32000 as -32000 (2^-1000).
__device__ __forceinline__ double exp32(double t, const double* table) {
    constexpr double kRound = 6755399441055744.0;        // 1.5 2^52: adding it rounds to a whole number
    t = fmax(t, -32000.0);
    const double u = t + kRound;
    const int k = (int)__double2loint(u);
    const double f = t - (u - kRound);
    double p = 0x1.5d87fe78a6731p-35;
    p = __builtin_fma(p, f, 0x1.3b2ab6fba4e77p-27);
    p = __builtin_fma(p, f, 0x1.c6b08d704a0c0p-20);
    p = __builtin_fma(p, f, 0x1.ebfbdff82c58fp-13);
    p = __builtin_fma(p, f, 0x1.62e42fefa39efp-6);
    const double b = table[k & 31];
    const double v = __builtin_fma(b * f, p, b);
    return __hiloint2double(__double2hiint(v) + ((k >> 5) << 20), __double2loint(v));
}
constexpr double kPerE = 46.166241308446828384;          // 32 / ln 2

struct SliceStat {
    uint32_t m;     // bits of the maximum of the allowed logits, -inf: none
    int32_t at;     // greedy rows: the lowest id of the maximum
    double s;       // sum of exp((x - m) / T)
};

struct DraftArgs {
    ultima_hsamp_draft d;
    SliceStat* stats;        // [jobs][S]
    double* rsum;            // [seqs][S]
    int32_t* count;          // [max_draft][seqs] slices of the position's rows that are done, then
    int32_t* drawn;          // [seqs] slices of the emitting row, and
    int32_t* rejected;       // [seqs] the lowest position known to be rejected
    int S;                   // slices per row
    int per;                 // slices in a row that one wave of k_draft_stats takes
    int sides;               // 2 with the drafter's logits
};

// What other XCDs' waves read in the same kernel goes past the caches both ways;
// a wave's values are there when its vmcnt is zero, before it counts itself done.
// (A release fence would write back the whole L2.)
template <class T>
__device__ __forceinline__ void put(T* p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ T get(const T* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put_stat(SliceStat* p, const SliceStat& v) {
    put(reinterpret_cast<u64*>(p), (u64)v.m | (u64)(uint32_t)v.at << 32);
    put(reinterpret_cast<u64*>(p) + 1, (u64)__double_as_longlong(v.s));
}
__device__ __forceinline__ SliceStat get_stat(const SliceStat* p) {
    const u64 a = get(reinterpret_cast<const u64*>(p)), s = get(reinterpret_cast<const u64*>(p) + 1);
    return SliceStat{(uint32_t)a, (int32_t)(a >> 32), __longlong_as_double((long long)s)};
}
// Whether this wave's n parts complete the `total` counted at p.
__device__ __forceinline__ bool completes(int32_t* p, int n, int total) {
    int before = 0;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if ((threadIdx.x & 63) == 0) before = __hip_atomic_fetch_add(p, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    before = __builtin_amdgcn_readfirstlane(before);
    asm volatile("" ::: "memory");
    return before + n == total;
}

struct Seq {
    int n, t0, d0;
    bool ok;
};

// A sequence's drafts and first rows; not ok: outside the arrays.
__device__ __forceinline__ Seq seq_of(const int32_t* n_draft, const int32_t* ts, const int32_t* ds, int b, int K,
                                      int rows, int drows) {
    Seq s;
    s.n = n_draft != nullptr ? n_draft[b] : K;
    s.t0 = ts != nullptr ? ts[b] : b * (K + 1);
    s.d0 = ds != nullptr ? ds[b] : b * K;
    s.ok = s.n >= 0 && s.n <= K && s.t0 >= 0 && (int64_t)s.t0 + s.n < rows &&
           (s.n == 0 || (s.d0 >= 0 && (int64_t)s.d0 + s.n <= drows));
    return s;
}
__device__ __forceinline__ Seq seq_of(const DraftArgs& a, int b) {
    return seq_of(a.d.n_draft, a.d.target_start, a.d.draft_start, b, a.d.max_draft, a.d.logits_rows, a.d.draft_rows);
}

// 32 / (T ln 2), the factor of the exponents; 0: greedy. (Above 0 at T = inf, so
// that -inf times it stays -inf.)
__device__ __forceinline__ double inv_temperature(const float* t, int b) {
    const float v = t != nullptr ? t[b] : 1.0f;
    return v > 0.0f ? fmax(1.0 / (double)v, 1e-300) * kPerE : 0.0;
}

// NaN as -inf, +inf as the largest finite float.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, kNegInf), kFltMax); }

// exp((x - m) / T) exactly 0 for what is not allowed, and below 2^-1000.
__device__ __forceinline__ double weight_of(float x, float m, double c, const double* table) {
    const double t = ((double)x - (double)m) * c;
    return x > kNegInf && t > -32000.0 ? exp32(t, table) : 0.0;
}

// A row as a wave reads it: slices of 16 KB in 16-byte chunks, chunk j of a lane
// the (64 j + lane)-th.
template <bool BF>
struct Row {
    static constexpr int VEC = BF ? 8 : 4;                 // ids per chunk
    static constexpr int SLICE = 64 * kChunks * VEC;       // ids per slice
    const void* row;
    const uint32_t* mask;    // the row's words or NULL
    int V;
    __device__ __forceinline__ static Row of(const void* base, int64_t stride, const uint32_t* mask, int64_t mstride,
                                             int row, int V) {
        Row r;
        r.row = static_cast<const unsigned char*>(base) + (int64_t)row * stride * (BF ? 2 : 4);
        r.mask = mask != nullptr ? mask + (int64_t)row * mstride : nullptr;
        r.V = V;
        return r;
    }
    __device__ __forceinline__ float one(int e) const {
        return BF ? __uint_as_float((uint32_t)static_cast<const uint16_t*>(row)[e] << 16)
                  : static_cast<const float*>(row)[e];
    }
    // an allowed id's logit, else -inf
    __device__ __forceinline__ float at(int e) const {
        if (mask != nullptr && (mask[e >> 5] >> (e & 31) & 1u) == 0) return kNegInf;
        return clean(one(e));
    }
    // the chunk at id e0 (a multiple of VEC); past the row's end -inf
    __device__ __forceinline__ u32x4 chunk(int e0) const {
        if (e0 + VEC <= V) {
            if (BF) return *reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(row) + e0);
            return *reinterpret_cast<const u32x4_a4*>(static_cast<const float*>(row) + e0);
        }
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = BF ? 0xFF80FF80u : 0xFF800000u;
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (e0 + k < V) {
                const uint32_t b = __float_as_uint(one(e0 + k));
                if (BF) w[k / 2] = k & 1 ? (w[k / 2] & 0xFFFFu) | (b & 0xFFFF0000u) : (w[k / 2] & 0xFFFF0000u) | b >> 16;
                else w[k % 4] = b;
            }
        return w;
    }
    __device__ __forceinline__ uint32_t bits(int e0) const {
        return mask != nullptr && e0 < V ? mask[e0 >> 5] >> (e0 & 31) : 0xFFFFFFFFu;
    }
    // id k of a chunk: its logit, -inf where it is not allowed
    __device__ __forceinline__ static float value(const u32x4& w, uint32_t bits, int k) {
        const float x = BF ? __uint_as_float(k & 1 ? w[k / 2] & 0xFFFF0000u : w[k / 2] << 16) : __uint_as_float(w[k % 4]);
        return (bits >> k & 1u) != 0 ? clean(x) : kNegInf;
    }
};

template <bool BF>
__device__ __forceinline__ Row<BF> target_row(const DraftArgs& a, int row) {
    return Row<BF>::of(a.d.logits, a.d.logits_stride, a.d.mask, a.d.mask_stride, row, a.d.vocab);
}
template <bool BF>
__device__ __forceinline__ Row<BF> draft_row(const DraftArgs& a, int row) {
    return Row<BF>::of(a.d.draft_logits, a.d.draft_stride, a.d.draft_mask, a.d.draft_mask_stride, row, a.d.vocab);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return v;
}

// A job is one row: position i of sequence b, the target's (side 0) or the
// drafter's; jobs of one position stand together.
__device__ __forceinline__ int job_of(const DraftArgs& a, int b, int i, int side) {
    return i < a.d.max_draft ? (i * a.d.seqs + b) * a.sides + side : a.d.max_draft * a.d.seqs * a.sides + b;
}

struct RowSum {
    float m;
    int at;
    double z;       // at the maximum; greedy rows 1; 0: nothing allowed
};

// One wave: a row's maximum and sum from its slices.
__device__ __forceinline__ RowSum row_sum(const SliceStat* st, int S, double c, const double* table) {
    const int lane = threadIdx.x & 63;
    float m = kNegInf;
    double z = 0.0;
    int at = INT32_MAX;
    for (int s0 = 0; s0 < S; s0 += 64) {
        SliceStat v{__float_as_uint(kNegInf), INT32_MAX, 0.0};
        if (s0 + lane < S) v = get_stat(st + s0 + lane);
        const float vm = __uint_as_float(v.m), top = fmaxf(m, wave_max(vm));
        if (c > 0.0) {
            z = z * weight_of(m, top, c, table) + wave_sum(v.s * weight_of(vm, top, c, table));
        } else {
            const int here = wave_min(vm == top && v.s > 0.0 ? v.at : INT32_MAX);
            at = top > m ? here : min(at, here);
        }
        m = top;
    }
    return RowSum{m, at, !(m > kNegInf) ? 0.0 : c > 0.0 ? z : 1.0};
}

__global__ __launch_bounds__(kThreads) void k_draft_start(DraftArgs a) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i < a.d.max_draft * a.d.seqs) a.count[i] = 0;
    if (i < a.d.seqs) {
        a.drawn[i] = 0;
        a.rejected[i] = INT32_MAX;
    }
}

// Draft i of sequence b, all slices of its rows known: one wave.
template <bool BF>
__device__ __forceinline__ void decide(const DraftArgs& a, const Seq& q, int b, int i, const double* table) {
    const double cp = inv_temperature(a.d.temperature, b), cq = inv_temperature(a.d.draft_temperature, b);
    const int tok = a.d.draft[q.d0 + i];
    const bool in = tok >= 0 && tok < a.d.vocab;
    auto chance = [&](const RowSum& r, double c, const Row<BF>& row) {
        if (!in || !(r.z > 0.0)) return 0.0;
        return c == 0.0 ? (tok == r.at ? 1.0 : 0.0) : weight_of(row.at(tok), r.m, c, table) / r.z;
    };
    const double p = chance(row_sum(a.stats + (int64_t)job_of(a, b, i, 0) * a.S, a.S, cp, table), cp,
                            target_row<BF>(a, q.t0 + i));
    double qd = in ? 1.0 : 0.0;
    if (a.sides == 2)
        qd = chance(row_sum(a.stats + (int64_t)job_of(a, b, i, 1) * a.S, a.S, cq, table), cq, draft_row<BF>(a, q.d0 + i));
    if ((threadIdx.x & 63) != 0) return;
    if (!(a.d.u_accept[q.d0 + i] * qd < p))
        __hip_atomic_fetch_min(&a.rejected[b], i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (a.d.accept_prob != nullptr) a.d.accept_prob[q.d0 + i] = p < qd ? (float)(p / qd) : p > 0.0 ? 1.0f : 0.0f;
}

template <bool BF, bool MASK>
__global__ __launch_bounds__(kThreads) void k_draft_stats(DraftArgs a) {
    using R = Row<BF>;
    __shared__ double table[32];
    load_table(table);
    const int lane = threadIdx.x & 63;
    const int groups = (a.S + a.per - 1) / a.per;        // waves per row
    const int w = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    const int job = w / groups, s0 = w % groups * a.per, s1 = min(a.S, s0 + a.per);
    const int drafted = a.d.max_draft * a.d.seqs * a.sides;
    if (job >= drafted + a.d.seqs) return;
    const int side = job < drafted ? job % a.sides : 0;
    const int i = job < drafted ? job / a.sides / a.d.seqs : a.d.max_draft;
    const int b = job < drafted ? job / a.sides % a.d.seqs : job - drafted;
    const Seq q = seq_of(a, b);
    // position n is the row after the last draft: in the place of position
    // max_draft for every sequence
    const int pos = job < drafted ? i : q.n;
    if (!q.ok || (job < drafted && i >= q.n)) return;
    if (pos > 0 && get(&a.rejected[b]) < pos) return;
    const R r = side == 0 ? target_row<BF>(a, q.t0 + pos) : draft_row<BF>(a, q.d0 + pos);
    const double c = inv_temperature(side == 0 ? a.d.temperature : a.d.draft_temperature, b);
    for (int s = s0; s < s1; ++s) {
        const int e0 = s * R::SLICE + lane * R::VEC;
        u32x4 x[kChunks];
        uint32_t bits[MASK ? kChunks : 1];
        if ((s + 1) * R::SLICE <= a.d.vocab) {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                if (BF) x[j] = *reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(r.row) + e0 + j * 64 * R::VEC);
                else x[j] = *reinterpret_cast<const u32x4_a4*>(static_cast<const float*>(r.row) + e0 + j * 64 * R::VEC);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kChunks; ++j) x[j] = r.chunk(e0 + j * 64 * R::VEC);
        }
        if (MASK)
#pragma unroll
            for (int j = 0; j < kChunks; ++j) bits[MASK ? j : 0] = r.bits(e0 + j * 64 * R::VEC);
        auto value = [&](int j, int k) { return R::value(x[j], MASK ? bits[MASK ? j : 0] : 0xFFFFFFFFu, k); };
        float m = kNegInf;
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int k = 0; k < R::VEC; ++k) m = fmaxf(m, value(j, k));
        m = wave_max(m);
        // (the values are unpacked again below: kept, they take twice the registers)
#pragma unroll
        for (int j = 0; j < kChunks; ++j) asm volatile("" : "+v"(x[j]));
        SliceStat st{__float_as_uint(m), INT32_MAX, 0.0};
        if (m > kNegInf) {
            if (c > 0.0) {
                // (what is not allowed adds 2^-1000 here)
                double sum = 0.0;
                const double md = m;
#pragma unroll
                for (int j = 0; j < kChunks; ++j)
#pragma unroll
                    for (int k = 0; k < R::VEC; ++k) sum += exp32(((double)value(j, k) - md) * c, table);
                st.s = wave_sum(sum);
            } else {
                int at = INT32_MAX;
#pragma unroll
                for (int j = 0; j < kChunks; ++j)
#pragma unroll
                    for (int k = 0; k < R::VEC; ++k)
                        if (value(j, k) == m) at = min(at, e0 + j * 64 * R::VEC + k);
                st.at = wave_min(at);
                st.s = 1.0;
            }
        }
        if (lane == 0) put_stat(a.stats + (int64_t)job * a.S + s, st);
    }
    if (job < drafted && completes(a.count + i * a.d.seqs + b, s1 - s0, a.sides * a.S)) decide<BF>(a, q, b, i, table);
}

// The weights of a chunk's ids: max(p - q, 0), or p; q on the drafter's row or on
// one id.
template <bool BF>
struct Weights {
    using R = Row<BF>;
    R p, q;
    RowSum sp, sq;
    double cp, cq;
    int point;
    bool two;
    __device__ __forceinline__ void load(int e0, const double* table, double (&w)[R::VEC]) const {
        const u32x4 x = p.chunk(e0);
        u32x4 y = x;
        if (two) y = q.chunk(e0);
        const uint32_t bx = p.bits(e0), by = two ? q.bits(e0) : 0u;
#pragma unroll
        for (int k = 0; k < R::VEC; ++k) {
            w[k] = weight_of(R::value(x, bx, k), sp.m, cp, table) / sp.z;
            if (two) w[k] = fmax(w[k] - weight_of(R::value(y, by, k), sq.m, cq, table) / sq.z, 0.0);
            if (e0 + k == point) w[k] = 0.0;
        }
    }
};

__device__ __forceinline__ double wave_incl_sum(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

// One wave: the first of n values above 0 where the running sum (from `base`)
// reaches `want`, else the last above 0 (-1: none); `before`: the sum before it.
template <class F>
__device__ __forceinline__ int first_reaching(F value, int n, double base, double want, double& before) {
    const int lane = threadIdx.x & 63;
    int last = -1;
    double last_before = base, run = base;
    for (int s0 = 0; s0 < n; s0 += 64) {
        const double v = s0 + lane < n ? value(s0 + lane) : 0.0;
        const double c = run + wave_incl_sum(v);
        const u64 hit = __ballot(v > 0.0 && c >= want);
        const u64 some = __ballot(v > 0.0);
        const int at = hit != 0 ? __ffsll((long long)hit) - 1 : some != 0 ? 63 - __clzll((long long)some) : -1;
        if (at >= 0) {
            last = s0 + at;
            last_before = __shfl(c - v, at, 64);
        }
        if (hit != 0) break;
        run = __shfl(c, 63, 64);
    }
    before = last_before;
    return last;
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void k_draft_draw(DraftArgs a) {
    using R = Row<BF>;
    __shared__ double table[32];
    load_table(table);
    const int lane = threadIdx.x & 63, S = a.S, K = a.d.max_draft;
    const int wv = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    const int b = wv / S, slice = wv % S;
    if (b >= a.d.seqs) return;
    const Seq q = seq_of(a, b);
    int32_t* out = a.d.out_tokens + (int64_t)b * (K + 1);
    const int m = q.ok ? min(a.rejected[b], q.n) : 0;
    if (slice == 0) {
        // all but the drawn token
        for (int i = lane; i <= K; i += 64)
            if (i != m) out[i] = q.ok && i < m ? a.d.draft[q.d0 + i] : -1;
        if (q.ok && a.d.accept_prob != nullptr)
            for (int i = m + 1 + lane; i < q.n; i += 64) a.d.accept_prob[q.d0 + i] = -1.0f;
    }
    Weights<BF> w;
    w.cp = inv_temperature(a.d.temperature, b);
    w.cq = inv_temperature(a.d.draft_temperature, b);
    const SliceStat* st = a.stats + (int64_t)job_of(a, b, m < q.n ? m : K, 0) * S;
    if (q.ok) w.sp = row_sum(st, S, w.cp, table);
    if (!q.ok || !(w.sp.z > 0.0) || w.cp == 0.0) {
        // no token, or a greedy one: max(p - q, 0) is 0 but there, and p is all there
        const bool some = q.ok && w.sp.z > 0.0;
        if (slice == 0 && lane == 0) {
            out[m] = some ? w.sp.at : -1;
            a.d.out_count[b] = m + (some ? 1 : 0);
        }
        return;
    }
    w.point = -1;
    w.two = false;
    w.p = w.q = target_row<BF>(a, q.t0 + m);
    w.sq = w.sp;
    if (m < q.n) {
        if (a.sides == 1) w.point = a.d.draft[q.d0 + m];
        else {
            w.sq = row_sum(a.stats + (int64_t)job_of(a, b, m, 1) * S, S, w.cq, table);
            if (w.sq.z > 0.0 && w.cq == 0.0) w.point = w.sq.at;
            w.two = w.sq.z > 0.0 && w.cq > 0.0;
            if (w.two) w.q = draft_row<BF>(a, q.d0 + m);
        }
    }
    auto p_slice = [&](int s) {
        const SliceStat v = get_stat(st + s);
        return v.s * weight_of(__uint_as_float(v.m), w.sp.m, w.cp, table) / w.sp.z;
    };
    // where the weights are p's, the slices' sums are known
    bool whole = !w.two && w.point < 0;
    double* rs = a.rsum + (int64_t)b * S;
    if (!whole) {
        double s = 0.0;
#pragma unroll 4
        for (int j = 0; j < kChunks; ++j) {
            double v[R::VEC];
            w.load(slice * R::SLICE + (j * 64 + lane) * R::VEC, table, v);
#pragma unroll
            for (int k = 0; k < R::VEC; ++k) s += v[k];
        }
        s = wave_sum(s);
        if (lane == 0) put(reinterpret_cast<u64*>(rs + slice), (u64)__double_as_longlong(s));
        if (!completes(&a.drawn[b], 1, S)) return;
    } else if (slice != 0) {
        return;
    }
    double total = whole ? 1.0 : 0.0;
    if (!whole) {
        for (int s = lane; s < S; s += 64) total += __longlong_as_double((long long)get(reinterpret_cast<const u64*>(rs + s)));
        total = wave_sum(total);
        if (!(total > 0.0)) {        // p = q to the last bit: the weights are p's
            whole = true;
            w.two = false;
            w.point = -1;
            total = 1.0;
        }
    }
    const double want = a.d.u_draw[b] * total;
    double before;
    const int at = max(0, first_reaching(
                              [&](int s) {
                                  return whole ? p_slice(s)
                                               : __longlong_as_double((long long)get(reinterpret_cast<const u64*>(rs + s)));
                              },
                              S, 0.0, want, before));
    // the slice's 64-chunk lines in id order, then the chunk, then the id
    int chunk = 0;
    double run = before;
    for (int j = 0; j < kChunks; ++j) {
        double v[R::VEC], s = 0.0;
        w.load(at * R::SLICE + (j * 64 + lane) * R::VEC, table, v);
#pragma unroll
        for (int k = 0; k < R::VEC; ++k) s += v[k];
        const double c = run + wave_incl_sum(s);
        const u64 hit = __ballot(s > 0.0 && c >= want), some = __ballot(s > 0.0);
        const int l = hit != 0 ? __ffsll((long long)hit) - 1 : some != 0 ? 63 - __clzll((long long)some) : -1;
        if (l >= 0) {
            chunk = j * 64 + l;
            before = __shfl(c - s, l, 64);
        }
        if (hit != 0) break;
        run = __shfl(c, 63, 64);
    }
    double v[R::VEC], c = before;
    w.load(at * R::SLICE + chunk * R::VEC, table, v);
    int found = 0;
    bool done = false;
#pragma unroll
    for (int k = 0; k < R::VEC; ++k) {
        c += v[k];
        if (!done && v[k] > 0.0) {
            found = k;
            done = c >= want;
        }
    }
    if (lane == 0) {
        out[m] = at * R::SLICE + chunk * R::VEC + found;
        a.d.out_count[b] = m + 1;
    }
}

// ---- kept sets ----------------------------------------------------------------------

__device__ __forceinline__ double set_prob(float p) { return p > 0.0f ? (double)p : 0.0; }

// The place of id among n ascending ids, -1: not among them.
__device__ __forceinline__ int find_id(const int32_t* ids, int n, int id) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ids[mid] < id) lo = mid + 1;
        else hi = mid;
    }
    return lo < n && ids[lo] == id ? lo : -1;
}

// One block per sequence.
__global__ __launch_bounds__(kThreads) void k_verify_sets(ultima_hsamp_draft_sets d) {
    __shared__ int lm[kThreads / 64];
    __shared__ double sums[kThreads];
    const int b = blockIdx.x, tid = threadIdx.x, K = d.max_draft;
    const Seq q = seq_of(d.n_draft, d.target_start, d.draft_start, b, K, d.rows, d.draft_rows);
    int32_t* out = d.out_tokens + (int64_t)b * (K + 1);
    const bool certain = d.draft_idx == nullptr;
    bool bad = !q.ok;
    if (!bad)
        for (int i = tid; i <= q.n; i += kThreads) {
            const int cp = d.kept_count[q.t0 + i];
            bad = bad || cp < 0 || cp > d.set_cap;
            if (!certain && i < q.n) {
                const int cq = d.draft_count[q.d0 + i];
                bad = bad || cq < 0 || cq > d.draft_cap;
            }
        }
    if (__syncthreads_or(bad)) {
        for (int i = tid; i <= K; i += kThreads) out[i] = -1;
        if (tid == 0) d.out_count[b] = 0;
        return;
    }
    int m = q.n;
    for (int i = tid; i < q.n; i += kThreads) {
        const int tok = d.draft[q.d0 + i];
        const int64_t tr = (int64_t)(q.t0 + i) * d.set_cap, dr = (int64_t)(q.d0 + i) * d.draft_cap;
        const int at = find_id(d.kept_idx + tr, d.kept_count[q.t0 + i], tok);
        const double p = at >= 0 ? set_prob(d.kept_prob[tr + at]) : 0.0;
        double qq = 1.0;
        if (!certain) {
            const int aq = find_id(d.draft_idx + dr, d.draft_count[q.d0 + i], tok);
            qq = aq >= 0 ? set_prob(d.draft_prob[dr + aq]) : 0.0;
        }
        if (!(d.u_accept[q.d0 + i] * qq < p)) m = min(m, i);
        if (d.accept_prob != nullptr) d.accept_prob[q.d0 + i] = p < qq ? (float)(p / qq) : p > 0.0 ? 1.0f : 0.0f;
    }
    m = wave_min(m);
    if ((tid & 63) == 0) lm[tid >> 6] = m;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) m = min(m, lm[w]);
    if (d.accept_prob != nullptr)
        for (int i = tid; i < q.n; i += kThreads)
            if (i > m) d.accept_prob[q.d0 + i] = -1.0f;
    // the emitting set: each thread a run of its entries
    const int n = d.kept_count[q.t0 + m];
    const int32_t* pi = d.kept_idx + (int64_t)(q.t0 + m) * d.set_cap;
    const float* pp = d.kept_prob + (int64_t)(q.t0 + m) * d.set_cap;
    const bool reject = m < q.n;
    const int point = reject && certain ? d.draft[q.d0 + m] : -1;
    const bool two = reject && !certain;
    const int64_t dr = two ? (int64_t)(q.d0 + m) * d.draft_cap : 0;
    const int nq = two ? d.draft_count[q.d0 + m] : 0;
    bool residual = true;
    auto weight = [&](int k) {
        double w = set_prob(pp[k]);
        if (!residual) return w;
        const int id = pi[k];
        if (reject && certain && id == point) return 0.0;
        if (two) {
            const int at = find_id(d.draft_idx + dr, nq, id);
            if (at >= 0) w = fmax(w - set_prob(d.draft_prob[dr + at]), 0.0);
        }
        return w;
    };
    const int run = (n + kThreads - 1) / kThreads;
    const int from = min(n, tid * run), to = min(n, from + run);
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        double s = 0.0;
        for (int k = from; k < to; ++k) s += weight(k);
        __syncthreads();
        sums[tid] = s;
        __syncthreads();
        total = 0.0;
        for (int k = tid & 63; k < kThreads; k += 64) total += sums[k];
        total = wave_sum(total);
        if (total > 0.0) break;
        residual = false;     // p = q to the last bit: the weights are p's
    }
    int token = -1;
    if (total > 0.0 && tid < 64) {
        const double want = d.u_draw[b] * total;
        double before;
        const int at = max(0, first_reaching([&](int k) { return sums[k]; }, kThreads, 0.0, want, before));
        double c = before;
        for (int k = min(n, at * run); k < min(n, at * run + run); ++k) {
            const double w = weight(k);
            c += w;
            if (w > 0.0) {
                token = pi[k];
                if (c >= want) break;
            }
        }
    }
    for (int i = tid; i <= K; i += kThreads)
        if (i != m) out[i] = i < m ? d.draft[q.d0 + i] : -1;
    if (tid == 0) {
        out[m] = token;
        d.out_count[b] = m + (total > 0.0 ? 1 : 0);
    }
}

struct Layout {
    int S;
    int64_t jobs, stats, rsum, counts, bytes;
};

int slices_of(int32_t vocab, bool bf) {
    const int slice = bf ? Row<true>::SLICE : Row<false>::SLICE;
    return (vocab + slice - 1) / slice;
}

// The workspace's parts (offsets in bytes), for either type.
bool layout_of(int32_t seqs, int32_t max_draft, int32_t vocab, Layout& l) {
    if (seqs < 1 || max_draft < 0 || max_draft > ULTIMA_HSAMP_MAX_DRAFT || vocab < 1 || vocab > ULTIMA_HSAMP_MAX_VOCAB)
        return false;
    l.S = slices_of(vocab, false);
    l.jobs = (int64_t)seqs * (2 * max_draft + 1);
    l.stats = 0;
    l.rsum = l.jobs * l.S * (int64_t)sizeof(SliceStat);
    l.counts = l.rsum + (int64_t)seqs * l.S * 8;
    l.bytes = l.counts + (int64_t)seqs * (max_draft + 2) * 4;
    return true;
}

template <bool BF>
hipError_t launch_draft(const DraftArgs& a, hipStream_t s) {
    const int64_t jobs = (int64_t)a.d.seqs * (a.sides * (int64_t)a.d.max_draft + 1);
    const int64_t waves = jobs * ((a.S + a.per - 1) / a.per), draws = (int64_t)a.d.seqs * a.S;
    const int64_t clear = std::max<int64_t>(1, (int64_t)a.d.max_draft) * a.d.seqs;
    auto blocks = [](int64_t n, int per) { return dim3((uint32_t)((n + per - 1) / per)); };
    hipLaunchKernelGGL(k_draft_start, blocks(clear, kThreads), dim3(kThreads), 0, s, a);
    if (a.d.mask != nullptr || a.d.draft_mask != nullptr)
        hipLaunchKernelGGL((k_draft_stats<BF, true>), blocks(waves, kWaves), dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((k_draft_stats<BF, false>), blocks(waves, kWaves), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(k_draft_draw<BF>, blocks(draws, kWaves), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace hsamp

extern "C" int64_t ultima_hsamp_verify_draft_work_bytes(int32_t seqs, int32_t max_draft, int32_t vocab) {
    hsamp::Layout l;
    return hsamp::layout_of(seqs, max_draft, vocab, l) ? l.bytes : -1;
}

extern "C" int ultima_hsamp_verify_draft(const ultima_hsamp_draft* d, void* hip_stream) {
    using namespace hsamp;
    Layout l;
    if (d == nullptr || !layout_of(d->seqs, d->max_draft, d->vocab, l)) return ULTIMA_HSAMP_ERR_INVALID;
    if (d->dtype != ULTIMA_HSAMP_F32 && d->dtype != ULTIMA_HSAMP_BF16) return ULTIMA_HSAMP_ERR_INVALID;
    if (d->logits == nullptr || d->u_draw == nullptr || d->out_tokens == nullptr || d->out_count == nullptr ||
        d->work == nullptr || reinterpret_cast<uintptr_t>(d->work) % 16 != 0)
        return ULTIMA_HSAMP_ERR_INVALID;
    if (d->logits_stride < d->vocab || d->logits_rows < 1 || d->draft_rows < 0) return ULTIMA_HSAMP_ERR_INVALID;
    if (d->draft_rows > 0 && (d->draft == nullptr || d->u_accept == nullptr)) return ULTIMA_HSAMP_ERR_INVALID;
    const int64_t words = ((int64_t)d->vocab + 31) / 32;
    if (d->mask != nullptr && d->mask_stride < words) return ULTIMA_HSAMP_ERR_INVALID;
    const bool drafter = d->draft_logits != nullptr;
    const uintptr_t es = d->dtype == ULTIMA_HSAMP_BF16 ? 2 : 4;
    if (reinterpret_cast<uintptr_t>(d->logits) % es != 0 || reinterpret_cast<uintptr_t>(d->draft_logits) % es != 0)
        return ULTIMA_HSAMP_ERR_INVALID;
    if (d->draft_logits != nullptr && d->draft_stride < d->vocab) return ULTIMA_HSAMP_ERR_INVALID;
    if (d->draft_mask != nullptr && (d->draft_logits == nullptr || d->draft_mask_stride < words))
        return ULTIMA_HSAMP_ERR_INVALID;
    // without starts of its own every sequence has its max_draft rows (plus one)
    if (d->target_start == nullptr && (int64_t)d->seqs * (d->max_draft + 1) > d->logits_rows)
        return ULTIMA_HSAMP_ERR_INVALID;
    if (d->draft_start == nullptr && (int64_t)d->seqs * d->max_draft > d->draft_rows) return ULTIMA_HSAMP_ERR_INVALID;
    DraftArgs a;
    a.d = *d;
    a.S = slices_of(d->vocab, d->dtype == ULTIMA_HSAMP_BF16);
    a.sides = drafter ? 2 : 1;
    // as many slices to a wave as leave a position's rows 4096 waves
    a.per = (int)std::clamp<int64_t>((int64_t)d->seqs * a.sides * a.S / 4096, 1, a.S);
    const int64_t jobs = (int64_t)d->seqs * (a.sides * (int64_t)d->max_draft + 1);
    // a wave per slice of a row, numbered in 32 bits by their threads
    if (jobs * a.S > ((int64_t)1 << 32) / 64 - kWaves) return ULTIMA_HSAMP_ERR_UNSUPPORTED;
    unsigned char* w = static_cast<unsigned char*>(d->work);
    a.stats = reinterpret_cast<SliceStat*>(w + l.stats);
    a.rsum = reinterpret_cast<double*>(w + l.rsum);
    a.count = reinterpret_cast<int32_t*>(w + l.counts);
    a.drawn = a.count + (int64_t)d->seqs * d->max_draft;
    a.rejected = a.drawn + d->seqs;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = d->dtype == ULTIMA_HSAMP_BF16 ? launch_draft<true>(a, s) : launch_draft<false>(a, s);
    return e == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}

extern "C" int ultima_hsamp_verify_sets(const ultima_hsamp_draft_sets* d, void* hip_stream) {
    using namespace hsamp;
    if (d == nullptr || d->seqs < 1 || d->max_draft < 0 || d->max_draft > ULTIMA_HSAMP_MAX_DRAFT)
        return ULTIMA_HSAMP_ERR_INVALID;
    if (d->rows < 1 || d->draft_rows < 0 || d->set_cap < 1 || d->set_cap > ULTIMA_HSAMP_MAX_VOCAB)
        return ULTIMA_HSAMP_ERR_INVALID;
    if (d->kept_idx == nullptr || d->kept_prob == nullptr || d->kept_count == nullptr || d->u_draw == nullptr ||
        d->out_tokens == nullptr || d->out_count == nullptr)
        return ULTIMA_HSAMP_ERR_INVALID;
    if (d->draft_rows > 0 && (d->draft == nullptr || d->u_accept == nullptr)) return ULTIMA_HSAMP_ERR_INVALID;
    const bool some = d->draft_idx != nullptr || d->draft_prob != nullptr || d->draft_count != nullptr;
    const bool all = d->draft_idx != nullptr && d->draft_prob != nullptr && d->draft_count != nullptr;
    if (some != all || (all && (d->draft_cap < 1 || d->draft_cap > ULTIMA_HSAMP_MAX_VOCAB)))
        return ULTIMA_HSAMP_ERR_INVALID;
    if (d->target_start == nullptr && (int64_t)d->seqs * (d->max_draft + 1) > d->rows) return ULTIMA_HSAMP_ERR_INVALID;
    if (d->draft_start == nullptr && (int64_t)d->seqs * d->max_draft > d->draft_rows) return ULTIMA_HSAMP_ERR_INVALID;
    hipLaunchKernelGGL(k_verify_sets, dim3(d->seqs), dim3(kThreads), 0, static_cast<hipStream_t>(hip_stream), *d);
    return hipGetLastError() == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}
