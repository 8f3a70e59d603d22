// Verification of drafted tokens by the rejection rule: on logits
// (ultima_hsamp_verify_draft) and on kept sets (ultima_hsamp_verify_sets). The
// formulas stand at their declarations.
//
// On logits:
//   k_draft_start    clears the call's counters
//   k_draft_stats    a wave per slice of a row (8 KB of logits): its maximum m_s
//                    and sum of exp((x - m_s) / T) in double, a greedy row's lowest
//                    id of the maximum. Positions first, sequences second: the block
//                    that completes a position's rows decides its draft, and blocks
//                    of later positions find the rejection and read nothing. What
//                    they skip is never used, whether they see it or not.
//   k_draft_exact    large bf16 calls only, whose sums above come from float
//                    exponentials: the emitting rows' slices again in double
//   k_draft_draw     a wave per part of a slice of each sequence's emitting row: its
//                    sum of max(p - q, 0); the block that completes a sequence
//                    finds the part where the running sum reaches u_draw, then the
//                    id.
//
// On kept sets: k_verify_sets, one launch or two.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "hsamp_wave.h"
#include "ultima_hsamp.h"

namespace hsamp {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kChunks = 8;                   // 16-byte loads of a lane per slice,
constexpr int kStep = 4;                     // of them a step, the next step's in flight
constexpr int kSteps = kChunks / kStep;
constexpr int kMaxParts = 4;                 // parts of a slice when a token is drawn
constexpr float kNegInf = -__builtin_inff();
constexpr float kFltMax = 3.402823466e38f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// exp(d) in double for d <= 0 by Tang's table method: d = (k + f) ln 2 / 32, |f| <=
// 1/2, exp(d) = 2^(k >> 5) 2^((k & 31) / 32) exp(f ln 2 / 32), the last a polynomial
// of the fourth degree (interpolated at the Chebyshev points, off by at most 1.6e-13:
// the decisions need 1e-11 or so, a float exponential's 1e-7 would move the draws).
// The 32 doubles of the table fill the 64 LDS banks once, so its reads never conflict.
__device__ const double kPow[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

// (in LDS without (k & 31) << 15 in the upper half: adding k << 15 there then adds
// k >> 5 to the exponent)
__device__ __forceinline__ void load_table(double* t) {
    const int k = threadIdx.x;
    if (k < 32) t[k] = __hiloint2double(__double2hiint(kPow[k]) - (k << 15), __double2loint(kPow[k]));
    __syncthreads();
}
__device__ __forceinline__ double power(const double* table, int k) {
    const double b = table[k & 31];
    return __hiloint2double(__double2hiint(b) + (k << 15), __double2loint(b));
}

constexpr double kPerE = 46.166241308446828384;          // 32 / ln 2
constexpr double kRound = 6755399441055744.0;            // 1.5 2^52: adding it rounds to a whole number

constexpr double kPoly[4] = {0x1.62e42fef8dc67p-6, 0x1.ebfbdff82240ap-13,
                             0x1.c6b13c3469da5p-20, 0x1.3b2b07bdf576cp-27};

// exp(d c ln 2 / 32) for d <= 0, d c >= -32600.
__device__ __forceinline__ double exp32(double d, double c, const double* table) {
    const double u = __builtin_fma(d, c, kRound);
    const int k = __double2loint(u);
    const double f = __builtin_fma(d, c, kRound - u);
    double p = __builtin_fma(kPoly[3], f, kPoly[2]);
    p = __builtin_fma(p, f, kPoly[1]);
    p = __builtin_fma(p, f, kPoly[0]);
    const double b = power(table, k);
    return __builtin_fma(b * f, p, b);
}

// N of them side by side, whose chains of operations overlap.
template <int N>
__device__ __forceinline__ void exp32n(const double (&d)[N], double c, const double* table, double (&v)[N]) {
    double u[N], f[N], p[N], b[N];
#pragma unroll
    for (int n = 0; n < N; ++n) u[n] = __builtin_fma(d[n], c, kRound);
#pragma unroll
    for (int n = 0; n < N; ++n) b[n] = power(table, __double2loint(u[n]));
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = kRound - u[n];
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = __builtin_fma(d[n], c, f[n]);
#pragma unroll
    for (int n = 0; n < N; ++n) p[n] = __builtin_fma(kPoly[3], f[n], kPoly[2]);
#pragma unroll
    for (int n = 0; n < N; ++n) p[n] = __builtin_fma(p[n], f[n], kPoly[1]);
#pragma unroll
    for (int n = 0; n < N; ++n) p[n] = __builtin_fma(p[n], f[n], kPoly[0]);
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = b[n] * f[n];
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = __builtin_fma(f[n], p[n], b[n]);
}

struct SliceStat {
    uint32_t m;     // bits of the maximum of the allowed logits, -inf: none
    int32_t at;     // greedy rows: the lowest id of the maximum
    double s;       // sum of exp((x - m) / T)
};

struct RowSum {
    float m;
    int at;
    double z;       // at the maximum; greedy rows 1; 0: nothing allowed
};

struct DraftArgs {
    ultima_hsamp_draft d;
    SliceStat* stats;        // [jobs][S]
    double* rsum;            // [seqs][parts of the row]
    RowSum* sums;            // [max_draft][seqs][sides] of the decided positions
    int32_t* count;          // [max_draft][seqs] slices of the position's rows that are done, then
    int32_t* drawn;          // [seqs] parts of the emitting row, and
    int32_t* rejected;       // [seqs] the lowest position known to be rejected
    int S;                   // slices per row
    int per;                 // slices in a row that one wave of k_draft_stats takes
    int sides;               // 2 with the drafter's logits
    int fast;                // float exponentials first
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
// Whether the block's n parts complete the `total` counted at p: for every thread
// of the block. One count a block: they queue at the address, 0.2 us each.
__device__ __forceinline__ bool completes(int32_t* p, int n, int total, int32_t* lds) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) *lds = __hip_atomic_fetch_add(p, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    return *lds + n == total;
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

// x between lo and the largest float, a quiet NaN as lo. A signalling one comes out as
// NaN: the instruction takes the minimum of the three in their order where one is NaN, and
// a minimum with a signalling NaN is NaN, without one the other value (hence x last, and
// a constant that the compiler does not know, which it would put there).
__device__ __forceinline__ float clamp(float x, float lo) {
    float most = kFltMax;
    asm("" : "+s"(most));
    return __builtin_amdgcn_fmed3f(lo, most, x);
}

// NaN as -inf, +inf as the largest finite float. (By comparisons: the compiler's maximum
// of three takes a signalling NaN for the other two.)
__device__ __forceinline__ float clean(float x) { return x > kNegInf ? (x < kFltMax ? x : kFltMax) : kNegInf; }

// exp((x - m) / T) exactly 0 for what is not allowed, and below 2^-1000.
__device__ __forceinline__ double weight_of(float x, float m, double c, const double* table) {
    const double d = (double)x - (double)m;
    return x > kNegInf && d * c > -32000.0 ? exp32(d, c, table) : 0.0;
}

// weight_of for many logits of a row with the maximum m: they are clamped to lo,
// 2^-1000 of the maximum, and lo's weight left out. Not for temperatures so low
// that lo is m or its neighbour, or so high that it is beyond the floats.
struct Scale {
    float m, lo;
    double md, c;
    bool fast;
    __device__ __forceinline__ Scale(float m_, double c_) : m(m_), md(m_), c(c_) {
        lo = (float)(md - 32000.0 / c);
        const double low = (md - (double)lo) * c;
        fast = lo > -3e38f && low > 31900.0 && low < 32100.0;
    }
    // (2^-1000 for what is not allowed, a signalling NaN's NaN)
    __device__ __forceinline__ double some(float x, const double* table) const {
        return exp32((double)clamp(x, lo) - md, c, table);
    }
    template <int N>
    __device__ __forceinline__ void some(const float (&x)[N], const double* table, double (&v)[N]) const {
        double d[N];
#pragma unroll
        for (int n = 0; n < N; ++n) d[n] = (double)clamp(x[n], lo) - md;
        exp32n(d, c, table, v);
    }
    // exactly 0 for what is not allowed and what lies below lo
    __device__ __forceinline__ void of4(const float (&x)[4], const double* table, double (&v)[4]) const {
        some(x, table, v);
        const bool all = (x[0] > lo) & (x[1] > lo) & (x[2] > lo) & (x[3] > lo);
        if (__ballot(!all) == 0) return;         // (a compare a value instead of three instructions)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            asm volatile("" : "+v"(v[n]));       // (else it is done without the branch)
            v[n] = x[n] > lo ? v[n] : 0.0;
        }
    }
    __device__ __forceinline__ double of(float x, const double* table) const {
        if (!fast) return weight_of(clean(x), m, c, table);
        return x > lo ? some(x, table) : 0.0;
    }
};

// A row as a wave reads it: slices of 8 KB in 16-byte chunks, chunk j of a lane
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
    // a chunk's ids that the bits leave out as -inf
    __device__ __forceinline__ static u32x4 masked(u32x4 w, uint32_t bits) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if ((bits >> k & 1u) == 0) {
                if (BF) w[k / 2] = k & 1 ? (w[k / 2] & 0xFFFFu) | 0xFF800000u : (w[k / 2] & 0xFFFF0000u) | 0xFF80u;
                else w[k % 4] = 0xFF800000u;
            }
        return w;
    }
    // id k of a chunk: its logit, -inf where it is masked
    __device__ __forceinline__ static float raw(const u32x4& w, uint32_t bits, int k) {
        const float x = BF ? __uint_as_float(k & 1 ? w[k / 2] & 0xFFFF0000u : w[k / 2] << 16) : __uint_as_float(w[k % 4]);
        return (bits >> k & 1u) != 0 ? x : kNegInf;
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

// Sums and maxima over the wave by DPP (shifts within 16 lanes, then the rows' ends
// carried on): lane 63 has the whole, and the inclusive sums are a scan's.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xF, false);
    return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double wave_incl_sum(double v) {
    v += dpp_f64<0x111, 0xF>(v);
    v += dpp_f64<0x112, 0xF>(v);
    v += dpp_f64<0x114, 0xF>(v);
    v += dpp_f64<0x118, 0xF>(v);
    v += dpp_f64<0x142, 0xA>(v);
    v += dpp_f64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane),
                            __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ double wave_sum(double v) { return lane_f64(wave_incl_sum(v), 63); }
__device__ __forceinline__ float wave_max(float v) {       // (of ordered bits: signed for positives, reversed below)
    const int b = __float_as_int(v);
    const uint32_t key = (uint32_t)(b ^ (b >> 31 & 0x7FFFFFFF)) ^ 0x80000000u;
    const uint32_t top = wave_max_u32(key) ^ 0x80000000u;
    return __int_as_float((int)top ^ ((int)top >> 31 & 0x7FFFFFFF));
}
__device__ __forceinline__ int wave_min(int v) {           // (of values >= 0)
    return (int)wave_min_u32((uint32_t)v);
}

// A job is one row: position i of sequence b, the target's (side 0) or the
// drafter's; jobs of one position stand together.
__device__ __forceinline__ int job_of(const DraftArgs& a, int b, int i, int side) {
    return i < a.d.max_draft ? (i * a.d.seqs + b) * a.sides + side : a.d.max_draft * a.d.seqs * a.sides + b;
}

// One wave: a row's maximum and sum from its slices; `first`: lane's slice of the
// first 64, loaded ahead.
template <class F>
__device__ __forceinline__ RowSum row_sum(F stat, SliceStat first, int S, double c, const double* table) {
    const int lane = threadIdx.x & 63;
    RowSum r{kNegInf, INT32_MAX, 0.0};
    for (int s0 = 0; s0 < S; s0 += 64) {
        if (s0 > 0) first = stat(s0 + lane);
        const float vm = s0 + lane < S ? __uint_as_float(first.m) : kNegInf;
        const double vs = s0 + lane < S ? first.s : 0.0;
        const float top = fmaxf(r.m, wave_max(vm));
        if (c > 0.0) {
            const double old = s0 > 0 ? r.z * weight_of(r.m, top, c, table) : 0.0;
            r.z = old + wave_sum(vs * weight_of(vm, top, c, table));
        } else {
            const int here = wave_min(vm == top && vs > 0.0 ? first.at : INT32_MAX);
            r.at = top > r.m ? here : min(r.at, here);
        }
        r.m = top;
    }
    if (!(r.m > kNegInf)) r.z = 0.0;
    else if (c == 0.0) r.z = 1.0;
    return r;
}

__global__ __launch_bounds__(kThreads) void k_draft_start(DraftArgs a) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i < a.d.max_draft * a.d.seqs) a.count[i] = 0;
    if (i < a.d.seqs) {
        a.drawn[i] = 0;
        a.rejected[i] = INT32_MAX;
    }
}

// Draft i of sequence b, all slices of its rows known: one wave. False, and nothing
// written: its u is within `margin` (of the larger side) of the border.
constexpr double kUnsure = 1e-5;             // each row's sum is off by at most 2.7e-6
template <bool BF>
__device__ __forceinline__ bool decide(const DraftArgs& a, const Seq& q, int b, int i, double margin, const double* table) {
    const int lane = threadIdx.x & 63;
    const double cp = inv_temperature(a.d.temperature, b), cq = inv_temperature(a.d.draft_temperature, b);
    const SliceStat* st = a.stats + (int64_t)job_of(a, b, i, 0) * a.S;     // (the drafter's row follows)
    auto stat = [&](int s) { return get_stat(st + min(s, a.S * a.sides - 1)); };
    auto stat_q = [&](int s) { return stat(a.S + s); };
    // every load that does not wait for another first
    const SliceStat fp = stat(lane), fq = stat_q(lane);
    const int tok = a.d.draft[q.d0 + i];
    const double u = a.d.u_accept[q.d0 + i];
    const bool in = tok >= 0 && tok < a.d.vocab;
    const float xp = in ? target_row<BF>(a, q.t0 + i).at(tok) : kNegInf;
    const float xq = in && a.sides == 2 ? draft_row<BF>(a, q.d0 + i).at(tok) : kNegInf;
    auto chance = [&](const RowSum& r, double c, float x) {
        if (!in || !(r.z > 0.0)) return 0.0;
        return c == 0.0 ? (tok == r.at ? 1.0 : 0.0) : weight_of(x, r.m, c, table) / r.z;
    };
    const RowSum rp = row_sum(stat, fp, a.S, cp, table);
    RowSum rq{};
    if (a.sides == 2) rq = row_sum(stat_q, fq, a.S, cq, table);
    const double p = chance(rp, cp, xp);
    const double qd = a.sides == 2 ? chance(rq, cq, xq) : in ? 1.0 : 0.0;
    if (fabs(u * qd - p) < margin * fmax(u * qd, p)) return false;
    if (lane != 0) return true;
    RowSum* left = a.sums + (int64_t)(i * a.d.seqs + b) * a.sides;
    left[0] = rp;
    if (a.sides == 2) left[1] = rq;
    if (!(u * qd < p)) __hip_atomic_fetch_min(&a.rejected[b], i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (a.d.accept_prob != nullptr) a.d.accept_prob[q.d0 + i] = p < qd ? (float)(p / qd) : p > 0.0 ? 1.0f : 0.0f;
    return true;
}

// One wave: slices s0 .. s1 - 1 of a row, each slice's statistics to to[s]. A step at
// a time, the next one's loads in flight.
//
// FAST: exponentials in float (a third of the instructions of those in double, which
// bound the pass). A slice's sum is then off by at most 45 2^-24 = 2.7e-6 of it: per term
// 2 |z| 2^-24 from the exponent z = (x - m) / T (the factor's rounding and the product's)
// and 2^-23 from exp2, where the terms' mean |z| is at most ln V < 17 (the entropy's
// bound); 9 2^-24 from the float additions. Enough to decide most drafts (kUnsure below), not
// to draw a token.
template <bool BF, bool MASK, bool FAST>
__device__ __forceinline__ void row_slices(const Row<BF>& r, double c, int s0, int s1, const double* table, SliceStat* to) {
    using R = Row<BF>;
    const int lane = threadIdx.x & 63;
    struct Step {
        u32x4 x[kStep];
        uint32_t bits[MASK ? kStep : 1];
    };
    auto load = [&](Step& h, int n) {          // a step wholly within the row
        const int e0 = n * (R::SLICE / kSteps) + lane * R::VEC;
#pragma unroll
        for (int j = 0; j < kStep; ++j) {
            if (BF) h.x[j] = *reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(r.row) + e0 + j * 64 * R::VEC);
            else h.x[j] = *reinterpret_cast<const u32x4_a4*>(static_cast<const float*>(r.row) + e0 + j * 64 * R::VEC);
        }
        if (MASK)
#pragma unroll
            for (int j = 0; j < kStep; ++j) h.bits[MASK ? j : 0] = r.mask != nullptr ? r.mask[(e0 + j * 64 * R::VEC) >> 5] : 0xFFFFFFFFu;
        if (MASK)
#pragma unroll
            for (int j = 0; j < kStep; ++j) h.bits[MASK ? j : 0] >>= (e0 + j * 64 * R::VEC) & 31;
    };
    float m = kNegInf;       // of the slice so far
    double sum = 0.0;        // the lane's, at m
    int at = INT32_MAX;
    auto add = [&](Step& h, int n) {
        auto value = [&](int j, int k) { return R::raw(h.x[j], MASK ? h.bits[MASK ? j : 0] : 0xFFFFFFFFu, k); };
        // the maximum by the bits as whole numbers, right where it comes out as a finite
        // float >= 0 (a NaN of positive sign lies above): half an instruction a value
        float top = -1.0f;
        {
            int t = INT32_MIN;
            if (MASK) {
#pragma unroll
                for (int j = 0; j < kStep; ++j)
#pragma unroll
                    for (int k = 0; k < R::VEC; ++k) t = max(t, __float_as_int(value(j, k)));
            } else if (BF) {
                s16x2 v = __builtin_bit_cast(s16x2, 0x80008000u);
#pragma unroll
                for (int j = 0; j < kStep; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t two = h.x[j][k];       // (a cast of the element itself takes the first)
                        v = __builtin_elementwise_max(v, __builtin_bit_cast(s16x2, two));
                    }
                t = max((int)v[0], (int)v[1]) << 16;
            } else {
#pragma unroll
                for (int j = 0; j < kStep; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) t = max(t, (int)h.x[j][k]);
            }
            t = (int)(wave_max_u32((uint32_t)t ^ 0x80000000u) ^ 0x80000000u);
            if (t >= 0 && t < 0x7F800000) top = __int_as_float(t);
        }
        if (top < 0.0f) {
            top = kNegInf;
#pragma unroll
            for (int j = 0; j < kStep; ++j)
#pragma unroll
                for (int k = 0; k < R::VEC; ++k) {
                    const float x = value(j, k);
                    top = x > top ? x : top;     // (a NaN is not above)
                }
            top = fminf(wave_max(top), kFltMax);
        }
        // (the values are unpacked again below: kept, they take twice the registers)
#pragma unroll
        for (int j = 0; j < kStep; ++j) asm volatile("" : "+v"(h.x[j]));
        if (c == 0.0) {
            if (!(top > m)) return;      // (the lowest id: the earlier step's)
            int here = INT32_MAX;        // (above top: +inf alone; a NaN is not at least top)
#pragma unroll
            for (int j = 0; j < kStep; ++j)
#pragma unroll
                for (int k = 0; k < R::VEC; ++k)
                    if (value(j, k) >= top) here = min(here, n * (R::SLICE / kSteps) + (j * 64 + lane) * R::VEC + k);
            at = wave_min(here);
            m = top;
            return;
        }
        if (top > m) {
            sum *= weight_of(m, top, c, table);
            m = top;
        }
        if (!(m > kNegInf)) return;
        const double per2 = c * 0.03125;             // log2 e / T
        const float flo = (float)((double)m - 160.0 / per2);
        const double flow = ((double)m - (double)flo) * per2;
        const float ch = (float)per2, mch = (float)((double)m * per2);
        if (FAST && flo > -3e38f && flow > 150.0 && flow < 170.0 && fabsf(mch) < 4096.0f) {
            // float exponentials of x ch - mch; what the rounding of mch moves all of them
            // by (below 2^-12) is taken out of their sum to the first order. Logits clamped
            // to flo, whose weight is 0 (not for the temperatures that Scale leaves out
            // either); the lane's four at a time in float, then in double
            const double moved = 1.0 - ((double)m * (double)ch - (double)mch) * 0.693147180559945309;
            float part = 0.0f;
#pragma unroll
            for (int j = 0; j < kStep; ++j)
#pragma unroll
                for (int k = 0; k < R::VEC; k += 4) {
                    float v[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float x = clamp(value(j, k + n), flo);
                        v[n] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, ch, -mch));
                    }
                    part += (v[0] + v[1]) + (v[2] + v[3]);
                }
            if (__ballot(part != part) == 0) {      // (a signalling NaN: by the loop below)
                sum += (double)part * moved;
                return;
            }
        }
        const Scale e(m, c);
        const double before = sum;
        if (e.fast) {
            // (what is not allowed adds 2^-1000 here)
#pragma unroll
            for (int j = 0; j < kStep; ++j)
#pragma unroll
                for (int k = 0; k < R::VEC; k += 4) {
                    float x[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) x[n] = value(j, k + n);
                    double v[4];
                    e.some(x, table, v);
                    sum += (v[0] + v[1]) + (v[2] + v[3]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            if (__ballot(sum != sum) == 0) return;
        }
        sum = before;
#pragma nounroll
        for (int j = 0; j < kStep * R::VEC; ++j) {
            const int id = n * (R::SLICE / kSteps) + j * 64 + lane;
            if (id < r.V) sum += weight_of(r.at(id), m, c, table);
        }
    };
    auto done = [&](int s) {
        const double z = wave_sum(sum);
        if (lane == 0)
            put_stat(to + s,
                     SliceStat{__float_as_uint(m), at, !(m > kNegInf) ? 0.0 : c > 0.0 ? z : 1.0});
        m = kNegInf;
        sum = 0.0;
        at = INT32_MAX;
    };
    // whole slices, their loads without a branch: else the compiler's wait for a step
    // is one for all loads, the next step's with them
    const int whole = min(s1, r.V / R::SLICE);
    Step h0, h1;
    if (s0 < whole) load(h0, kSteps * s0);
    for (int s = s0; s < whole; ++s) {
        for (int n = kSteps * s; n < kSteps * (s + 1); n += 2) {
            load(h1, n + 1);
            add(h0, n);
            load(h0, min(n + 2, kSteps * whole - 2));
            add(h1, n + 1);
        }
        done(s);
    }
    if (max(s0, whole) >= s1) return;
    // the row's last ids
#pragma nounroll
    for (int n = kSteps * (s1 - 1); n < kSteps * s1; ++n) {
        const int e0 = n * (R::SLICE / kSteps) + lane * R::VEC;
#pragma unroll
        for (int j = 0; j < kStep; ++j) {
            h0.x[j] = r.chunk(e0 + j * 64 * R::VEC);
            if (MASK) h0.bits[MASK ? j : 0] = r.bits(e0 + j * 64 * R::VEC);
        }
        add(h0, n);
    }
    done(s1 - 1);
}

// Bound by the bytes of the rows that are read and, as much, by the exponentials beside
// them: 64 sequences of 4 drafts over 151936 f32 logits 69 us, 311 MB at 4.5 TB/s (350 MB
// are there, the drafts up to the rejected ones need 267); 256 of 8 in bf16 179 us, 811 MB
// at 4.5 TB/s (1.3 GB there, 726 needed). 16 of 15 without a drafter 32 us, 87 MB (160
// there with their masks, 26 needed): positions in the air before a rejection is known.
// One sequence of 4: 11 us for 6 MB, the reads that wait for each other: a slice, and in
// the block that completes a position its count, the slices' sums, the drafted id, the
// logits at it. Four waves a SIMD: their registers.
template <bool BF, bool MASK, bool FAST>
__global__ __launch_bounds__(kThreads, 4) void k_draft_stats(DraftArgs a) {
    using R = Row<BF>;
    __shared__ double table[32];
    __shared__ int32_t shared;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int take = a.per * kWaves, groups = (a.S + take - 1) / take;       // slices per block, blocks per row
    const int job = blockIdx.x / groups, b0 = blockIdx.x % groups * take;
    const int s0 = min(a.S, b0 + wave * a.per), s1 = min(a.S, s0 + a.per);
    const int drafted = a.d.max_draft * a.d.seqs * a.sides;
    const int side = job < drafted ? job % a.sides : 0;
    const int i = job < drafted ? job / a.sides / a.d.seqs : a.d.max_draft;
    const int b = job < drafted ? job / a.sides % a.d.seqs : job - drafted;
    const Seq q = seq_of(a, b);
    // position n is the row after the last draft: in the place of position
    // max_draft for every sequence
    const int pos = job < drafted ? i : q.n;
    if (!q.ok || (job < drafted && i >= q.n)) return;
    if (threadIdx.x == 0) shared = pos > 0 ? get(&a.rejected[b]) : INT32_MAX;
    load_table(table);
    if (shared < pos) return;
    const R r = side == 0 ? target_row<BF>(a, q.t0 + pos) : draft_row<BF>(a, q.d0 + pos);
    const double c = inv_temperature(side == 0 ? a.d.temperature : a.d.draft_temperature, b);
    row_slices<BF, MASK, FAST>(r, c, s0, s1, table, a.stats + (int64_t)job * a.S);
    if (job >= drafted || !completes(a.count + i * a.d.seqs + b, min(take, a.S - b0), a.sides * a.S, &shared)) return;
    __shared__ int32_t unsure;
    if (wave == 0) {
        const bool far = decide<BF>(a, q, b, i, FAST ? kUnsure : 0.0, table);
        if (lane == 0) unsure = far ? 0 : 1;
    }
    if (!FAST) return;
    __syncthreads();
    if (unsure == 0) return;
    // too near to tell (once in 50 000 drafts): both rows again in double
    for (int sd = 0; sd < a.sides; ++sd) {
        const R row = sd == 0 ? target_row<BF>(a, q.t0 + i) : draft_row<BF>(a, q.d0 + i);
        const double cs = inv_temperature(sd == 0 ? a.d.temperature : a.d.draft_temperature, b);
        const int each = (a.S + kWaves - 1) / kWaves, from = min(a.S, wave * each);
        row_slices<BF, MASK, false>(row, cs, from, min(a.S, from + each), table, a.stats + (int64_t)job_of(a, b, i, sd) * a.S);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (wave == 0) decide<BF>(a, q, b, i, 0.0, table);
}

// FAST calls: the emitting rows' slices in double. (Greedy rows need none.) Bound by the
// exponentials: 256 sequences, 148 MB, 52 us.
template <bool BF, bool MASK>
__global__ __launch_bounds__(kThreads, 4) void k_draft_exact(DraftArgs a) {
    __shared__ double table[32];
    load_table(table);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int groups = (a.S + kWaves - 1) / kWaves;
    const int row = blockIdx.x / groups, s0 = blockIdx.x % groups * kWaves + wave;
    const int b = row / a.sides, side = row % a.sides;
    const Seq q = seq_of(a, b);
    if (!q.ok || s0 >= a.S) return;
    const int m = min(a.rejected[b], q.n);
    const double cp = inv_temperature(a.d.temperature, b), cq = inv_temperature(a.d.draft_temperature, b);
    if (cp == 0.0 || (side == 1 && (m == q.n || cq == 0.0))) return;
    const Row<BF> r = side == 0 ? target_row<BF>(a, q.t0 + m) : draft_row<BF>(a, q.d0 + m);
    row_slices<BF, MASK, false>(r, side == 0 ? cp : cq, s0, s0 + 1, table,
                                a.stats + (int64_t)job_of(a, b, m < q.n ? m : a.d.max_draft, side) * a.S);
}

// The weights of a chunk's ids, in units of 1 / the target's Z: max(p - q, 0), or p;
// q on the drafter's row or on one id.
template <bool BF>
struct Weights {
    using R = Row<BF>;
    R p, q;
    Scale ep, eq;
    double share;       // Z of the target over Z of the drafter
    int point;
    bool two;
    struct Chunk {
        u32x4 x, y;
        uint32_t bx, by;
        __device__ __forceinline__ void load(const R& p, const R& q, bool two, int e0) {
            x = y = p.chunk(e0);
            bx = by = p.bits(e0);
            if (two) {
                y = q.chunk(e0);
                by = q.bits(e0);
            }
        }
    };
    __device__ __forceinline__ Chunk load(int e0) const {
        Chunk c;
        c.load(p, q, two, e0);
        return c;
    }
    // a chunk's weights
    __device__ __forceinline__ void all(const Chunk& c, int e0, const double* table, double (&w)[R::VEC]) const {
        if (!ep.fast || !eq.fast) {
#pragma unroll
            for (int k = 0; k < R::VEC; ++k) w[k] = of(c, e0, k, table);
            return;
        }
        // (masks and the drafted id by branches that the whole block takes)
        u32x4 cx = c.x, cy = c.y;
        if (p.mask != nullptr) cx = R::masked(cx, c.bx);
        if (two && q.mask != nullptr) cy = R::masked(cy, c.by);
#pragma unroll
        for (int k0 = 0; k0 < R::VEC; k0 += 4) {
            float x[4];
            double v[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) x[n] = R::raw(cx, 0xFFFFFFFFu, k0 + n);
            ep.of4(x, table, v);
            if (two) {
                float y[4];
                double q[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) y[n] = R::raw(cy, 0xFFFFFFFFu, k0 + n);
                eq.of4(y, table, q);
#pragma unroll
                for (int n = 0; n < 4; ++n) v[n] = fmax(__builtin_fma(-share, q[n], v[n]), 0.0);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) w[k0 + n] = v[n];
        }
        if (point >= 0)
#pragma unroll
            for (int k = 0; k < R::VEC; ++k) w[k] = e0 + k == point ? 0.0 : w[k];
    }
    __device__ __forceinline__ double of(const Chunk& c, int e0, int k, const double* table) const {
        double w = ep.of(R::raw(c.x, c.bx, k), table);
        if (two) w = fmax(__builtin_fma(-share, eq.of(R::raw(c.y, c.by, k), table), w), 0.0);
        return e0 + k == point ? 0.0 : w;
    }
};

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
            last_before = lane_f64(c - v, at);
        }
        if (hit != 0) break;
        run = lane_f64(c, 63);
    }
    before = last_before;
    return last;
}

// TH threads a block, a wave per part of a slice (PARTS of them). Few sequences: bound by
// what waits for each other (statistics, part, count, parts' sums, the part again): one
// 9 us. Many: two exponentials an id: 256 over 151936 76 us.
template <bool BF, int TH, int PARTS>
__global__ __launch_bounds__(TH) void k_draft_draw(DraftArgs a) {
    using R = Row<BF>;
    __shared__ double table[32];
    __shared__ int32_t shared;
    load_table(table);
    constexpr int PART = R::SLICE / PARTS, CH = kChunks / PARTS;       // ids and chunks of a lane per part
    const int lane = threadIdx.x & 63, S = a.S, P = a.S * PARTS, K = a.d.max_draft;
    constexpr int NW = TH / 64;
    static_assert(NW >= PARTS && PARTS <= kMaxParts);
    const int groups = (P + NW - 1) / NW;
    const int b = blockIdx.x / groups, first = blockIdx.x % groups * NW;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = first + wave;
    const Seq q = seq_of(a, b);
    int32_t* out = a.d.out_tokens + (int64_t)b * (K + 1);
    const int m = q.ok ? min(a.rejected[b], q.n) : 0;
    if (part == 0) {
        // all but the drawn token
        for (int i = lane; i <= K; i += 64)
            if (i != m) out[i] = q.ok && i < m ? a.d.draft[q.d0 + i] : -1;
        if (q.ok && a.d.accept_prob != nullptr)
            for (int i = m + 1 + lane; i < q.n; i += 64) a.d.accept_prob[q.d0 + i] = -1.0f;
    }
    const double cp = inv_temperature(a.d.temperature, b), cq = inv_temperature(a.d.draft_temperature, b);
    // a rejected position's rows, their loads ahead of everything else
    const bool reject = q.ok && m < q.n, drafter = reject && a.sides == 2;
    Row<BF> pr{}, qr{};
    if (q.ok) pr = qr = target_row<BF>(a, q.t0 + m);
    if (drafter) qr = draft_row<BF>(a, q.d0 + m);
    typename Weights<BF>::Chunk c[CH];
    if (reject && cp > 0.0)
#pragma unroll
        for (int j = 0; j < CH; ++j) c[j].load(pr, qr, drafter, part * PART + (j * 64 + lane) * R::VEC);
    RowSum sp{kNegInf, INT32_MAX, 0.0}, sq = sp;
    const SliceStat* st = a.stats + (int64_t)job_of(a, b, K, 0) * S;      // of the row after the last draft
    if (reject) {
        st = a.stats + (int64_t)job_of(a, b, m, 0) * S;                   // (the drafter's row follows)
    }
    if (reject && !a.fast) {
        const RowSum* left = a.sums + (int64_t)(m * a.d.seqs + b) * a.sides;
        sp = left[0];
        if (drafter) sq = left[1];
    } else if (q.ok) {
        auto stat = [&](int s) { return st[min(s, S - 1)]; };
        auto stat_q = [&](int s) { return st[S + min(s, S - 1)]; };
        const SliceStat fp = stat(lane), fq = drafter ? stat_q(lane) : fp;
        sp = row_sum(stat, fp, S, cp, table);
        if (drafter) sq = row_sum(stat_q, fq, S, cq, table);
    }
    if (!(sp.z > 0.0) || cp == 0.0) {
        // no token, or a greedy one: max(p - q, 0) is 0 but there, and p is all there
        const bool some = sp.z > 0.0;
        if (part == 0 && lane == 0) {
            out[m] = some ? sp.at : -1;
            a.d.out_count[b] = m + (some ? 1 : 0);
        }
        return;
    }
    const bool two = drafter && sq.z > 0.0 && cq > 0.0;
    Weights<BF> w{pr, qr, Scale(sp.m, cp), Scale(two ? sq.m : sp.m, two ? cq : cp), two ? sp.z / sq.z : 0.0, -1, two};
    if (reject && a.sides == 1) w.point = a.d.draft[q.d0 + m];
    else if (drafter && sq.z > 0.0 && !two) w.point = sq.at;
    // where the weights are p's, the slices' sums are known
    bool whole = !two && w.point < 0;
    double* rs = a.rsum + (int64_t)b * P;
    if (!whole) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            double v[R::VEC];
            w.all(c[j], part * PART + (j * 64 + lane) * R::VEC, table, v);
#pragma unroll
            for (int k = 0; k < R::VEC; ++k) s += v[k];
        }
        s = wave_sum(s);
        if (lane == 0 && part < P) put(reinterpret_cast<u64*>(rs + part), (u64)__double_as_longlong(s));
        if (!completes(&a.drawn[b], min(NW, P - first), P, &shared)) return;
    } else if (first != 0) {
        return;
    }
    // one block of the sequence is left
    auto r_part = [&](int s) { return __longlong_as_double((long long)get(reinterpret_cast<const u64*>(rs + s))); };
    auto p_slice = [&](int s) { return st[s].s * weight_of(__uint_as_float(st[s].m), sp.m, cp, table); };
    // the first parts' sums, a few a lane, loaded once
    constexpr int HELD = 4;
    double held[HELD] = {}, total = 0.0;
    if (!whole) {
#pragma unroll
        for (int n = 0; n < HELD; ++n) held[n] = n * 64 + lane < P ? r_part(n * 64 + lane) : 0.0;
#pragma unroll
        for (int n = 0; n < HELD; ++n) total += held[n];
        for (int n = HELD * 64 + lane; n < P; n += 64) total += r_part(n);
        total = wave_sum(total);
    }
    if (!(total > 0.0)) {        // p's weights; also where p = q to the last bit
        whole = true;
        w.two = false;
        w.point = -1;
        total = sp.z;
    }
    const double want = a.d.u_draw[b] * total;
    double run;
    auto r_held = [&](int s) {
        const int n = s >> 6;
        return n == 0 ? held[0] : n == 1 ? held[1] : n == 2 ? held[2] : n == 3 ? held[3] : r_part(s);
    };
    // the part: of the parts' sums, or of the slice's that the known sums lead to
    int at;
    if (whole) {
        const int slice = max(0, first_reaching(p_slice, S, 0.0, want, run));
        __shared__ double sums[PARTS];
        if (wave < PARTS) {
            double v = 0.0;
#pragma unroll
            for (int j = 0; j < CH; ++j) c[j] = w.load((slice * PARTS + wave) * PART + (j * 64 + lane) * R::VEC);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                double x[R::VEC];
                w.all(c[j], (slice * PARTS + wave) * PART + (j * 64 + lane) * R::VEC, table, x);
#pragma unroll
                for (int k = 0; k < R::VEC; ++k) v += x[k];
            }
            v = wave_sum(v);
            if (lane == 0) sums[wave] = v;
        }
        __syncthreads();
        at = slice * PARTS + max(0, first_reaching([&](int n) { return sums[n]; }, PARTS, run, want, run));
    } else {
        at = max(0, first_reaching(r_held, P, 0.0, want, run));
    }
    if (wave != 0) return;
    // the part again, each lane CH chunks in a row: the lane, then the id among its
    // weights, a lane each
    constexpr int IDS = CH * R::VEC;
    static_assert(IDS <= 64);
    __shared__ double weights[64][IDS + 1];
    const int e0 = at * PART + lane * IDS;
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < CH; ++j) c[j] = w.load(e0 + j * R::VEC);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        double v[R::VEC];
        w.all(c[j], e0 + j * R::VEC, table, v);
#pragma unroll
        for (int k = 0; k < R::VEC; ++k) {
            weights[lane][j * R::VEC + k] = v[k];
            s += v[k];
        }
    }
    const double cum = run + wave_incl_sum(s);
    const u64 hit = __ballot(s > 0.0 && cum >= want), some = __ballot(s > 0.0);
    const int l = hit != 0 ? __ffsll((long long)hit) - 1 : some != 0 ? 63 - __clzll((long long)some) : 0;
    run = lane_f64(cum - s, l);
    __builtin_amdgcn_wave_barrier();
    const double mine = lane < IDS ? weights[l][lane] : 0.0;
    const double sum = run + wave_incl_sum(mine);
    const u64 reach = __ballot(mine > 0.0 && sum >= want), any = __ballot(mine > 0.0);
    const int id = reach != 0 ? __ffsll((long long)reach) - 1 : any != 0 ? 63 - __clzll((long long)any) : 0;
    if (lane == 0) {
        out[m] = at * PART + l * IDS + id;
        a.d.out_count[b] = m + 1;
    }
}

// ---- kept sets ----------------------------------------------------------------------

__device__ __forceinline__ double set_prob(float p) { return p > 0.0f ? (double)p : 0.0; }

// One wave: the places of id among the ascending ids of both sets, -1: not among
// them. Each step reads 64 of a set's ids, evenly spread over what is left, and both
// sets' reads are in flight together.
__device__ __forceinline__ void find_id(const int32_t* const (&ids)[2], int (&n)[2], int id, int (&at)[2]) {
    const int lane = threadIdx.x & 63;
    int from[2] = {};
    while (n[0] > 64 || n[1] > 64) {
        int piece[2], v[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            // the ends of pieces of n / 64 ids, rounded up
            piece[s] = (n[s] + 63) >> 6;
            v[s] = n[s] > 64 ? ids[s][from[s] + min(n[s], (lane + 1) * piece[s]) - 1] : id;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int skip = min(n[s], __popcll(__ballot(v[s] < id)) * piece[s]);      // pieces wholly below id
            from[s] += skip;
            n[s] = n[s] > 64 ? min(piece[s], n[s] - skip) : n[s];
        }
    }
    int v[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) v[s] = lane < n[s] ? ids[s][from[s] + lane] : 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const u64 hit = __ballot(lane < n[s] && v[s] == id);
        at[s] = hit != 0 ? from[s] + __ffsll((long long)hit) - 1 : -1;
    }
}

// One wave: where among the n ascending ids those from `low` to `high` begin and end.
__device__ __forceinline__ void range_of(const int32_t* ids, int n, int low, int high, int& begin, int& end) {
    const int lane = threadIdx.x & 63, key[2] = {low, high};
    int from[2] = {}, left[2] = {n, n};
    auto below = [&](int s, int v) { return s == 0 ? v < key[s] : v <= key[s]; };
    while (left[0] > 64 || left[1] > 64) {
        int piece[2], v[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            piece[s] = (left[s] + 63) >> 6;
            v[s] = left[s] > 0 ? ids[from[s] + min(left[s], (lane + 1) * piece[s]) - 1] : 0;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int skip = min(left[s], __popcll(__ballot(below(s, v[s]))) * piece[s]);
            from[s] += skip;
            left[s] = min(piece[s], left[s] - skip);
        }
    }
    int v[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) v[s] = lane < left[s] ? ids[from[s] + lane] : 0;
    begin = from[0] + __popcll(__ballot(lane < left[0] && below(0, v[0])));
    end = from[1] + __popcll(__ballot(lane < left[1] && below(1, v[1])));
}

constexpr int kEach = 8;                       // entries of a thread per tile
constexpr int kSetThreads = 512;
constexpr int kSetTile = kSetThreads * kEach;

// A thread's eight entries at e of a set of n >= 1 (the last one's past the end).
__device__ __forceinline__ void eight_of(const int32_t* ids, const float* probs, int e, int n, int (&id)[kEach], float (&p)[kEach]) {
    if (e + kEach <= n) {
#pragma unroll
        for (int k = 0; k < kEach; k += 4) {
            const u32x4 i4 = *reinterpret_cast<const u32x4_a4*>(ids + e + k), p4 = *reinterpret_cast<const u32x4_a4*>(probs + e + k);
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                id[k + f] = (int)i4[f];
                p[k + f] = __uint_as_float(p4[f]);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            id[k] = ids[min(e + k, n - 1)];
            p[k] = probs[min(e + k, n - 1)];
        }
    }
}

struct SetsArgs {
    ultima_hsamp_draft_sets d;
    double* sums;            // [seqs][T] of the emitting set's tiles, and
    int32_t* emits;          // [seqs] its position, -1: none (sets of several tiles)
    int T;                   // tiles that set_cap holds
    int blocks;              // per sequence
};

enum SetsPart { kSetsWhole, kSetsTiles, kSetsPick };

// The drafts' probabilities by a wave per position; then the emitting set in tiles of
// eight entries per thread, the drafter's entries of the tile's ids through LDS, where
// each entry of the target's looks for its own. What bounds it are the chains of reads
// that wait for each other (rows, counts, three or four steps of a search, a tile): 8 us
// for one sequence of sets up to 64, 11 for 64 of up to 1024. Larger sets would follow
// one block's tiles one after the other: 32 of up to 32768 ids 62 us, as here 21 + 15.
//   kSetsWhole: sets of one tile, one block per sequence
//   kSetsTiles: the tiles' sums, tiles shared out to a sequence's blocks (each finds
//               the emitting position by itself)
//   kSetsPick:  from these sums the tile, from it the token, one block per sequence
template <int PART>
__global__ __launch_bounds__(kSetThreads) void k_verify_sets(SetsArgs a) {
    const ultima_hsamp_draft_sets& d = a.d;
    constexpr int TILE = kSetTile, TH = kSetThreads, NW = TH / 64;
    __shared__ __attribute__((aligned(16))) int32_t lq[TILE];
    __shared__ __attribute__((aligned(16))) float lp[TILE];
    __shared__ double waves[NW];
    __shared__ int32_t first;
    const int b = PART == kSetsTiles ? blockIdx.x / a.blocks : blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int t0 = PART == kSetsTiles ? blockIdx.x % a.blocks : 0, K = d.max_draft;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Seq q = seq_of(d.n_draft, d.target_start, d.draft_start, b, K, d.rows, d.draft_rows);
    int32_t* out = d.out_tokens + (int64_t)b * (K + 1);
    const bool certain = d.draft_idx == nullptr, writes = PART != kSetsTiles || t0 == 0;
    int m;
    if (PART != kSetsPick) {
        if (tid == 0) first = INT32_MAX;
        bool bad = !q.ok, more = false;
        if (!bad)
            for (int i = tid; i <= q.n; i += TH) {
                const int cp = d.kept_count[q.t0 + i];
                bad = bad || cp < 0 || cp > d.set_cap;
                more = more || cp > t0 * TILE;
                if (!certain && i < q.n) {
                    const int cq = d.draft_count[q.d0 + i];
                    bad = bad || cq < 0 || cq > d.draft_cap;
                }
            }
        if (__syncthreads_or(bad)) {
            if (!writes) return;
            for (int i = tid; i <= K; i += TH) out[i] = -1;
            if (q.ok && d.accept_prob != nullptr)      // (else its rows are not known)
                for (int i = tid; i < q.n; i += TH) d.accept_prob[q.d0 + i] = -1.0f;
            if (tid == 0) d.out_count[b] = 0;
            if (PART == kSetsTiles && tid == 0) a.emits[b] = -1;
            return;
        }
        if (!writes && !__syncthreads_or(more)) return;        // (no set of the sequence has this tile)
        for (int i = wave; i < q.n; i += NW) {
            const int tok = d.draft[q.d0 + i];
            const double u = d.u_accept[q.d0 + i];
            const int64_t tr = (int64_t)(q.t0 + i) * d.set_cap, dr = (int64_t)(q.d0 + i) * d.draft_cap;
            const int32_t* const ids[2] = {d.kept_idx + tr, certain ? d.kept_idx : d.draft_idx + dr};
            int n[2] = {d.kept_count[q.t0 + i], certain ? 0 : d.draft_count[q.d0 + i]}, at[2];
            find_id(ids, n, tok, at);
            const double p = at[0] >= 0 ? set_prob(d.kept_prob[tr + at[0]]) : 0.0;
            const double qd = certain ? 1.0 : at[1] >= 0 ? set_prob(d.draft_prob[dr + at[1]]) : 0.0;
            if (lane == 0) {
                if (!(u * qd < p)) atomicMin(&first, i);
                if (writes && d.accept_prob != nullptr)
                    d.accept_prob[q.d0 + i] = p < qd ? (float)(p / qd) : p > 0.0 ? 1.0f : 0.0f;
            }
        }
        __syncthreads();
        m = min(first, q.n);
        if (writes && d.accept_prob != nullptr)
            for (int i = m + 1 + tid; i < q.n; i += TH) d.accept_prob[q.d0 + i] = -1.0f;
        if (writes)
            for (int i = tid; i <= K; i += TH)
                if (i != m) out[i] = i < m ? d.draft[q.d0 + i] : -1;
        if (PART == kSetsTiles && writes && tid == 0) a.emits[b] = m;
    } else {
        m = a.emits[b];
        if (m < 0) return;
    }
    const int n = d.kept_count[q.t0 + m];
    const int32_t* pi = d.kept_idx + (int64_t)(q.t0 + m) * d.set_cap;
    const float* pp = d.kept_prob + (int64_t)(q.t0 + m) * d.set_cap;
    const bool reject = m < q.n, two = reject && !certain;
    const int point = reject && certain ? d.draft[q.d0 + m] : -1;
    const int32_t* qi = two ? d.draft_idx + (int64_t)(q.d0 + m) * d.draft_cap : nullptr;
    const float* qp = two ? d.draft_prob + (int64_t)(q.d0 + m) * d.draft_cap : nullptr;
    const int nq = two ? d.draft_count[q.d0 + m] : 0;

    // A tile's weights, the thread's eight consecutive entries.
    int id[kEach];
    double w[kEach];
    auto tile = [&](int t, bool residual) {
        float p[kEach];
        eight_of(pi, pp, t * TILE + tid * kEach, n, id, p);
#pragma unroll
        for (int k = 0; k < kEach; ++k) w[k] = t * TILE + tid * kEach + k < n ? set_prob(p[k]) : 0.0;
        if (residual && reject && certain)
#pragma unroll
            for (int k = 0; k < kEach; ++k)
                if (id[k] == point) w[k] = 0.0;
        if (!residual || !two) return;
        // the drafter's ids of the tile's range: all of them in LDS, or the ends of as
        // many pieces as it holds, whose ids are looked through where they are
        int begin = 0, end = nq;
        if (nq > TILE) range_of(qi, nq, pi[t * TILE], pi[min(t * TILE + TILE, n) - 1], begin, end);
        const int in = max(0, end - begin), step = (in + TILE - 1) / TILE;
        if (in == 0) return;
        const int c = (in + step - 1) / step;
        int qid[kEach];
        if (step == 1) {
            eight_of(qi, qp, begin + tid * kEach, nq, qid, p);
        } else {
#pragma unroll
            for (int k = 0; k < kEach; ++k) qid[k] = qi[begin + (int)min((int64_t)in, (int64_t)(tid * kEach + k + 1) * step) - 1];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kEach; k += 4) {
            *reinterpret_cast<u32x4*>(&lq[tid * kEach + k]) =
                u32x4{(uint32_t)qid[k], (uint32_t)qid[k + 1], (uint32_t)qid[k + 2], (uint32_t)qid[k + 3]};
            *reinterpret_cast<f32x4*>(&lp[tid * kEach + k]) = f32x4{p[k], p[k + 1], p[k + 2], p[k + 3]};
        }
        __syncthreads();
        // the number of the LDS ids below each entry: of the first and the last in
        // step, then of those between within these bounds
        int lo[kEach] = {};
        for (int half = TILE; half > 0; half >>= 1)
#pragma unroll
            for (int k = 0; k < kEach; k += kEach - 1) {
                const int mid = lo[k] + half;
                if (mid <= c && lq[mid - 1] < id[k]) lo[k] = mid;
            }
        const int span = lo[kEach - 1] - lo[0];
#pragma unroll
        for (int k = 1; k < kEach - 1; ++k) lo[k] = lo[0];
        for (int half = span > 0 ? 1 << (31 - __clz(span)) : 0; __any(half > 0); half >>= 1)
#pragma unroll
            for (int k = 1; k < kEach - 1; ++k) {
                const int mid = lo[k] + half;
                if (half > 0 && mid <= lo[kEach - 1] && lq[mid - 1] < id[k]) lo[k] = mid;
            }
        if (step == 1) {
#pragma unroll
            for (int k = 0; k < kEach; ++k)
                if (lo[k] < c && lq[lo[k]] == id[k]) w[k] = fmax(w[k] - set_prob(lp[lo[k]]), 0.0);
            return;
        }
        int base[kEach], at[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            base[k] = begin + min(lo[k], c - 1) * step;
            at[k] = 0;
        }
        for (int half = 1 << (31 - __clz(step - 1)); half > 0; half >>= 1)
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const int mid = at[k] + half;
                if (qi[min(base[k] + mid, end) - 1] < id[k] && base[k] + mid < end) at[k] = mid;
            }
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (qi[base[k] + at[k]] == id[k]) w[k] = fmax(w[k] - set_prob(qp[base[k] + at[k]]), 0.0);
    };
    auto mine = [&]() {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) s += w[k];
        return s;
    };
    // a tile's sum, the waves' in LDS; for every thread
    auto tile_sum = [&](int t, bool residual) {
        tile(t, residual);
        const double s = wave_sum(mine());
        __syncthreads();
        if (lane == 0) waves[wave] = s;
        __syncthreads();
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < NW; ++k) v += waves[k];
        return v;
    };
    const int T = (n + TILE - 1) / TILE;
    double* sums = a.sums + (int64_t)b * a.T;
    auto all_tiles = [&](int from, int step, bool residual) {
        for (int t = from; t < T; t += step) {
            const double s = tile_sum(t, residual);
            if (tid == 0) sums[t] = s;
        }
    };
    if (PART == kSetsTiles) {
        all_tiles(t0, a.blocks, true);
        return;
    }
    double total = 0.0, run = 0.0;
    int at = 0;
    // (p = q to the last bit: the weights are p's)
    for (int pass = 0; pass < 2 && n > 0 && !(total > 0.0); ++pass) {
        if (PART == kSetsWhole) {
            total = tile_sum(0, pass == 0);
            continue;
        }
        if (pass > 0) {
            all_tiles(0, 1, false);
            __syncthreads();
        }
        total = 0.0;
        for (int t = lane; t < T; t += 64) total += sums[t];
        total = wave_sum(total);
        if (!(total > 0.0)) continue;
        at = max(0, first_reaching([&](int t) { return sums[t]; }, T, 0.0, d.u_draw[b] * total, run));
        tile_sum(at, pass == 0);
    }
    if (!(total > 0.0)) {
        if (tid == 0) {
            out[m] = -1;
            d.out_count[b] = m;
        }
        return;
    }
    const double want = d.u_draw[b] * total;
    // the wave, the thread, the entry
    const int hit = max(0, first_reaching([&](int k) { return waves[k]; }, NW, run, want, run));
    if (wave != hit) return;
    const double own = mine(), cum = run + wave_incl_sum(own);
    const u64 reach = __ballot(own > 0.0 && cum >= want), any = __ballot(own > 0.0);
    const int l = reach != 0 ? __ffsll((long long)reach) - 1 : any != 0 ? 63 - __clzll((long long)any) : 0;
    if (lane == l) {
        double c = cum - own;
        int token = id[0];
        bool done = false;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            c += w[k];
            if (!done && w[k] > 0.0) {
                token = id[k];
                done = c >= want;
            }
        }
        out[m] = token;
        d.out_count[b] = m + 1;
    }
}

// Float exponentials first, and the emitting rows (one or two of the 2 max_draft + 1)
// again in double: for bf16 rows, whose doubles take longer than their bytes, where
// many more rows are read than emit. 256 sequences of 8 drafts over 151936 ids (1.3 GB):
// the call 303 us against 353. Time against that of doubles alone, over 151936, 50257 and
// 32000 ids: 128 MB of 4 drafts 1.09, 1.12, 1.12, of 8 1.04, 1.09, 1.05; 512 MB of 4 0.90,
// 1.00, 0.97, of 8 1.03, 1.12, 1.09; 1 GB of 4 0.84, 1.01, 0.95, of 8 0.89, 0.90, 0.92;
// 2 GB of 4 0.87, 0.95, 0.96, of 8 0.76, 0.95, 0.91; of 2 drafts 1 GB 0.95, 1.02, 1.02.
constexpr int64_t kFastBytes = (int64_t)1 << 30;

struct Layout {
    int S;
    int64_t jobs, stats, sums, rsum, counts, bytes;
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
    l.sums = l.jobs * l.S * (int64_t)sizeof(SliceStat);
    l.rsum = l.sums + l.jobs * (int64_t)sizeof(RowSum);
    l.counts = l.rsum + (int64_t)seqs * l.S * kMaxParts * 8;
    l.bytes = l.counts + (int64_t)seqs * (max_draft + 2) * 4;
    return true;
}

template <bool BF>
hipError_t launch_draft(const DraftArgs& a, hipStream_t s) {
    const int64_t jobs = (int64_t)a.d.seqs * (a.sides * (int64_t)a.d.max_draft + 1);
    auto blocks = [](int64_t n, int per) { return (n + per - 1) / per; };
    const dim3 rows((uint32_t)(jobs * blocks(a.S, a.per * kWaves)));
    hipLaunchKernelGGL(k_draft_start, dim3((uint32_t)blocks(std::max<int64_t>(1, a.d.max_draft) * a.d.seqs, kThreads)),
                       dim3(kThreads), 0, s, a);
    const bool mask = a.d.mask != nullptr || a.d.draft_mask != nullptr;
    const dim3 emitting((uint32_t)((int64_t)a.d.seqs * a.sides * blocks(a.S, kWaves)));
    auto stats = [&](auto masked, auto fast) {
        constexpr bool MASK = decltype(masked)::value, FAST = decltype(fast)::value;
        hipLaunchKernelGGL((k_draft_stats<BF, MASK, FAST>), rows, dim3(kThreads), 0, s, a);
        if constexpr (FAST) hipLaunchKernelGGL((k_draft_exact<BF, MASK>), emitting, dim3(kThreads), 0, s, a);
    };
    auto by_mask = [&](auto fast) {
        if (mask) stats(std::true_type(), fast);
        else stats(std::false_type(), fast);
    };
    if constexpr (BF) {
        if (a.fast) by_mask(std::true_type());
        else by_mask(std::false_type());
    } else {
        by_mask(std::false_type());
    }
    auto draw = [&](auto th, auto parts) {
        constexpr int TH = decltype(th)::value, PARTS = decltype(parts)::value;
        hipLaunchKernelGGL((k_draft_draw<BF, TH, PARTS>), dim3((uint32_t)(a.d.seqs * blocks((int64_t)a.S * PARTS, TH / 64))),
                           dim3(TH), 0, s, a);
    };
    // few rows: more waves a slice, for its latency; many: fewer (each starts with the
    // sequence's own data), in smaller blocks. 4 of 512 threads against 2 of 256: one
    // sequence 9.0 and 11.4 us, 64 (f32) 31 and 28, 256 (bf16) 97 and 79.
    if ((int64_t)a.d.seqs * a.S < 4096) draw(std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
    else draw(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
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
    // (up to a block's waves more per row)
    if (std::max(jobs, (int64_t)d->seqs * kMaxParts) * (a.S + 8) > ((int64_t)1 << 32) / 64) return ULTIMA_HSAMP_ERR_UNSUPPORTED;
    // the rows and drafts that there are: with lengths of their own no more than the arrays hold
    const int64_t held = d->n_draft == nullptr ? jobs : std::min(jobs, (int64_t)d->logits_rows + (drafter ? d->draft_rows : 0));
    const bool drafts = d->max_draft >= 4 && (d->n_draft == nullptr || d->draft_rows / 4 >= d->seqs);
    a.fast = d->dtype == ULTIMA_HSAMP_BF16 && drafts && held * d->vocab * (int64_t)es > kFastBytes;
    unsigned char* w = static_cast<unsigned char*>(d->work);
    a.stats = reinterpret_cast<SliceStat*>(w + l.stats);
    a.sums = reinterpret_cast<RowSum*>(w + l.sums);
    a.rsum = reinterpret_cast<double*>(w + l.rsum);
    a.count = reinterpret_cast<int32_t*>(w + l.counts);
    a.drawn = a.count + (int64_t)d->seqs * d->max_draft;
    a.rejected = a.drawn + d->seqs;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = d->dtype == ULTIMA_HSAMP_BF16 ? launch_draft<true>(a, s) : launch_draft<false>(a, s);
    return e == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}

extern "C" int64_t ultima_hsamp_verify_sets_work_bytes(int32_t seqs, int32_t set_cap) {
    if (seqs < 1 || set_cap < 1 || set_cap > ULTIMA_HSAMP_MAX_VOCAB) return -1;
    const int64_t tiles = ((int64_t)set_cap + hsamp::kSetTile - 1) / hsamp::kSetTile;
    return tiles == 1 ? 0 : seqs * (tiles * 8 + 4);
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
    if (d->seqs > 1 << 21) return ULTIMA_HSAMP_ERR_UNSUPPORTED;        // (a launch's threads in 32 bits)
    SetsArgs a;
    a.d = *d;
    a.T = (d->set_cap + kSetTile - 1) / kSetTile;
    a.sums = static_cast<double*>(d->work);
    a.emits = reinterpret_cast<int32_t*>(a.sums + (int64_t)d->seqs * a.T);
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    if (a.T == 1) {
        a.blocks = 1;
        hipLaunchKernelGGL(k_verify_sets<kSetsWhole>, dim3(d->seqs), dim3(kSetThreads), 0, s, a);
    } else {
        if (d->work == nullptr || reinterpret_cast<uintptr_t>(d->work) % 16 != 0) return ULTIMA_HSAMP_ERR_INVALID;
        // a tile a block up to the 1024 blocks that the card holds at once
        a.blocks = std::clamp(1024 / d->seqs, 1, a.T);
        hipLaunchKernelGGL(k_verify_sets<kSetsTiles>, dim3(d->seqs * a.blocks), dim3(kSetThreads), 0, s, a);
        hipLaunchKernelGGL(k_verify_sets<kSetsPick>, dim3(d->seqs), dim3(kSetThreads), 0, s, a);
    }
    return hipGetLastError() == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}
