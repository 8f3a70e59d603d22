// Verification of drafted tokens by the rejection rule: on logits
// (ultima_hsamp_verify_draft) and on kept sets (ultima_hsamp_verify_sets). The
// formulas stand at their declarations.
//
// On logits, four kernels:
//   k_draft_stats    every row in slices of 8192 ids: the slice's maximum m_s and
//                    sum of exp((x - m_s) / T) in double; greedy rows the lowest
//                    id of the maximum
//   k_draft_decide   one block per sequence: the rows' Z from their slices, the
//                    acceptance of every draft, the accepted tokens
//   k_draft_residual the slices' sums of max(p - q, 0) at the first rejected row
//   k_draft_pick     one block per sequence: the slice where the running sum
//                    reaches u_draw, then the id in it
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "ultima_hsamp.h"

namespace hsamp {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 8192;                 // ids per slice
constexpr float kNegInf = -__builtin_inff();
constexpr float kFltMax = 3.402823466e38f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

struct SliceStat {
    float m;        // maximum of the allowed logits, -inf: none
    int32_t at;     // greedy rows: the lowest id of the maximum
    double s;       // sum of exp((x - m) / T)
};

// What the later kernels need of a sequence's emitting row.
struct SeqRec {
    double zp, zq;           // the rows' sums at their maxima
    double cp, cq;           // 1 / T
    float mp, mq;            // maxima
    int32_t row, drow;       // target row; drafted row, -1: the weights are p's
    int32_t job;             // of the target row's slices
    int32_t pos;             // m
    int32_t point;           // >= 0: q is all on this id
    int32_t token;           // >= -1: known already; -2: to be drawn
};

struct DraftArgs {
    ultima_hsamp_draft d;
    SliceStat* stats;        // [jobs][S]
    double* rsum;            // [seqs][S]
    SeqRec* rec;             // [seqs]
    int S;
    int sides;               // 2 with the drafter's logits
};

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

// 1 / T as the exponents' factor; 0: greedy. (Above 0 at T = inf, so that
// -inf times it stays -inf.)
__device__ __forceinline__ double inv_temperature(const float* t, int b) {
    const float v = t != nullptr ? t[b] : 1.0f;
    return v > 0.0f ? fmax(1.0 / (double)v, 1e-300) : 0.0;
}

// NaN as -inf, +inf as the largest finite float.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, kNegInf), kFltMax); }

__device__ __forceinline__ double weight_of(float x, float m, double c) {
    return x > kNegInf ? exp(((double)x - (double)m) * c) : 0.0;
}

// VEC ids of a row at id e0 (a multiple of VEC), disallowed ones and those past
// the row's end as -inf.
template <bool BF>
struct RowReader {
    static constexpr int VEC = BF ? 8 : 4;
    const void* row;
    const uint32_t* mask;    // the row's words or NULL
    int V;
    __device__ __forceinline__ void load(int e0, float (&x)[VEC]) const {
        if (e0 + VEC <= V) {
            if (BF) {
                const u32x4 w = *reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(row) + e0);
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    x[k] = __uint_as_float(k & 1 ? w[k / 2] & 0xFFFF0000u : w[k / 2] << 16);
            } else {
                const u32x4 w = *reinterpret_cast<const u32x4_a4*>(static_cast<const float*>(row) + e0);
#pragma unroll
                for (int k = 0; k < VEC; ++k) x[k] = __uint_as_float(w[k % 4]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[k] = e0 + k < V ? one(e0 + k) : kNegInf;
        }
        uint32_t bits = 0xFFFFFFFFu;
        if (mask != nullptr && e0 < V) bits = mask[e0 >> 5] >> (e0 & 31);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = (bits >> k & 1u) != 0 ? clean(x[k]) : kNegInf;
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
};

template <bool BF>
__device__ __forceinline__ RowReader<BF> reader(const void* base, int64_t stride, const uint32_t* mask,
                                                int64_t mstride, int row, int V) {
    RowReader<BF> r;
    r.row = static_cast<const unsigned char*>(base) + (int64_t)row * stride * (BF ? 2 : 4);
    r.mask = mask != nullptr ? mask + (int64_t)row * mstride : nullptr;
    r.V = V;
    return r;
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
__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = lds[0];
    for (int w = 1; w < kThreads / 64; ++w) t += lds[w];
    return t;
}

// A job is one row: position i of sequence b, the target's (side 0) or the
// drafter's; jobs of one position stand together.
__device__ __forceinline__ int job_of(const DraftArgs& a, int b, int i, int side) {
    return i < a.d.max_draft ? (i * a.d.seqs + b) * a.sides + side : a.d.max_draft * a.d.seqs * a.sides + b;
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void k_draft_stats(DraftArgs a) {
    constexpr int VEC = RowReader<BF>::VEC, NC = kSlice / (kThreads * VEC);
    __shared__ float lm[kThreads / 64];
    __shared__ int li[kThreads / 64];
    __shared__ double ls[kThreads / 64];
    const int S = a.S, tid = threadIdx.x;
    const int job = blockIdx.x / S, slice = blockIdx.x % S;
    const int drafted = a.d.max_draft * a.d.seqs * a.sides;
    const int side = job < drafted ? job % a.sides : 0;
    const int i = job < drafted ? job / a.sides / a.d.seqs : a.d.max_draft;
    const int b = job < drafted ? job / a.sides % a.d.seqs : job - drafted;
    const Seq q = seq_of(a.d.n_draft, a.d.target_start, a.d.draft_start, b, a.d.max_draft, a.d.logits_rows,
                         a.d.draft_rows);
    if (!q.ok || i > q.n || (side == 1 && i == q.n)) return;
    const RowReader<BF> r =
        side == 0 ? reader<BF>(a.d.logits, a.d.logits_stride, a.d.mask, a.d.mask_stride, q.t0 + i, a.d.vocab)
                  : reader<BF>(a.d.draft_logits, a.d.draft_stride, a.d.draft_mask, a.d.draft_mask_stride, q.d0 + i,
                               a.d.vocab);
    const double c = inv_temperature(side == 0 ? a.d.temperature : a.d.draft_temperature, b);
    float x[NC][VEC];
    float m = kNegInf;
#pragma unroll
    for (int j = 0; j < NC; ++j) r.load(slice * kSlice + (j * kThreads + tid) * VEC, x[j]);
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) m = fmaxf(m, x[j][k]);
    m = wave_max(m);
    if ((tid & 63) == 0) lm[tid >> 6] = m;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, lm[w]);
    SliceStat st;
    st.m = m;
    st.at = 0;
    st.s = 0.0;
    if (c > 0.0) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) s += weight_of(x[j][k], m, c);
        st.s = block_sum(s, ls);
    } else {
        int at = INT32_MAX;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (x[j][k] == m) at = min(at, slice * kSlice + (j * kThreads + tid) * VEC + k);
        at = wave_min(at);
        if ((tid & 63) == 0) li[tid >> 6] = at;
        __syncthreads();
        for (int w = 0; w < kThreads / 64; ++w) at = min(at, li[w]);
        st.at = at;
        st.s = m > kNegInf ? 1.0 : 0.0;
    }
    if (tid == 0) a.stats[(int64_t)job * S + slice] = st;
}

struct RowSum {
    float m;
    int at;
    double z;       // at the maximum; greedy rows 1; 0: nothing allowed
};

// One wave: a row's maximum and sum from its slices.
__device__ __forceinline__ RowSum row_sum(const SliceStat* st, int S, double c) {
    const int lane = threadIdx.x & 63;
    RowSum r;
    float m = kNegInf;
    for (int s = lane; s < S; s += 64) m = fmaxf(m, st[s].m);
    r.m = m = wave_max(m);
    double z = 0.0;
    int at = INT32_MAX;
    for (int s = lane; s < S; s += 64) {
        const SliceStat v = st[s];
        if (c > 0.0) z += v.s * weight_of(v.m, m, c);
        else if (v.m == m && v.s > 0.0) at = min(at, v.at);
    }
    r.at = wave_min(at);
    r.z = c > 0.0 ? wave_sum(z) : (m > kNegInf ? 1.0 : 0.0);
    if (!(m > kNegInf)) r.z = 0.0;
    return r;
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void k_draft_decide(DraftArgs a) {
    __shared__ RowSum rp[ULTIMA_HSAMP_MAX_DRAFT + 1], rq[ULTIMA_HSAMP_MAX_DRAFT];
    __shared__ int lm[kThreads / 64];
    const int b = blockIdx.x, tid = threadIdx.x, K = a.d.max_draft, V = a.d.vocab;
    const Seq q = seq_of(a.d.n_draft, a.d.target_start, a.d.draft_start, b, K, a.d.logits_rows, a.d.draft_rows);
    int32_t* out = a.d.out_tokens + (int64_t)b * (K + 1);
    SeqRec rec{};
    rec.drow = -1;
    rec.point = -1;
    rec.token = -1;
    if (!q.ok) {
        for (int i = tid; i <= K; i += kThreads) out[i] = -1;
        if (tid == 0) {
            a.d.out_count[b] = 0;
            rec.pos = -1;
            a.rec[b] = rec;
        }
        return;
    }
    const double cp = inv_temperature(a.d.temperature, b), cq = inv_temperature(a.d.draft_temperature, b);
    for (int j = tid >> 6; j < 2 * q.n + 1; j += kThreads / 64) {
        const int i = j >> 1, side = j & 1;
        if (side == 1 && a.sides == 1) continue;
        const RowSum r = row_sum(a.stats + (int64_t)job_of(a, b, i, side) * a.S, a.S, side == 0 ? cp : cq);
        if ((tid & 63) == 0) (side == 0 ? rp[i] : rq[i]) = r;
    }
    __syncthreads();
    // p(d) and q(d) of draft i
    auto chance = [&](int i, int side, int tok) {
        if (tok < 0 || tok >= V) return 0.0;
        if (side == 1 && a.sides == 1) return 1.0;
        const RowSum r = side == 0 ? rp[i] : rq[i];
        if (!(r.z > 0.0)) return 0.0;
        const double c = side == 0 ? cp : cq;
        if (c == 0.0) return tok == r.at ? 1.0 : 0.0;
        const RowReader<BF> rd =
            side == 0 ? reader<BF>(a.d.logits, a.d.logits_stride, a.d.mask, a.d.mask_stride, q.t0 + i, V)
                      : reader<BF>(a.d.draft_logits, a.d.draft_stride, a.d.draft_mask, a.d.draft_mask_stride, q.d0 + i, V);
        return weight_of(rd.at(tok), r.m, c) / r.z;
    };
    int m = q.n;
    for (int i = tid; i < q.n; i += kThreads) {
        const int tok = a.d.draft[q.d0 + i];
        const double p = chance(i, 0, tok), qq = chance(i, 1, tok);
        if (!(a.d.u_accept[q.d0 + i] * qq < p)) m = min(m, i);
        if (a.d.accept_prob != nullptr) a.d.accept_prob[q.d0 + i] = p < qq ? (float)(p / qq) : p > 0.0 ? 1.0f : 0.0f;
    }
    m = wave_min(m);
    if ((tid & 63) == 0) lm[tid >> 6] = m;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) m = min(m, lm[w]);
    for (int i = tid; i <= K; i += kThreads) out[i] = i < m ? a.d.draft[q.d0 + i] : -1;
    // (the same threads wrote these above)
    if (a.d.accept_prob != nullptr)
        for (int i = tid; i < q.n; i += kThreads)
            if (i > m) a.d.accept_prob[q.d0 + i] = -1.0f;
    if (tid != 0) return;
    rec.pos = m;
    rec.row = q.t0 + m;
    rec.job = job_of(a, b, m, 0);
    rec.mp = rp[m].m;
    rec.zp = rp[m].z;
    rec.cp = cp;
    if (rec.zp > 0.0 && cp == 0.0) rec.token = rp[m].at;   // max(p - q, 0) is 0 but there; p is all there
    else if (rec.zp > 0.0) {
        rec.token = -2;
        if (m < q.n) {
            const int tok = a.d.draft[q.d0 + m];
            if (a.sides == 1) rec.point = tok;
            else if (rq[m].z > 0.0 && cq == 0.0) rec.point = rq[m].at;
            else if (rq[m].z > 0.0) {
                rec.drow = q.d0 + m;
                rec.mq = rq[m].m;
                rec.zq = rq[m].z;
                rec.cq = cq;
            }
        }
    }
    a.d.out_count[b] = m + (rec.token != -1 ? 1 : 0);
    a.rec[b] = rec;
}

// The weights of VEC ids from e0 on: max(p - q, 0), or p.
template <bool BF>
struct Weights {
    static constexpr int VEC = RowReader<BF>::VEC;
    RowReader<BF> p, q;
    float mp, mq;
    double cp, cq, zp, zq;
    int point;
    bool two;
    __device__ __forceinline__ Weights(const DraftArgs& a, const SeqRec& r) {
        p = reader<BF>(a.d.logits, a.d.logits_stride, a.d.mask, a.d.mask_stride, r.row, a.d.vocab);
        two = r.drow >= 0;
        q = two ? reader<BF>(a.d.draft_logits, a.d.draft_stride, a.d.draft_mask, a.d.draft_mask_stride, r.drow, a.d.vocab)
                : p;
        mp = r.mp, mq = r.mq, cp = r.cp, cq = r.cq, zp = r.zp, zq = r.zq, point = r.point;
    }
    __device__ __forceinline__ void load(int e0, double (&w)[VEC]) const {
        float x[VEC], y[VEC];
        p.load(e0, x);
        if (two) q.load(e0, y);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            w[k] = weight_of(x[k], mp, cp) / zp;
            if (two) w[k] = fmax(w[k] - weight_of(y[k], mq, cq) / zq, 0.0);
            if (e0 + k == point) w[k] = 0.0;
        }
    }
};

template <bool BF>
__global__ __launch_bounds__(kThreads) void k_draft_residual(DraftArgs a) {
    constexpr int VEC = RowReader<BF>::VEC, NC = kSlice / (kThreads * VEC);
    __shared__ double ls[kThreads / 64];
    const int b = blockIdx.x / a.S, slice = blockIdx.x % a.S;
    const SeqRec r = a.rec[b];
    if (r.token != -2) return;
    const Weights<BF> w(a, r);
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        double v[VEC];
        w.load(slice * kSlice + (j * kThreads + (int)threadIdx.x) * VEC, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) s += v[k];
    }
    s = block_sum(s, ls);
    if (threadIdx.x == 0) a.rsum[(int64_t)b * a.S + slice] = s;
}

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
        const unsigned long long hit = __ballot(v > 0.0 && c >= want);
        const unsigned long long some = __ballot(v > 0.0);
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
__global__ __launch_bounds__(kThreads) void k_draft_pick(DraftArgs a) {
    constexpr int VEC = RowReader<BF>::VEC, NC = kSlice / (kThreads * VEC);
    __shared__ double sums[NC * kThreads];
    __shared__ int pick[1];
    __shared__ double before_s[1];
    const int b = blockIdx.x, tid = threadIdx.x, S = a.S;
    SeqRec r = a.rec[b];
    if (r.pos < 0) return;
    int32_t* out = a.d.out_tokens + (int64_t)b * (a.d.max_draft + 1) + r.pos;
    if (r.token != -2) {
        if (tid == 0) *out = r.token;
        return;
    }
    const double* rs = a.rsum + (int64_t)b * S;
    const SliceStat* st = a.stats + (int64_t)r.job * S;
    double total = 0.0;
    for (int s = tid & 63; s < S; s += 64) total += rs[s];
    total = wave_sum(total);
    // p = q to the last bit: the weights are p's
    const bool whole = !(total > 0.0);
    if (whole) {
        r.drow = -1;
        r.point = -1;
        total = 1.0;
    }
    const double want = a.d.u_draw[b] * total;
    if (tid < 64) {
        double before;
        const int s = first_reaching(
            [&](int k) { return whole ? st[k].s * weight_of(st[k].m, r.mp, r.cp) / r.zp : rs[k]; }, S, 0.0, want, before);
        if (tid == 0) {
            pick[0] = s;
            before_s[0] = before;
        }
    }
    __syncthreads();
    const int slice = max(pick[0], 0);
    const Weights<BF> w(a, r);
    // the slice's chunks of VEC ids, in id order
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        double v[VEC], s = 0.0;
        w.load(slice * kSlice + (j * kThreads + tid) * VEC, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) s += v[k];
        sums[j * kThreads + tid] = s;
    }
    __syncthreads();
    if (tid >= 64) return;
    double before;
    const int chunk = max(0, first_reaching([&](int k) { return sums[k]; }, NC * kThreads, before_s[0], want, before));
    double v[VEC];
    w.load(slice * kSlice + chunk * VEC, v);
    int found = -1;
    double c = before;
    bool done = false;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        c += v[k];
        if (!done && v[k] > 0.0) {
            found = k;
            done = c >= want;
        }
    }
    if (tid == 0) *out = slice * kSlice + chunk * VEC + found;
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
    int64_t jobs, stats, rsum, rec, bytes;
};

// S slices of the row; the workspace's parts (offsets in bytes).
bool layout_of(int32_t seqs, int32_t max_draft, int32_t vocab, Layout& l) {
    if (seqs < 1 || max_draft < 0 || max_draft > ULTIMA_HSAMP_MAX_DRAFT || vocab < 1 || vocab > ULTIMA_HSAMP_MAX_VOCAB)
        return false;
    l.S = (vocab + kSlice - 1) / kSlice;
    l.jobs = (int64_t)seqs * (2 * max_draft + 1);
    l.stats = 0;
    l.rsum = l.jobs * l.S * (int64_t)sizeof(SliceStat);
    l.rec = l.rsum + (int64_t)seqs * l.S * 8;
    l.bytes = l.rec + (int64_t)seqs * (int64_t)sizeof(SeqRec);
    return true;
}

template <bool BF>
hipError_t launch_draft(const DraftArgs& a, int64_t jobs, hipStream_t s) {
    hipLaunchKernelGGL(k_draft_stats<BF>, dim3((uint32_t)(jobs * a.S)), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(k_draft_decide<BF>, dim3(a.d.seqs), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(k_draft_residual<BF>, dim3((uint32_t)a.d.seqs * a.S), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(k_draft_pick<BF>, dim3(a.d.seqs), dim3(kThreads), 0, s, a);
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
    a.S = l.S;
    a.sides = drafter ? 2 : 1;
    const int64_t jobs = (int64_t)d->seqs * (a.sides * (int64_t)d->max_draft + 1);
    // one block per slice of a row, numbered in 32 bits by their threads
    if (jobs * l.S > ((int64_t)1 << 32) / kThreads - 1) return ULTIMA_HSAMP_ERR_UNSUPPORTED;
    unsigned char* w = static_cast<unsigned char*>(d->work);
    a.stats = reinterpret_cast<SliceStat*>(w + l.stats);
    a.rsum = reinterpret_cast<double*>(w + l.rsum);
    a.rec = reinterpret_cast<SeqRec*>(w + l.rec);
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = d->dtype == ULTIMA_HSAMP_BF16 ? launch_draft<true>(a, jobs, s) : launch_draft<false>(a, jobs, s);
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
