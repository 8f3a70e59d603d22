// The product with its epilogue (ultima_hsamp_linear): out = act(x W^T + bias) +
// residual, 16-bit inputs on the matrix cores with float sums.
//
// v_mfma_f32_16x16x32: lane 16 q + i feeds row i's elements 8q .. 8q + 7 of each
// operand. W is the first operand, so that a lane's four sums are four
// consecutive output columns of one row of x: bias, residual and output go in
// pieces of four.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "ultima_hsamp.h"

namespace hsamp {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));      // 16 bytes on any element's boundary
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <bool BF>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF>
__device__ __forceinline__ float to_f32(uint16_t h) {
    return BF ? __uint_as_float((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}
template <bool BF>
__device__ __forceinline__ uint16_t from_f32(float f) {   // to nearest, ties to even
    if (BF) return __builtin_bit_cast(uint16_t, (__bf16)f);
    return __builtin_bit_cast(uint16_t, (_Float16)f);
}

// 1 / (1 + exp(-t)) by the hardware's exp2 and reciprocal (one step of 2^-23
// each); the roundings of the exponent and of log2 e move exp(-t) by 1.3 |t| 2^-24 of
// it (5e-6 at 64), at most 2^-17 where the value is below 2^-126. exp(-t) past the
// largest float is infinite, the result 0.
// (With expf and a division the epilogue of 256 x 256 tiles took 90 of 554 us.)
__device__ __forceinline__ float sigmoid(float t) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t * -1.44269504f));
}

// c tanh(t), t = y / c: up to 1/2 by tanh's Taylor series (the next term is 10^-7 of the
// value there) as y (1 + t^2 ...), right also where t is subnormal or 0; from there by
// tanh(t) = 1 - 2 / (1 + exp(2 |t|)).
__device__ __forceinline__ float cap_of(float y, float t, float c) {
    const float z = t * t, u = fabsf(t);
    float p = 21844.0f / 6081075.0f;
    p = __builtin_fmaf(p, z, -1382.0f / 155925.0f);
    p = __builtin_fmaf(p, z, 62.0f / 2835.0f);
    p = __builtin_fmaf(p, z, -17.0f / 315.0f);
    p = __builtin_fmaf(p, z, 2.0f / 15.0f);
    p = __builtin_fmaf(p, z, -1.0f / 3.0f);
    const float low = __builtin_fmaf(y * z, p, y);
    const float high = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * 2.88539008f)), 1.0f);
    return u <= 0.5f ? low : c * __builtin_copysignf(high, t);       // (NaN: high's NaN)
}

using Args = ultima_hsamp_linear_args;

// The eight values of row m's columns n .. n + 7, where all of them are there.
__device__ __forceinline__ u32x4 eight(const Args& a, const void* base, int64_t at, int m, int n) {
    if (base == nullptr || m >= a.rows || n + 8 > a.out_dim) return u32x4{0, 0, 0, 0};
    return *reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(base) + at);
}
__device__ __forceinline__ u32x4 residual8(const Args& a, int g, int m, int n) {
    return eight(a, a.residual, g * a.residual_group + m * a.residual_stride + n, m, n);
}
__device__ __forceinline__ u32x4 bias8(const Args& a, int g, int n) {
    return eight(a, a.bias, g * a.bias_group + n, 0, n);
}

// E outputs (columns n .. n + E - 1 of row m, those there are) from their finished
// sums; bias, residual: eight()'s values.
template <bool BF, int E>
__device__ __forceinline__ void finish(const Args& a, int g, int m, int n, float (&y)[E], u32x4 bias, u32x4 residual) {
    typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
    const int left = a.out_dim - n;
    if (m >= a.rows || left <= 0) return;
    auto add = [&](const void* base, int64_t at, u32x4 v) {
        const uint16_t* p = static_cast<const uint16_t*>(base) + at;
        if (E == 8 && left >= 8) {
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] += to_f32<BF>((uint16_t)(v[e / 2 % 4] >> (16 * (e & 1))));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < left) y[e] += to_f32<BF>(p[e]);
        }
    };
    if (a.bias != nullptr) add(a.bias, g * a.bias_group + n, bias);
    switch (a.act) {
        case ULTIMA_HSAMP_ACT_RELU:
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = y[e] < 0.0f ? 0.0f : y[e];       // (NaN stays)
            break;
        case ULTIMA_HSAMP_ACT_SILU:
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = y[e] * sigmoid(y[e]);
            break;
        case ULTIMA_HSAMP_ACT_GELU:            // (by erfc: 1 + erf of a negative y cancels, at -5 to four places in a hundred)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float h = 0.5f * erfcf(fabsf(y[e]) * 0.70710678118654752f);
                y[e] = y[e] < 0.0f ? y[e] * h : y[e] * (1.0f - h);
            }
            break;
        case ULTIMA_HSAMP_ACT_GELU_TANH:       // (1 + tanh(t)) / 2 = 1 / (1 + exp(-2 t))
#pragma unroll
            for (int e = 0; e < E; ++e)
                y[e] = y[e] * sigmoid(1.59576912160573071f * (y[e] + 0.044715f * y[e] * y[e] * y[e]));
            break;
        case ULTIMA_HSAMP_ACT_SOFTCAP: {
            // (both scaled where 1 / c would be subnormal or infinite)
            const float c = a.act_param, scale = c < 0x1p-64f ? 0x1p64f : c > 0x1p64f ? 0x1p-64f : 1.0f;
            const float inv = 1.0f / (c * scale);
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = cap_of(y[e], y[e] * scale * inv, c);
            break;
        }
    }
    if (a.residual != nullptr) add(a.residual, g * a.residual_group + m * a.residual_stride + n, residual);
    const int64_t at = g * a.out_group + m * a.out_stride + n;
    if (a.out_dtype == ULTIMA_HSAMP_F32) {
        float* p = static_cast<float*>(a.out) + at;
        if (E == 8 && left >= 8) {
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<f32x4_a4*>(p + e) = f32x4{y[e], y[(e + 1) % E], y[(e + 2) % E], y[(e + 3) % E]};
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < left) p[e] = y[e];
        }
        return;
    }
    uint16_t* p = static_cast<uint16_t*>(a.out) + at;
    if (E == 8 && left >= 8) {
        u32x4 v = {};
#pragma unroll
        for (int e = 0; e < E / 2; ++e) v[e] = (uint32_t)from_f32<BF>(y[2 * e]) | (uint32_t)from_f32<BF>(y[(2 * e + 1) % E]) << 16;
        *reinterpret_cast<u32x4_a2*>(p) = v;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < left) p[e] = from_f32<BF>(y[e]);
    }
}

// A wave's 16 TM rows by 16 TN columns of sums, out through its own 16 rows of
// 16 TN + 4 floats of LDS, so that every lane finishes eight neighbouring
// columns.
template <bool BF, int TN, int TM>
__device__ __forceinline__ void store_tiles(const Args& a, int g, int m0, int n0, const f32x4 (&acc)[TN][TM], float* lds) {
    constexpr int LS = 16 * TN + 4, PR = 2 * TN;       // pieces of eight columns per row
    constexpr int NP = TN < 2 ? 1 : TN / 2;            // pieces of one lane per 16 rows
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const int c = lane % PR * 8, row = lane / PR;
    const bool on = row < 16;
    u32x4 res[NP], bias = bias8(a, g, n0 + c);
#pragma unroll
    for (int p = 0; p < NP; ++p) res[p] = residual8(a, g, m0 + row + 64 / PR * p, n0 + c);
#pragma unroll
    for (int u = 0; u < TM; ++u) {
        u32x4 next[NP] = {};
        if (u + 1 < TM)
#pragma unroll
            for (int p = 0; p < NP; ++p) next[p] = residual8(a, g, m0 + 16 * (u + 1) + row + 64 / PR * p, n0 + c);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < TN; ++s) *reinterpret_cast<f32x4*>(&lds[i * LS + 16 * s + 4 * q]) = acc[s][u];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int r = row + 64 / PR * p;
            if (!on) continue;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(&lds[r * LS + c]);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(&lds[r * LS + c + 4]);
            float y[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            finish<BF, 8>(a, g, m0 + 16 * u + r, n0 + c, y, bias, res[p]);
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) res[p] = next[p];
    }
}

// 16 WM TM rows of x by 16 WN TN rows of W by WM x WN x WK waves (WK of
// them sharing each tile's columns): global memory to LDS without registers, ST
// stages in the air or in LDS; the next step's operands are read while one is
// multiplied. A stage is 64 columns in two steps (WK = 1), or 32 WK columns, one
// step for each wave, whose sums meet in LDS at the end.
//
// Few rows: W's stream bounds it (one row of 4096 x 4096 8.3 us, 4.0 TB/s with the
// launch and the ramp in it; four groups of 64 rows 29 us, 134 MB at 4.6 TB/s): hence
// narrow tiles, whose waves share K instead of columns, and many loads in the air.
// Many: per stage the loads to LDS and the LDS reads beside the products: hence the
// widest tile that the accumulators allow, whose operands are read least often
// (4096 rows of 4096 x 16384 462 us, 1190 TFLOP/s, where 8192 cubed reaches 1215 to
// 1415 in the library, by card and clock; with bias, tanh and residual 533). Of its 1350
// MB from memory x is most: an XCD's 32 tiles in the air are all 16 of the rows by 2 of
// the columns, so each reads x four times (8 x 4 x 34 MB), the weight and the residual
// (134 MB each) come once. 320 rows of 4096 x 151936: 440 us (with the soft cap in float
// 463), 905 TFLOP/s: 194 MB are written, and two and a half tiles of rows need 160 of 128.
// ANY: rows at any element's address, a last piece of less than eight columns
// (loads to LDS take neither): one stage in registers, two in LDS.
template <bool BF, bool ANY, int WM, int WN, int WK, int TM, int TN, int ST>
__global__ __launch_bounds__(64 * WM * WN * WK) void k_linear_tile(Args a, int tiles_m, int tiles_n) {
#ifdef __HIP_DEVICE_COMPILE__    // (the buffer resource's type is the device compiler's alone)
    constexpr int NW = WM * WN * WK;
    constexpr int BM = 16 * WM * TM, BN = 16 * WN * TN, NS = WK == 1 ? 1 : WK / 2, BK = 64 * NS;
    constexpr int CX = BM / 8, CR = (BM + BN) / 8;       // loads (8 rows of 64 columns) of x, of all rows
    constexpr int CT = CR * NS;                          // per stage
    constexpr int NL = (CT + NW - 1) / NW;                     // of one wave, at most
    constexpr uint32_t kOutside = 0x80000000u;           // a buffer offset past every buffer: reads as zeros
    typedef __attribute__((address_space(3))) void* lds_ptr;
    constexpr int SB = (BM + BN) * BK;                   // elements per stage: by 64 columns x's rows, then W's
    constexpr int EB = WK == 1 ? NW * 16 * (16 * TN + 4) : NW * 256 * TM * TN;   // floats of the waves' sums in LDS
    static_assert((ST & (ST - 1)) == 0 && (!ANY || ST == 2) && ST * SB * 2 >= EB * 4 && ST * SB * 2 <= 160 * 1024);
    __shared__ __attribute__((aligned(16))) uint16_t sm[ST * SB];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int K = a.in_dim, g = blockIdx.z;
    // eight XCDs take blocks in turn: each gets a run of tiles, rows fastest, so
    // that its L2 holds what neighbours share
    const int total = tiles_m * tiles_n, per = total / 8, more = total % 8;
    const int xcd = blockIdx.x % 8, tile = xcd * per + min(xcd, more) + blockIdx.x / 8;
    const int m0 = tile % tiles_m * BM, n0 = tile / tiles_m * BN;
    const uint16_t* X = static_cast<const uint16_t*>(a.x) + g * a.x_group + m0 * a.x_stride;
    const uint16_t* W = static_cast<const uint16_t*>(a.weight) + g * a.weight_group + n0 * a.weight_stride;
    const auto rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(X), 0, 0x7FFFFFFF, 0x00027000);
    const auto rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(W), 0, 0x7FFFFFFF, 0x00027000);
    // A load takes 8 rows of 128 bytes: whole lines (with 64 bytes of 16 rows the
    // next stage's loads find their lines still in flight, and the cache stalls).
    // A 16-byte LDS read serves 16 lanes at a time: q = 0 of rows 0 - 3 and
    // 12 - 15 with q = 1 of rows 4 - 11, and so on. Row r's piece p stands at
    // p ^ (r / 2 % 8), which puts each such sixteen into all 64 banks.
    uint32_t vo[NL];
    const uint16_t* row[ANY ? NL : 1];
    int col[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int c = wave + NW * j, rc = c % CR, r = (rc < CX ? rc : rc - CX) * 8 + (lane >> 3);
        col[j] = c / CR * 64 + ((lane & 7) ^ (r >> 1 & 7)) * 8;
        const bool in = rc < CX ? m0 + r < a.rows : n0 + r < a.out_dim;
        if (ANY) row[j] = rc < CX ? X + min(r, a.rows - 1 - m0) * a.x_stride : W + min(r, a.out_dim - 1 - n0) * a.weight_stride;
        else vo[j] = in ? (uint32_t)(r * (int)(rc < CX ? a.x_stride : a.weight_stride) + col[j]) * 2u : kOutside;
    }
    const int T = (K + BK - 1) / BK;
    const bool full = wave + NW * (NL - 1) < CT;          // this wave has NL loads a stage, not NL - 1
    // Each XCD starts at another eighth of the columns: rows a power of two apart
    // lie in the same memory channels, and blocks in step would all read one.
    const int t0 = (int)((int64_t)xcd * T / 8);
    auto issue = [&](int s) {
        const int t = s + t0 < T ? s + t0 : s + t0 - T;
        const int left = s < T ? K - t * BK : 0;
        uint16_t* to = sm + (s & (ST - 1)) * SB;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const int c = wave + NW * j;
            const uint32_t v = col[j] < left ? vo[j] : kOutside;
            if (j == NL - 1 && CT % NW != 0 && !full) {
            } else if ((NS == 1 && NW * j + NW - 1 < CX) || c % CR < CX)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr)(to + c * 512), 16, v, t * BK * 2, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr)(to + c * 512), 16, v, t * BK * 2, 0, 0);
        }
    };
    u32x4 held[ANY ? NL : 1];
    auto fetch = [&](int s) {
        const int t = s + t0 < T ? s + t0 : s + t0 - T;
        if (s >= T) return;
        const int left = K - t * BK;
        if (left >= BK) {
#pragma unroll
            for (int j = 0; j < NL; ++j)
                if (CT % NW == 0 || j < NL - 1 || full)
                    held[j] = *reinterpret_cast<const u32x4_a2*>(row[j] + (int64_t)t * BK + col[j]);
            return;
        }
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            if (CT % NW != 0 && j == NL - 1 && !full) continue;
            const uint16_t* p = row[j] + (int64_t)t * BK + col[j];
            u32x4 v = {0, 0, 0, 0};
            if (col[j] + 8 <= left) v = *reinterpret_cast<const u32x4_a2*>(p);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col[j] + e < left) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
            held[j] = v;
        }
    };
    auto store = [&](int s) {
#pragma unroll
        for (int j = 0; j < NL; ++j)
            if (CT % NW == 0 || j < NL - 1 || full)
                *reinterpret_cast<u32x4*>(&sm[(s & 1) * SB + (wave + NW * j) * 512 + lane * 8]) = held[j];
    };
    // all but this wave's loads of the last `stages` stages are in LDS, its reads done
    auto wait = [&](auto stages) {
        constexpr int S = decltype(stages)::value, A = S * NL, B = S * (NL - 1);
        static_assert(A < 64);
        constexpr int wa = (A & 15) | (A >> 4) << 14 | 7 << 4, wb = (B & 15) | (B >> 4) << 14 | 7 << 4;
        if (CT % NW == 0 || full) __builtin_amdgcn_s_waitcnt(wa);
        else __builtin_amdgcn_s_waitcnt(wb);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    struct Operands {
        u32x4 w[TN], x[TM];
    };
    const int wk = wave / (WM * WN), wm = wave % WM * 16 * TM, wn = wave / WM % WN * 16 * TN;
    auto read = [&](Operands& o, int t, int step) {
        const uint16_t* from = sm + (t & (ST - 1)) * SB + step / 2 * (CR * 512) + ((step % 2 * 4 + q) ^ (i >> 1)) * 8;
#pragma unroll
        for (int s = 0; s < TN; ++s) o.w[s] = *reinterpret_cast<const u32x4*>(from + (BM + wn + 16 * s + i) * 64);
#pragma unroll
        for (int s = 0; s < TM; ++s) o.x[s] = *reinterpret_cast<const u32x4*>(from + (wm + 16 * s + i) * 64);
        __builtin_amdgcn_sched_barrier(0);      // (and the reads ahead of the products)
    };
    f32x4 acc[TN][TM] = {};
    auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int s = 0; s < TN; ++s)
#pragma unroll
            for (int u = 0; u < TM; ++u) acc[s][u] = mfma<BF>(o.w[s], o.x[u], acc[s][u]);
        __builtin_amdgcn_sched_barrier(0);      // (the products stay ahead of the next wait)
    };
    using std::integral_constant;
    Operands oa, ob;
    if constexpr (ANY) {
        fetch(0);
        store(0);
        fetch(1);
        __syncthreads();
        if (WK == 1) read(oa, 0, 0);
        for (int t = 0; t < T; ++t) {
            // (the place of stage t + 1 was read before the last barrier)
            if (t + 1 < T) store(t + 1);
            fetch(t + 2);
            read(WK == 1 ? ob : oa, t, WK == 1 ? 1 : wk);
            multiply(oa);
            __syncthreads();
            if (WK == 1) {
                if (t + 1 < T) read(oa, t + 1, 0);
                multiply(ob);
            }
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int t = 0; t < ST; ++t) issue(t);
        wait(integral_constant<int, ST - 1>());
        // (a stage past the last reads as zeros)
        if (WK == 1) {
            read(oa, 0, 0);
            for (int t = 0; t < T; ++t) {
                read(ob, t, 1);
                multiply(oa);
                wait(integral_constant<int, ST - 2>());
                issue(t + ST);
                read(oa, t + 1, 0);
                multiply(ob);
            }
        } else {
            read(oa, 0, wk);
            for (int t = 0; t < T; t += 2) {
                wait(integral_constant<int, ST - 2>());
                issue(t + ST);
                read(ob, t + 1, wk);
                multiply(oa);
                wait(integral_constant<int, ST - 2>());
                issue(t + 1 + ST);
                read(oa, t + 2, wk);
                multiply(ob);
            }
        }
        wait(integral_constant<int, 0>());
    }
    float* sums = reinterpret_cast<float*>(sm);
    if (WK == 1) {
        store_tiles<BF, TN, TM>(a, g, m0 + wm, n0 + wn, acc, sums + wave * 16 * (16 * TN + 4));
        return;
    }
    // rows of 4 TN pieces of four floats, row r's piece p at p ^ r % (4 TN): the 16
    // rows of a store lie in different banks
    constexpr int PC = 4 * TN;
    auto place = [&](int w, int r, int p) { return ((w * 16 * TM + r) * PC + (p ^ (r & (PC - 1)))) * 4; };
#pragma unroll
    for (int u = 0; u < TM; ++u)
#pragma unroll
        for (int s = 0; s < TN; ++s) *reinterpret_cast<f32x4*>(&sums[place(wave, 16 * u + i, 4 * s + q)]) = acc[s][u];
    __syncthreads();
    constexpr int E = BM * BN >= 64 * NW * 8 ? 8 : 1;
    for (int o = tid; o < BM * BN / E; o += 64 * NW) {
        const int m = o / (BN / E), n = o % (BN / E) * E;
        const int w = n / (16 * TN) * WM + m / (16 * TM), p = n % (16 * TN) / 4;
        float y[E] = {};
#pragma unroll
        for (int k = 0; k < WK; ++k)
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                const float* from = &sums[place(w + k * WM * WN, m % (16 * TM), p + e / 4)];
                if (E == 1) {
                    y[0] += from[n % 4];
                } else {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(from);
#pragma unroll
                    for (int f = 0; f < 4; ++f) y[(e + f) % E] += v[f];
                }
            }
        finish<BF, E>(a, g, m0 + m, n0 + n, y, E == 8 ? bias8(a, g, n0 + n) : u32x4{},
                      E == 8 ? residual8(a, g, m0 + m, n0 + n) : u32x4{});
    }
#endif
}

// A form of k_linear_tile: its tile, how many blocks one CU holds, and what a
// round of one block per CU (one[0]) and of two (one[1]) costs, in us at
// K = 4096. Measured, N = 4096 and 16384 (bf16), rows 1 to 4096:
//   16 x 16 rows 1: 7.8, 25 us; 32 x 32 rows 32: 14.5, 26; 64 x 16 rows 64: 15, 56;
//   64 x 32 rows 64: 17.5, 37, rows 256: 31, 120; 64 x 64 by 8 waves rows 256: 34, 75,
//   rows 512: 39, 133; by 16, with twice the bytes in the air and one block to a CU,
//   rows 64: -, 32, rows 256: 24, -; 128 x 128 rows 256: 41, 56, rows 1024: 52, 168;
//   160 x 128 rows 512: 63, 83, rows 2048: 76, 284; 256 x 256 rows 1024: 101, 123, rows
//   4096 (f16): -, 462.
// Rows at any alignment take the nearest of three tiles by the same costs, which are not
// theirs. K = 4097, the tile it takes and the best of the three: N = 4096, rows 64 22, 22;
// 256 47, 36; 512 58, 56; 1024 68, 66; 2048 99, 95. N = 16384, rows 64 47, 36; 128 58,
// 57; 256 68, 66; 1024 191, 187.
struct Form {
    int bm, bn, blocks;
    float one[2];
};
constexpr Form kForms[] = {
    {16, 16, 2, {8, 12}}, {32, 32, 2, {13, 25}}, {64, 16, 1, {14.5f, 0}}, {64, 32, 1, {15.5f, 0}}, {64, 64, 2, {32, 39}},
    {64, 64, 1, {24, 0}}, {128, 128, 1, {44, 0}}, {160, 128, 2, {62, 84}}, {256, 256, 1, {112, 0}},
};

// Blocks of one group.
int64_t blocks_of(const Form& f, const Args& a) {
    return (((int64_t)a.rows + f.bm - 1) / f.bm) * (((int64_t)a.out_dim + f.bn - 1) / f.bn);
}

// Up to 32 rows: the narrowest form that holds them (bound by W's stream at any
// width). More: the form whose rounds over the 256 CUs cost least.
int choose(const Args& a) {
    if (a.rows <= 32) return a.rows <= 16 ? 0 : 1;
    int best = 0;
    float least = 0;
    for (int f = 2; f < (int)(sizeof(kForms) / sizeof(kForms[0])); ++f) {
        const Form& v = kForms[f];
        const int64_t blocks = blocks_of(v, a) * a.groups;
        const int64_t round = 256 * v.blocks, rest = blocks % round;
        const float cost = (float)(blocks / round) * v.one[v.blocks - 1] +
                           (rest == 0 ? 0.0f : rest <= 256 ? v.one[0] : v.one[v.blocks - 1]);
        if (f == 2 || cost < least) {
            best = f;
            least = cost;
        }
    }
    return best;
}

template <bool BF, bool ANY, int WM, int WN, int WK, int TM, int TN, int ST>
hipError_t launch_tile(const Args& a, hipStream_t s) {
    const int tm = (a.rows + 16 * WM * TM - 1) / (16 * WM * TM), tn = (a.out_dim + 16 * WN * TN - 1) / (16 * WN * TN);
    hipLaunchKernelGGL((k_linear_tile<BF, ANY, WM, WN, WK, TM, TN, ST>), dim3(tm * tn, 1, a.groups),
                       dim3(64 * WM * WN * WK), 0, s, a, tm, tn);
    return hipGetLastError();
}

template <bool BF>
hipError_t launch_linear(const Args& a, hipStream_t s) {
    // 16-byte loads of whole pieces, 32-bit offsets within a tile
    const bool aligned = a.in_dim % 8 == 0 && a.x_stride % 8 == 0 && a.weight_stride % 8 == 0 && a.x_group % 8 == 0 &&
                         a.weight_group % 8 == 0 &&
                         (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.weight)) % 16 == 0 &&
                         std::max(a.x_stride, a.weight_stride) <= 1 << 20;
    const int f = choose(a);
    if (!aligned) switch (f) {
            case 0: return launch_tile<BF, true, 1, 1, 8, 1, 1, 2>(a, s);
            case 1: return launch_tile<BF, true, 1, 1, 8, 2, 2, 2>(a, s);
            case 2:
            case 3: return launch_tile<BF, true, 1, 2, 4, 4, 1, 2>(a, s);
            case 4:
            case 5: return launch_tile<BF, true, 2, 2, 2, 2, 2, 2>(a, s);
            default: return launch_tile<BF, true, 2, 4, 1, 4, 2, 2>(a, s);
        }
    switch (f) {
        case 0: return launch_tile<BF, false, 1, 1, 4, 1, 1, 8>(a, s);
        case 1: return launch_tile<BF, false, 1, 1, 4, 2, 2, 4>(a, s);
        case 2: return launch_tile<BF, false, 1, 1, 8, 4, 1, 4>(a, s);
        case 3: return launch_tile<BF, false, 1, 2, 4, 4, 1, 4>(a, s);
        case 4: return launch_tile<BF, false, 2, 2, 2, 2, 2, 4>(a, s);
        case 5: return launch_tile<BF, false, 2, 2, 4, 2, 2, 4>(a, s);
        case 6: return launch_tile<BF, false, 2, 4, 1, 4, 2, 4>(a, s);
        case 7: return launch_tile<BF, false, 2, 4, 1, 5, 2, 2>(a, s);
        default: return launch_tile<BF, false, 2, 4, 1, 8, 4, 2>(a, s);
    }
}

}  // namespace
}  // namespace hsamp

extern "C" int ultima_hsamp_linear(const ultima_hsamp_linear_args* a, void* hip_stream) {
    using namespace hsamp;
    if (a == nullptr || a->x == nullptr || a->weight == nullptr || a->out == nullptr) return ULTIMA_HSAMP_ERR_INVALID;
    if (a->out == a->x || a->out == a->weight || a->out == a->bias) return ULTIMA_HSAMP_ERR_INVALID;
    if (a->rows < 1 || a->in_dim < 1 || a->out_dim < 1 || a->groups < 1) return ULTIMA_HSAMP_ERR_INVALID;
    if (a->dtype != ULTIMA_HSAMP_BF16 && a->dtype != ULTIMA_HSAMP_F16) return ULTIMA_HSAMP_ERR_INVALID;
    if (a->out_dtype != a->dtype && a->out_dtype != ULTIMA_HSAMP_F32) return ULTIMA_HSAMP_ERR_INVALID;
    if (a->act < ULTIMA_HSAMP_ACT_NONE || a->act > ULTIMA_HSAMP_ACT_SOFTCAP) return ULTIMA_HSAMP_ERR_INVALID;
    if (a->act == ULTIMA_HSAMP_ACT_SOFTCAP && !(a->act_param > 0.0f && a->act_param <= 3.402823466e38f))
        return ULTIMA_HSAMP_ERR_INVALID;
    if (a->x_stride < a->in_dim || a->weight_stride < a->in_dim || a->out_stride < a->out_dim ||
        (a->residual != nullptr && a->residual_stride < a->out_dim))
        return ULTIMA_HSAMP_ERR_INVALID;
    const uintptr_t odd = reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->weight) |
                          reinterpret_cast<uintptr_t>(a->bias) | reinterpret_cast<uintptr_t>(a->residual);
    const uintptr_t os = a->out_dtype == ULTIMA_HSAMP_F32 ? 4 : 2;
    if (odd % 2 != 0 || reinterpret_cast<uintptr_t>(a->out) % os != 0) return ULTIMA_HSAMP_ERR_INVALID;
    // an output over its residual: the same place for every element, or none
    if (a->residual == a->out &&
        (a->out_dtype != a->dtype || a->residual_stride != a->out_stride ||
         (a->groups > 1 && a->residual_group != a->out_group)))
        return ULTIMA_HSAMP_ERR_INVALID;
    // the groups' outputs lie apart, one behind the other or side by side in each row
    const int64_t og = a->out_group < 0 ? -(a->out_group + 1) : a->out_group;
    if (a->groups > 1 && og / a->out_stride < a->rows &&
        og < (a->rows - 1) * a->out_stride + a->out_dim &&
        !(a->out_group >= a->out_dim && og < a->out_stride && (a->groups - 1) * og + a->out_dim <= a->out_stride))
        return ULTIMA_HSAMP_ERR_INVALID;
    // 32-bit rows and columns; a launch counts its threads in 32 bits
    if (a->groups > 65535 || std::max({a->rows, a->in_dim, a->out_dim}) > 1 << 30 ||
        std::max(blocks_of(kForms[choose(*a)], *a), blocks_of(kForms[6], *a)) > 1 << 22)
        return ULTIMA_HSAMP_ERR_UNSUPPORTED;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = a->dtype == ULTIMA_HSAMP_BF16 ? launch_linear<true>(*a, s) : launch_linear<false>(*a, s);
    return e == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}
