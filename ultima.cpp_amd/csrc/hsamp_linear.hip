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

// 1 / (1 + exp(-t)); exp(-t) past the largest float is infinite, the result then 0.
__device__ __forceinline__ float sigmoid(float t) {
    return 1.0f / (1.0f + expf(-t));
}

using Args = ultima_hsamp_linear_args;

// E outputs (columns n .. n + E - 1 of row m, those there are) from their finished sums.
template <bool BF, int E>
__device__ __forceinline__ void finish(const Args& a, int g, int m, int n, float (&y)[E]) {
    typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
    const int left = a.out_dim - n;
    if (m >= a.rows || left <= 0) return;
    auto add = [&](const void* base, int64_t at) {
        const uint16_t* p = static_cast<const uint16_t*>(base) + at;
        if (E == 8 && left >= 8) {
            const u32x4 v = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] += to_f32<BF>((uint16_t)(v[e / 2 % 4] >> (16 * (e & 1))));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < left) y[e] += to_f32<BF>(p[e]);
        }
    };
    if (a.bias != nullptr) add(a.bias, g * a.bias_group + n);
    switch (a.act) {
        case ULTIMA_HSAMP_ACT_RELU:
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = y[e] < 0.0f ? 0.0f : y[e];       // (NaN stays)
            break;
        case ULTIMA_HSAMP_ACT_SILU:
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = y[e] * sigmoid(y[e]);
            break;
        case ULTIMA_HSAMP_ACT_GELU:
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = 0.5f * y[e] * (1.0f + erff(y[e] * 0.70710678118654752f));
            break;
        case ULTIMA_HSAMP_ACT_GELU_TANH:       // (1 + tanh(t)) / 2 = 1 / (1 + exp(-2 t))
#pragma unroll
            for (int e = 0; e < E; ++e)
                y[e] = y[e] * sigmoid(1.59576912160573071f * (y[e] + 0.044715f * y[e] * y[e] * y[e]));
            break;
        case ULTIMA_HSAMP_ACT_SOFTCAP:
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = a.act_param * tanhf(y[e] / a.act_param);
            break;
    }
    if (a.residual != nullptr) add(a.residual, g * a.residual_group + m * a.residual_stride + n);
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
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
#pragma unroll
    for (int u = 0; u < TM; ++u) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < TN; ++s) *reinterpret_cast<f32x4*>(&lds[i * LS + 16 * s + 4 * q]) = acc[s][u];
        __builtin_amdgcn_wave_barrier();
#pragma nounroll
        for (int o = lane; o < 16 * PR; o += 64) {
            const int r = o / PR, c = o % PR * 8;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(&lds[r * LS + c]);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(&lds[r * LS + c + 4]);
            float y[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            finish<BF, 8>(a, g, m0 + 16 * u + r, n0 + c, y);
        }
    }
}

// 64 x 64 outputs by four waves, 64 columns of x and W at a time through LDS.
template <bool BF>
__global__ __launch_bounds__(256) void k_linear(Args a) {
    constexpr int BK = 64, LS = BK + 8;
    __shared__ __attribute__((aligned(16))) uint16_t ws[64 * LS], xs[64 * LS];   // (ws: also 4 x 16 x 36 floats)
    static_assert(sizeof(ws) + 0 >= 4 * 16 * 36 * 4);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, q = lane >> 4;
    const int g = blockIdx.z, K = a.in_dim;
    const int n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
    const uint16_t* W = static_cast<const uint16_t*>(a.weight) + g * a.weight_group;
    const uint16_t* X = static_cast<const uint16_t*>(a.x) + g * a.x_group;
    // eight columns of a row, zeros past K and past the last row
    auto load = [&](const uint16_t* base, int64_t stride, int row, int rows, int k) {
        u32x4 v = {0, 0, 0, 0};
        if (row < rows) {
            const uint16_t* p = base + row * stride + k;
            if (k + 8 <= K) v = *reinterpret_cast<const u32x4_a2*>(p);
            else
                for (int e = 0; e < 8; ++e)
                    if (k + e < K) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
        }
        return v;
    };
    f32x4 acc[2][2] = {};
    const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
    for (int k0 = 0; k0 < K; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int c = tid + 256 * t, r = c >> 3, k = (c & 7) * 8;
            *reinterpret_cast<u32x4*>(&ws[r * LS + k]) = load(W, a.weight_stride, n0 + r, a.out_dim, k0 + k);
            *reinterpret_cast<u32x4*>(&xs[r * LS + k]) = load(X, a.x_stride, m0 + r, a.rows, k0 + k);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BK; k += 32) {
            u32x4 wf[2], xf[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                wf[t] = *reinterpret_cast<const u32x4*>(&ws[(wn + 16 * t + i) * LS + k + 8 * q]);
                xf[t] = *reinterpret_cast<const u32x4*>(&xs[(wm + 16 * t + i) * LS + k + 8 * q]);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int s = 0; s < 2; ++s) acc[t][s] = mfma<BF>(wf[t], xf[s], acc[t][s]);
        }
    }
    __syncthreads();
    store_tiles<BF, 2, 2>(a, g, m0 + wm, n0 + wn, acc, reinterpret_cast<float*>(ws) + wave * 16 * (32 + 4));
}

// Up to 16 NT rows of x: the weights' stream. Eight waves share 16 rows of W,
// each a part of the columns, from global memory straight into the operands'
// layout; their sums meet in LDS.
template <bool BF, int NT>
__global__ __launch_bounds__(512) void k_linear_rows(Args a) {
    constexpr int U = NT >= 4 ? 4 : 8;       // steps of 32 columns in flight, twice
    constexpr int NN = 16, MM = 16 * NT, LS = NN + 4;
    __shared__ __attribute__((aligned(16))) float part[8][MM * LS];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = blockIdx.z, K = a.in_dim, n0 = blockIdx.x * NN, m0 = blockIdx.y * MM;
    const uint16_t* wp = static_cast<const uint16_t*>(a.weight) + g * a.weight_group +
                         min(n0 + i, a.out_dim - 1) * a.weight_stride + 8 * q;
    const uint16_t* xp[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
        xp[t] = static_cast<const uint16_t*>(a.x) + g * a.x_group + min(m0 + 16 * t + i, a.rows - 1) * a.x_stride + 8 * q;
    f32x4 acc[NT] = {};
    const int steps = K / 32;
    const int s0 = (int)((int64_t)steps * wave / 8), s1 = (int)((int64_t)steps * (wave + 1) / 8);
    struct Group {
        u32x4 w[U], x[U][NT];
    };
    // (steps past the wave's last are loaded as its last and not multiplied)
    auto load = [&](Group& r, int s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = (int64_t)min(s + u, s1 - 1) * 32;
            r.w[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2*>(wp + k));
#pragma unroll
            for (int t = 0; t < NT; ++t) r.x[u][t] = *reinterpret_cast<const u32x4_a2*>(xp[t] + k);
        }
    };
    auto multiply = [&](const Group& r, int s) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u < s1)
#pragma unroll
                for (int v = 0; v < NT; ++v) acc[v] = mfma<BF>(r.w[u], r.x[u][v], acc[v]);
    };
    if (s0 < s1) {
        Group ra, rb;
        load(ra, s0);
        for (int s = s0; s < s1; s += 2 * U) {
            load(rb, s + U);
            __builtin_amdgcn_sched_barrier(0);
            multiply(ra, s);
            __builtin_amdgcn_sched_barrier(0);
            load(ra, s + 2 * U);
            __builtin_amdgcn_sched_barrier(0);
            multiply(rb, s + U);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // the columns past the last whole step
    if (wave == 7 && K % 32 != 0) {
        auto tail = [&](const uint16_t* p) {
            u32x4 v = {0, 0, 0, 0};
            for (int e = 0; e < 8; ++e)
                if (steps * 32 + 8 * q + e < K) v[e >> 1] |= (uint32_t)p[(int64_t)steps * 32 + e] << (16 * (e & 1));
            return v;
        };
        u32x4 xf[NT];
#pragma unroll
        for (int v = 0; v < NT; ++v) xf[v] = tail(xp[v]);
        const u32x4 wf = tail(wp);
#pragma unroll
        for (int v = 0; v < NT; ++v) acc[v] = mfma<BF>(wf, xf[v], acc[v]);
    }
#pragma unroll
    for (int v = 0; v < NT; ++v) *reinterpret_cast<f32x4*>(&part[wave][(16 * v + i) * LS + 4 * q]) = acc[v];
    __syncthreads();
    for (int o = tid; o < MM * NN; o += 512) {
        const int m = o / NN, n = o % NN;
        float y[1] = {};
#pragma unroll
        for (int w = 0; w < 8; ++w) y[0] += part[w][m * LS + n];
        finish<BF, 1>(a, g, m0 + m, n0 + n, y);
    }
}

// 16 WM TM rows of x by 16 WN TN rows of W by WM x WN x WK waves (WK of
// them sharing each tile's columns): global memory to LDS without registers, ST
// stages in the air or in LDS; the next step's operands are read while one is
// multiplied. A stage is 64 columns in two steps (WK = 1), or 32 WK columns, one
// step for each wave, whose sums meet in LDS at the end.
template <bool BF, int WM, int WN, int WK, int TM, int TN, int ST>
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
    static_assert((ST & (ST - 1)) == 0 && ST * SB * 2 >= EB * 4 && ST * SB * 2 <= 160 * 1024);
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
    int col[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int c = wave + NW * j, rc = c % CR, r = (rc < CX ? rc : rc - CX) * 8 + (lane >> 3);
        col[j] = c / CR * 64 + ((lane & 7) ^ (r >> 1 & 7)) * 8;
        const bool in = rc < CX ? m0 + r < a.rows : n0 + r < a.out_dim;
        vo[j] = in ? (uint32_t)(r * (int)(rc < CX ? a.x_stride : a.weight_stride) + col[j]) * 2u : kOutside;
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
#ifndef NOSB
        __builtin_amdgcn_sched_barrier(0);      // (and the reads ahead of the products)
#endif
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
        finish<BF, E>(a, g, m0 + m, n0 + n, y);
    }
#endif
}

// A form of k_linear_tile: its tile, how many blocks one CU holds, and what a
// round of one block per CU (one[0]) and of two (one[1]) costs, in us at
// K = 4096. Measured, N = 4096 and 16384 (bf16), rows 1 to 4096:
//   16 x 16 rows 1: 7.8, 25 us; 32 x 32 rows 32: 14.5, 26; 64 x 16 rows 64: 15, 56;
//   64 x 32 rows 64: 17.5, 37, rows 256: 31, 120; 64 x 64 rows 256: 34, 75, rows 512:
//   39, 133; 128 x 128 rows 256: 41, 56, rows 1024: 52, 168; 160 x 128 rows 512:
//   63, 83, rows 2048: 76, 284; 256 x 256 rows 1024: 101, 123, rows 4096 (f16): -, 462.
struct Form {
    int bm, bn, blocks;
    float one[2];
};
constexpr Form kForms[] = {
    {16, 16, 2, {8, 12}},   {32, 32, 2, {13, 25}},   {64, 16, 1, {14.5f, 0}}, {64, 32, 1, {15.5f, 0}},
    {64, 64, 2, {32, 39}},  {128, 128, 1, {44, 0}},  {160, 128, 2, {62, 84}}, {256, 256, 1, {112, 0}},
};

// The form whose rounds over the 256 CUs cost least.
int choose(const Args& a) {
    int best = 0;
    float least = 0;
    for (int f = 0; f < (int)(sizeof(kForms) / sizeof(kForms[0])); ++f) {
        const Form& v = kForms[f];
        const int64_t blocks = (int64_t)((a.rows + v.bm - 1) / v.bm) * ((a.out_dim + v.bn - 1) / v.bn) * a.groups;
        const int64_t round = 256 * v.blocks, rest = blocks % round;
        const float cost = (float)(blocks / round) * v.one[v.blocks - 1] +
                           (rest == 0 ? 0.0f : rest <= 256 ? v.one[0] : v.one[v.blocks - 1]);
        if (f == 0 || cost < least) {
            best = f;
            least = cost;
        }
    }
    return best;
}

template <bool BF>
hipError_t launch_linear(const Args& a, hipStream_t s) {
    const int M = a.rows, N = a.out_dim;
    using std::integral_constant;
    // 16-byte loads of every row, 32-bit offsets within a tile
    const bool tiles = a.in_dim % 8 == 0 && a.x_stride % 8 == 0 && a.weight_stride % 8 == 0 && a.x_group % 8 == 0 &&
                       a.weight_group % 8 == 0 &&
                       (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.weight)) % 16 == 0 &&
                       std::max(a.x_stride, a.weight_stride) <= 1 << 20;
    if (tiles) {
        auto go = [&](auto wm, auto wn, auto wk, auto tm, auto tn, auto st) {
            constexpr int WM = decltype(wm)::value, WN = decltype(wn)::value, WK = decltype(wk)::value;
            constexpr int TM = decltype(tm)::value, TN = decltype(tn)::value, ST = decltype(st)::value;
            const int tm_ = (M + 16 * WM * TM - 1) / (16 * WM * TM), tn_ = (N + 16 * WN * TN - 1) / (16 * WN * TN);
            hipLaunchKernelGGL((k_linear_tile<BF, WM, WN, WK, TM, TN, ST>), dim3(tm_ * tn_, 1, a.groups),
                               dim3(64 * WM * WN * WK), 0, s, a, tm_, tn_);
            return hipGetLastError();
        };
        constexpr integral_constant<int, 1> c1;
        constexpr integral_constant<int, 2> c2;
        constexpr integral_constant<int, 4> c4;
        constexpr integral_constant<int, 5> c5;
        constexpr integral_constant<int, 8> c8;
        switch (choose(a)) {
            case 0: return go(c1, c1, c4, c1, c1, c8);
            case 1: return go(c1, c1, c4, c2, c2, c4);
            case 2: return go(c1, c1, c8, c4, c1, c4);
            case 3: return go(c1, c2, c4, c4, c1, c4);
            case 4: return go(c2, c2, c2, c2, c2, c4);
            case 5: return go(c2, c4, c1, c4, c2, c4);
            case 6: return go(c2, c4, c1, c5, c2, c2);
            default: return go(c2, c4, c1, c8, c4, c2);
        }
    }
    auto rows = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        hipLaunchKernelGGL((k_linear_rows<BF, NT>), dim3((N + 15) / 16, (M + 16 * NT - 1) / (16 * NT), a.groups),
                           dim3(512), 0, s, a);
        return hipGetLastError();
    };
    if (M <= 16) return rows(integral_constant<int, 1>());
    if (M <= 128) return rows(integral_constant<int, 4>());
    hipLaunchKernelGGL(k_linear<BF>, dim3((N + 63) / 64, (M + 63) / 64, a.groups), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace hsamp

extern "C" int ultima_hsamp_linear(const ultima_hsamp_linear_args* a, void* hip_stream) {
    using namespace hsamp;
    if (a == nullptr || a->x == nullptr || a->weight == nullptr || a->out == nullptr) return ULTIMA_HSAMP_ERR_INVALID;
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
    // 32-bit columns, grid sizes
    if (a->groups > 65535 || a->rows >= 65535 * 64 || a->in_dim > 1 << 30 || a->out_dim > 1 << 30)
        return ULTIMA_HSAMP_ERR_UNSUPPORTED;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = a->dtype == ULTIMA_HSAMP_BF16 ? launch_linear<true>(*a, s) : launch_linear<false>(*a, s);
    return e == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}
