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

__device__ __forceinline__ float activate(float y, int act, float c) {
    switch (act) {
        case ULTIMA_HSAMP_ACT_RELU: return y < 0.0f ? 0.0f : y;       // (NaN stays)
        case ULTIMA_HSAMP_ACT_SILU: return y / (1.0f + expf(-y));
        case ULTIMA_HSAMP_ACT_GELU: return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
        case ULTIMA_HSAMP_ACT_GELU_TANH:
            return 0.5f * y * (1.0f + tanhf(0.79788456080286536f * (y + 0.044715f * y * y * y)));
        case ULTIMA_HSAMP_ACT_SOFTCAP: return c * tanhf(y / c);
        default: return y;
    }
}

using Args = ultima_hsamp_linear_args;

// One output from its finished sum.
template <bool BF>
__device__ __forceinline__ void finish(const Args& a, int g, int m, int n, float y) {
    if (a.bias != nullptr) y += to_f32<BF>(static_cast<const uint16_t*>(a.bias)[g * a.bias_group + n]);
    y = activate(y, a.act, a.act_param);
    if (a.residual != nullptr)
        y += to_f32<BF>(static_cast<const uint16_t*>(a.residual)[g * a.residual_group + m * a.residual_stride + n]);
    const int64_t at = g * a.out_group + m * a.out_stride + n;
    if (a.out_dtype == ULTIMA_HSAMP_F32) static_cast<float*>(a.out)[at] = y;
    else static_cast<uint16_t*>(a.out)[at] = from_f32<BF>(y);
}

// 64 x 64 outputs by four waves, 64 columns of x and W at a time through LDS.
template <bool BF>
__global__ __launch_bounds__(256) void k_linear(Args a) {
    constexpr int BK = 64, LS = BK + 8;
    __shared__ __attribute__((aligned(16))) uint16_t ws[64 * LS], xs[64 * LS];
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
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + wn + 16 * t + 4 * q + r, m = m0 + wm + 16 * s + i;
                if (n < a.out_dim && m < a.rows) finish<BF>(a, g, m, n, acc[t][s][r]);
            }
}

template <bool BF>
hipError_t launch_linear(const Args& a, hipStream_t s) {
    hipLaunchKernelGGL(k_linear<BF>, dim3((a.out_dim + 63) / 64, (a.rows + 63) / 64, a.groups), dim3(256), 0, s, a);
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
