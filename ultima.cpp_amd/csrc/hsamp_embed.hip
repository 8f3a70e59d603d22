// The embedding (ultima_hsamp_embed) and its gradient (ultima_hsamp_embed_grad).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "ultima_hsamp.h"

namespace hsamp {
namespace {

constexpr int N = 8;             // columns of one lane: 16 bytes of a 16-bit type
template <class T>
struct Eight {
    typedef T type __attribute__((ext_vector_type(N)));
};

// Eight values at any element's address; those past the row's end are not there.
template <class T>
__device__ __forceinline__ void load(const T* p, int left, float (&v)[N]) {
    typedef typename Eight<T>::type V;
    struct __attribute__((packed, aligned(sizeof(T)))) Any { V v; };
    if (left >= N) {
        const V t = reinterpret_cast<const Any*>(p)->v;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = e < left ? (float)p[e] : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store(T* p, int left, const float (&v)[N]) {
    typedef typename Eight<T>::type V;
    struct __attribute__((packed, aligned(sizeof(T)))) Any { V v; };
    if (left >= N) {
        V t;
#pragma unroll
        for (int e = 0; e < N; ++e) t[e] = (T)v[e];
        reinterpret_cast<Any*>(p)->v = t;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < left) p[e] = (T)v[e];
    }
}

// ---- The rows of the tokens -------------------------------------------------------
// A thread per eight columns of a token. Bound by the rows' reads and writes.
template <class T, class O>
__global__ __launch_bounds__(256) void k_embed(ultima_hsamp_embed_args a, int slices) {
    const int64_t i = blockIdx.x / slices;
    const int c = (blockIdx.x % slices * 256 + threadIdx.x) * N, left = a.width - c;
    if (left <= 0) return;
    const int id = a.ids[i];
    float v[N] = {};
    if (id >= 0 && id < a.vocab) {
        load(static_cast<const T*>(a.table) + id * a.table_stride + c, left, v);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= a.scale;
    }
    store(static_cast<O*>(a.out) + i * a.out_stride + c, left, v);
}

// ---- The gradient -------------------------------------------------------------------
// Positions sorted by id, each id's in order, then each id's rows added up: no atomics
// on sums, so that their order is the tokens' alone.
//
// The sort in one launch: a block owns a range of ids and looks at all of the tokens
// twice. What lies below its range is where its positions begin, so that no block waits
// for another; each of its waves counts and later places a run of consecutive tokens,
// wave after wave, 64 after 64, lane after lane. Its reads are the tokens (4 bytes each)
// once for each block, out of the caches.
struct Sorted {
    int32_t* start;      // [vocab + 1] where an id's positions begin
    int32_t* order;      // [tokens] the positions
};
constexpr int kWaves = 16, kRange = 1024;      // waves of a block; ids of one, at most

int ranges_of(int vocab) { return std::max((vocab + kRange - 1) / kRange, std::min(256, (vocab + 63) / 64)); }

__global__ __launch_bounds__(64 * kWaves) void k_sort_ids(const int32_t* ids, int tokens, int vocab, int range, Sorted out) {
    __shared__ int at[kWaves * kRange];     // a wave's tokens of an id, then where its next one goes
    __shared__ int below[kWaves], sums[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lo = blockIdx.x * range, hi = min(vocab, lo + range);
    for (int k = tid; k < kWaves * kRange; k += 64 * kWaves) at[k] = 0;
    __syncthreads();
    const int64_t per = ((int64_t)tokens + 64 * kWaves - 1) / (64 * kWaves) * 64;      // of one wave
    const int first = (int)min((int64_t)tokens, wave * per), last = (int)min((int64_t)tokens, (wave + 1) * per);
    int lower = 0;
    for (int k = first; k < last; k += 64) {
        const int id = k + lane < last ? ids[k + lane] : -1;
        lower += id >= 0 && id < lo;
        if (id >= lo && id < hi) atomicAdd(&at[wave * kRange + id - lo], 1);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) lower += __shfl_xor(lower, d);
    if (lane == 0) below[wave] = lower;
    __syncthreads();
    // a thread per id: its tokens, those of the ids before it, of the waves before
    int count = 0;
    for (int w = 0; w < kWaves; ++w) count += at[w * kRange + tid];
    int scan = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(scan, d);
        if (lane >= d) scan += v;
    }
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    int from = scan - count;
    for (int w = 0; w < kWaves; ++w) {
        from += below[w];
        if (w < wave) from += sums[w];
    }
    if (lo + tid < hi) {
        out.start[lo + tid] = from;
        if (lo + tid == vocab - 1) out.start[vocab] = from + count;
    }
    for (int w = 0; w < kWaves; ++w) {
        const int c = at[w * kRange + tid];
        at[w * kRange + tid] = from;
        from += c;
    }
    __syncthreads();
    for (int k = first; k < last; k += 64) {
        const int id = k + lane < last ? ids[k + lane] : -1;
        uint64_t todo = __ballot(id >= lo && id < hi);
        while (todo != 0) {          // once for each id there is among the 64
            const int leader = __builtin_ctzll(todo), which = __builtin_amdgcn_readlane(id, leader);
            const uint64_t same = __ballot(id == which);
            int next = 0;
            if (lane == leader) next = atomicAdd(&at[wave * kRange + which - lo], __popcll(same));
            next = __builtin_amdgcn_readlane(next, leader);
            if (id == which) out.order[next + __popcll(same & ((1ull << lane) - 1))] = k + lane;
            todo &= ~same;
        }
    }
}

// Chunks of `chunk` sorted positions that hold a single id are added up first, a block
// per chunk and 2048 columns, so that a frequent id's rows are read by many blocks.
int chunk_of(int tokens) { return std::max(64, (tokens + 1023) / 1024); }

template <class T>
__global__ __launch_bounds__(256) void k_embed_chunks(ultima_hsamp_embed_grad_args a, Sorted s, float* partial, int chunk, int slices) {
    const int c = (blockIdx.x % slices * 256 + threadIdx.x) * N, left = a.width - c;
    const int64_t at = blockIdx.x / slices, first = at * chunk;
    if (first + chunk > s.start[a.vocab]) return;
    if (a.ids[s.order[first]] != a.ids[s.order[first + chunk - 1]] || left <= 0) return;
    float sum[N] = {};
    for (int64_t k = first; k < first + chunk; ++k) {
        float v[N];
        load(static_cast<const T*>(a.d_out) + s.order[k] * a.d_out_stride + c, left, v);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += v[e];
    }
    const int64_t padded = (a.width + N - 1) / N * N;
    store(partial + at * padded + c, N, sum);
}

// A wave per id and 512 columns: the rows before its first whole chunk, the chunks, the
// rows behind them.
template <class T, class O>
__global__ __launch_bounds__(256) void k_embed_rows(ultima_hsamp_embed_grad_args a, Sorted s, const float* partial, int chunk, int slices) {
    const int64_t item = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    const int64_t id = item / slices;
    const int c = (int)(item % slices * 64 + threadIdx.x % 64) * N, left = a.width - c;
    if (id >= a.vocab || left <= 0) return;
    const int first = s.start[id], last = s.start[id + 1];
    O* out = static_cast<O*>(a.out) + id * a.out_stride + c;
    float sum[N] = {};
    if (first == last) {
        if (!a.accumulate) store(out, left, sum);
        return;
    }
    auto add = [&](int from, int to) {
        for (int k = from; k < to; ++k) {
            float v[N];
            load(static_cast<const T*>(a.d_out) + s.order[k] * a.d_out_stride + c, left, v);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += v[e];
        }
    };
    const int whole = (first + chunk - 1) / chunk, end = last / chunk;
    if (whole < end) {
        const int64_t padded = (a.width + N - 1) / N * N;
        add(first, whole * chunk);
        for (int64_t k = whole; k < end; ++k) {
            float v[N];
            load(partial + k * padded + c, N, v);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += v[e];
        }
        add(end * chunk, last);
    } else {
        add(first, last);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] *= a.scale;
    if (a.accumulate) {
        float v[N];
        load(out, left, v);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += v[e];
    }
    store(out, left, sum);
}

int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }

template <class T, class O>
hipError_t launch_grad(const ultima_hsamp_embed_grad_args& a, hipStream_t s) {
    char* work = static_cast<char*>(a.work);
    const Sorted sorted = {reinterpret_cast<int32_t*>(work), reinterpret_cast<int32_t*>(work + up16(4 * ((int64_t)a.vocab + 1)))};
    float* partial = reinterpret_cast<float*>(work + up16(4 * ((int64_t)a.vocab + 1)) + up16(4 * (int64_t)a.tokens));
    const int blocks = ranges_of(a.vocab), range = (a.vocab + blocks - 1) / blocks, chunk = chunk_of(a.tokens);
    hipLaunchKernelGGL(k_sort_ids, dim3((a.vocab + range - 1) / range), dim3(64 * kWaves), 0, s, a.ids, a.tokens, a.vocab, range, sorted);
    const int wide = (a.width + 2047) / 2048, slices = (a.width + 511) / 512;
    if (a.tokens >= chunk)
        hipLaunchKernelGGL(k_embed_chunks<T>, dim3(a.tokens / chunk * wide), dim3(256), 0, s, a, sorted, partial, chunk, wide);
    hipLaunchKernelGGL((k_embed_rows<T, O>), dim3((uint32_t)(((int64_t)a.vocab * slices + 3) / 4)), dim3(256), 0, s, a, sorted,
                       (const float*)partial, chunk, slices);
    return hipGetLastError();
}

template <class T, class O>
hipError_t launch_embed(const ultima_hsamp_embed_args& a, hipStream_t s) {
    const int slices = (a.width + 2047) / 2048;
    hipLaunchKernelGGL((k_embed<T, O>), dim3((uint32_t)((int64_t)a.tokens * slices)), dim3(256), 0, s, a, slices);
    return hipGetLastError();
}

uintptr_t size_of(int dtype) { return dtype == ULTIMA_HSAMP_F32 ? 4 : 2; }

// Sizes and types that both calls share.
int check_embed(int tokens, int width, int vocab, int dtype, int out_dtype) {
    if (tokens < 1 || width < 1 || vocab < 1 || vocab > ULTIMA_HSAMP_MAX_VOCAB) return ULTIMA_HSAMP_ERR_INVALID;
    if (dtype != ULTIMA_HSAMP_F32 && dtype != ULTIMA_HSAMP_BF16 && dtype != ULTIMA_HSAMP_F16) return ULTIMA_HSAMP_ERR_INVALID;
    if (out_dtype != dtype && out_dtype != ULTIMA_HSAMP_F32) return ULTIMA_HSAMP_ERR_INVALID;
    // 32-bit columns and positions; a launch counts its threads in 32 bits
    if (width > 1 << 24 || tokens > 1 << 30) return ULTIMA_HSAMP_ERR_UNSUPPORTED;
    if (((int64_t)width + 511) / 512 * std::max((int64_t)tokens, ((int64_t)vocab + 3) / 4) > (1 << 24) - 1)
        return ULTIMA_HSAMP_ERR_UNSUPPORTED;
    return ULTIMA_HSAMP_OK;
}

}  // namespace
}  // namespace hsamp

extern "C" int ultima_hsamp_embed(const ultima_hsamp_embed_args* a, void* hip_stream) {
    using namespace hsamp;
    if (a == nullptr || a->table == nullptr || a->ids == nullptr || a->out == nullptr) return ULTIMA_HSAMP_ERR_INVALID;
    if (a->out == a->table || a->out == static_cast<const void*>(a->ids)) return ULTIMA_HSAMP_ERR_INVALID;
    const int status = check_embed(a->tokens, a->width, a->vocab, a->dtype, a->out_dtype);
    if (status != ULTIMA_HSAMP_OK) return status;
    if (a->table_stride < a->width || a->out_stride < a->width) return ULTIMA_HSAMP_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(a->table) % size_of(a->dtype) != 0 || reinterpret_cast<uintptr_t>(a->out) % size_of(a->out_dtype) != 0 ||
        reinterpret_cast<uintptr_t>(a->ids) % 4 != 0)
        return ULTIMA_HSAMP_ERR_INVALID;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    hipError_t e;
    if (a->dtype == ULTIMA_HSAMP_F32) e = launch_embed<float, float>(*a, s);
    else if (a->dtype == ULTIMA_HSAMP_BF16) e = a->out_dtype == ULTIMA_HSAMP_F32 ? launch_embed<__bf16, float>(*a, s) : launch_embed<__bf16, __bf16>(*a, s);
    else e = a->out_dtype == ULTIMA_HSAMP_F32 ? launch_embed<_Float16, float>(*a, s) : launch_embed<_Float16, _Float16>(*a, s);
    return e == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}

extern "C" int64_t ultima_hsamp_embed_grad_work_bytes(int32_t tokens, int32_t width, int32_t vocab) {
    using namespace hsamp;
    if (tokens < 1 || width < 1 || vocab < 1 || vocab > ULTIMA_HSAMP_MAX_VOCAB) return -1;
    const int64_t padded = ((int64_t)width + N - 1) / N * N;
    return up16(4 * ((int64_t)vocab + 1)) + up16(4 * (int64_t)tokens) + tokens / chunk_of(tokens) * padded * 4;
}

extern "C" int ultima_hsamp_embed_grad(const ultima_hsamp_embed_grad_args* a, void* hip_stream) {
    using namespace hsamp;
    if (a == nullptr || a->d_out == nullptr || a->ids == nullptr || a->out == nullptr || a->work == nullptr) return ULTIMA_HSAMP_ERR_INVALID;
    if (a->out == a->d_out || a->out == static_cast<const void*>(a->ids) || a->out == a->work) return ULTIMA_HSAMP_ERR_INVALID;
    const int status = check_embed(a->tokens, a->width, a->vocab, a->dtype, a->out_dtype);
    if (status != ULTIMA_HSAMP_OK) return status;
    if (a->d_out_stride < a->width || a->out_stride < a->width) return ULTIMA_HSAMP_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(a->d_out) % size_of(a->dtype) != 0 || reinterpret_cast<uintptr_t>(a->out) % size_of(a->out_dtype) != 0 ||
        reinterpret_cast<uintptr_t>(a->ids) % 4 != 0 || reinterpret_cast<uintptr_t>(a->work) % 16 != 0)
        return ULTIMA_HSAMP_ERR_INVALID;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    hipError_t e;
    if (a->dtype == ULTIMA_HSAMP_F32) e = launch_grad<float, float>(*a, s);
    else if (a->dtype == ULTIMA_HSAMP_BF16) e = a->out_dtype == ULTIMA_HSAMP_F32 ? launch_grad<__bf16, float>(*a, s) : launch_grad<__bf16, __bf16>(*a, s);
    else e = a->out_dtype == ULTIMA_HSAMP_F32 ? launch_grad<_Float16, float>(*a, s) : launch_grad<_Float16, _Float16>(*a, s);
    return e == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}
