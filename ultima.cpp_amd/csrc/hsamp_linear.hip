// The product with its epilogue (ultima_hsamp_linear): out = act(x W^T + bias) +
// residual, 16-bit inputs on the matrix cores with float sums.
#include "hsamp_product.h"

namespace hsamp {
namespace {

template <bool BF>
struct Linear {
    static constexpr bool kByRows = false;
    using Args = ultima_hsamp_linear_args;
    using Element = uint16_t;
    using Sum = f32x4;
    using Columns = u32x4;      // eight columns' bias
    using Row = u32x4;          // eight values of the residual
    static __device__ __forceinline__ Sum mfma(u32x4 w, u32x4 x, Sum c) { return hsamp::mfma<BF>(w, x, c); }
    template <int E>
    static __device__ __forceinline__ Columns columns(const Args& a, int g, int n) {
        return E == 8 ? bias8(a, g, n) : u32x4{};
    }
    template <int E>
    static __device__ __forceinline__ Row row(const Args& a, int g, int m, int n) {
        return E == 8 ? residual8(a, g, m, n) : u32x4{};
    }
    template <int E>
    static __device__ __forceinline__ void finish(const Args& a, int g, int m, int n, float (&y)[E], Columns c, Row r) {
        hsamp::finish<BF, E>(a, g, m, n, y, c, r);
    }
    template <int TN, int TM, int WM, int WN>
    static __device__ __forceinline__ void tiles(const Args& a, int g, int m0, int n0, int wave, const Sum (&acc)[TN][TM], float* lds) {
        store_tiles<Linear, TN, TM>(a, g, m0 + wave % WM * 16 * TM, n0 + wave / WM % WN * 16 * TN, acc,
                                    lds + wave * 16 * (16 * TN + 4));
    }
};

}  // namespace
}  // namespace hsamp

extern "C" int ultima_hsamp_linear(const ultima_hsamp_linear_args* a, void* hip_stream) {
    using namespace hsamp;
    if (a == nullptr) return ULTIMA_HSAMP_ERR_INVALID;
    const int status = check_product(*a, 2);
    if (status != ULTIMA_HSAMP_OK) return status;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = a->dtype == ULTIMA_HSAMP_BF16 ? launch_product<Linear<true>>(*a, s) : launch_product<Linear<false>>(*a, s);
    return e == hipSuccess ? ULTIMA_HSAMP_OK : ULTIMA_HSAMP_ERR_HIP;
}
