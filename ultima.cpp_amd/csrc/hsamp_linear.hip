// The product with its epilogue (ultima_hsamp_linear): out = act(x W^T + bias) +
// residual, 16-bit inputs on the matrix cores with float sums.
#include "hsamp_product.h"

namespace hsamp {
namespace {

template <bool BF>
struct Linear : RowsOfK<ultima_hsamp_linear_args, uint16_t> {
    static constexpr bool kByRows = false;
    static constexpr int kBand = 0;      // (tiles on the XCDs that they were on: the same bits)
    using Args = ultima_hsamp_linear_args;
    using Sum = f32x4;
    using Columns = u32x4;      // a piece of the bias
    using Row = u32x4;          // a piece of the residual
    static __device__ __forceinline__ Sum mfma(u32x4 w, u32x4 x, Sum c) { return hsamp::mfma<BF>(w, x, c); }
    template <int E>
    static __device__ __forceinline__ Columns columns(const Args& a, int g, int n) {
        return bias_piece<E>(a, g, n);
    }
    template <int E>
    static __device__ __forceinline__ Row row(const Args& a, int g, int m, int n) {
        return residual_piece<E>(a, g, m, n);
    }
    template <int E, int ACT = kAnyAct, bool WHOLE = false>
    static __device__ __forceinline__ void finish(const Args& a, int g, int m, int n, float (&y)[E], Columns c, Row r) {
        hsamp::finish<BF, E, ACT, WHOLE>(a, g, m, n, y, c, r);
    }
    template <int TN, int TM, int WM, int WN, int PU>
    static __device__ __forceinline__ void tiles(const Args& a, int g, int m0, int n0, int wave, const Sum (&acc)[TN][TM], float* lds) {
        by_act(a.act, [&](auto act) {
            store_tiles<Linear, decltype(act)::value, TN, TM, PU>(a, g, m0 + wave % WM * 16 * TM, n0 + wave / WM % WN * 16 * TN, acc, lds + wave * 256 * PU * TN);
        });
    }
    template <int TN, int TM>
    static __device__ __forceinline__ void wide(const Args& a, int g, int m0, int n0, const Sum (&acc)[TN][TM], uint16_t* lds) {
        by_act(a.act, [&](auto act) { store_sixteens<Linear, decltype(act)::value>(a, g, m0, n0, acc, lds); });
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
