// geglu_train.hip — GEGLU y = a gelu(g) (exact erf form) on rows [a | g] with its gradient, the input kept for the backward as it is or in
// 8 bits (act8.h); fp16, bf16, float32. The feed-forward of a transformer block that trains; groupnorm.hip's k_geglu is the frozen form.
//   gelu(g) = g Phi(g);  da = dy gelu(g),  dg = dy a (Phi(g) + g phi(g))
// Elementwise and memory bound: forward reads 2 n and writes n values a row (+ 2 n bytes of codes), backward reads 2 n (or 2 n bytes) and
// n and writes 2 n. A thread takes 8 channels of a and the same 8 of g: 16-byte loads and stores.
// Measured, 8192 rows of 2 x 1280 fp16 with 8-bit input: 19.3 us forward and 19.0 backward, 85 MB each, 4.4 TB/s (a 2 GiB copy: 4.9).
#include "act8.h"

using namespace sdfx;

namespace {

__device__ __forceinline__ float normal_cdf(float g) { return 0.5f * (1.0f + erff(g * 0.70710678118654752f)); }

template <typename T, bool Q8>
__global__ __launch_bounds__(256) void k_geglu_fwd(const T* __restrict__ x, uint64_t rows, uint32_t nv, T* __restrict__ y, u2n* __restrict__ codes,
                                                  uint8_t* __restrict__ scales) {
    const uint64_t total = rows * nv;
    for (uint64_t v = (uint64_t)blockIdx.x * 256 + threadIdx.x; v < total; v += (uint64_t)gridDim.x * 256) {
        const uint64_t r = v / nv, ia = r * 2 * nv + (v - r * nv), ig = ia + nv;
        const Raw8<T> ra = load8(x + ia * 8), rg = load8(x + ig * 8);
        float a[8], g[8];
        widen(ra, a);
        widen(rg, g);
        if (Q8) {                             // (nv % 4 == 0: a quad's four vectors are one block of a, and one of g)
            uint32_t sa, sg;
            codes[ia] = encode8(a, sa);
            codes[ig] = encode8(g, sg);
            if ((threadIdx.x & 3u) == 0) { scales[ia >> 2] = (uint8_t)sa; scales[ig >> 2] = (uint8_t)sg; }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = a[i] * (g[i] * normal_cdf(g[i]));
        store8(y + v * 8, a);
    }
}

template <typename T, bool Q8>
__global__ __launch_bounds__(256) void k_geglu_bwd(const void* __restrict__ x, const uint8_t* __restrict__ scales, const T* __restrict__ dy, uint64_t rows,
                                                  uint32_t nv, T* __restrict__ dx) {
    const uint64_t total = rows * nv;
    for (uint64_t v = (uint64_t)blockIdx.x * 256 + threadIdx.x; v < total; v += (uint64_t)gridDim.x * 256) {
        const uint64_t r = v / nv, ia = r * 2 * nv + (v - r * nv), ig = ia + nv;
        const Saved<T, Q8> ra = load_saved<T, Q8>(x, scales, ia), rg = load_saved<T, Q8>(x, scales, ig);
        const Raw8<T> rd = load8(dy + v * 8);
        float a[8], g[8], d[8];
        widen_saved(ra, a);
        widen_saved(rg, g);
        widen(rd, d);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float cdf = normal_cdf(g[i]), pdf = 0.3989422804014327f * __expf(-0.5f * g[i] * g[i]);
            const float da = d[i] * (g[i] * cdf);
            g[i] = d[i] * a[i] * __builtin_fmaf(g[i], pdf, cdf);
            a[i] = da;
        }
        store8(dx + ia * 8, a);
        store8(dx + ig * 8, g);
    }
}

uint32_t grid_of(uint64_t total) { return (uint32_t)(total < 256ull * 16384 ? (total + 255) / 256 : 16384); }

template <typename T>
void fwd(const void* x, uint64_t rows, uint32_t n, void* y, uint8_t* saved, hipStream_t st) {
    const dim3 grid(grid_of(rows * (n / 8)));
    const T* xp = static_cast<const T*>(x);
    T* yp = static_cast<T*>(y);
    if (saved)
        hipLaunchKernelGGL((k_geglu_fwd<T, true>), grid, dim3(256), 0, st, xp, rows, n / 8, yp, reinterpret_cast<u2n*>(saved), saved + rows * 2 * n);
    else
        hipLaunchKernelGGL((k_geglu_fwd<T, false>), grid, dim3(256), 0, st, xp, rows, n / 8, yp, static_cast<u2n*>(nullptr), static_cast<uint8_t*>(nullptr));
}
template <typename T>
void bwd(const void* x, int eight, const void* dy, uint64_t rows, uint32_t n, void* dx, hipStream_t st) {
    const dim3 grid(grid_of(rows * (n / 8)));
    const T* dp = static_cast<const T*>(dy);
    T* xp = static_cast<T*>(dx);
    if (eight)
        hipLaunchKernelGGL((k_geglu_bwd<T, true>), grid, dim3(256), 0, st, x, static_cast<const uint8_t*>(x) + rows * 2 * n, dp, rows, n / 8, xp);
    else
        hipLaunchKernelGGL((k_geglu_bwd<T, false>), grid, dim3(256), 0, st, x, static_cast<const uint8_t*>(nullptr), dp, rows, n / 8, xp);
}

}  // namespace

extern "C" {

int sdfx_geglu_train_forward(const void* x, uint64_t rows, uint32_t n, int dtype, void* y, void* saved8, sdfx_stream_t stream) {
    if (rows == 0) return SDFX_OK;                   // (an empty tensor has no address)
    SDFX_REQUIRE(x && y, "geglu_train_forward: null pointer");
    SDFX_REQUIRE(dtype >= 0 && dtype <= 2, "geglu_train_forward: dtype %d (0 fp16, 1 bf16, 2 float32)", dtype);
    SDFX_REQUIRE(n > 0 && n % 8 == 0, "geglu_train_forward: n must be a positive multiple of 8 (got %u)", n);
    SDFX_REQUIRE(!saved8 || n % 32 == 0, "geglu_train_forward: the 8-bit form needs n %% 32 == 0 (got %u)", n);
    SDFX_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(saved8)) % 16) == 0,
                 "geglu_train_forward: misaligned pointer");
    uint8_t* sv = static_cast<uint8_t*>(saved8);
    hipStream_t st = as_stream(stream);
    if (dtype == 0) fwd<_Float16>(x, rows, n, y, sv, st);
    else if (dtype == 1) fwd<__bf16>(x, rows, n, y, sv, st);
    else fwd<float>(x, rows, n, y, sv, st);
    return check_launch("geglu_train_forward");
}

int sdfx_geglu_train_backward(const void* x, int eight_bits, const void* dy, uint64_t rows, uint32_t n, int dtype, void* dx, sdfx_stream_t stream) {
    if (rows == 0) return SDFX_OK;                   // (an empty tensor has no address)
    SDFX_REQUIRE(x && dy && dx, "geglu_train_backward: null pointer");
    SDFX_REQUIRE(dtype >= 0 && dtype <= 2, "geglu_train_backward: dtype %d (0 fp16, 1 bf16, 2 float32)", dtype);
    SDFX_REQUIRE(n > 0 && n % 8 == 0, "geglu_train_backward: n must be a positive multiple of 8 (got %u)", n);
    SDFX_REQUIRE(!eight_bits || n % 32 == 0, "geglu_train_backward: the 8-bit form needs n %% 32 == 0 (got %u)", n);
    SDFX_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx)) % 16) == 0,
                 "geglu_train_backward: misaligned pointer");
    hipStream_t st = as_stream(stream);
    if (dtype == 0) bwd<_Float16>(x, eight_bits, dy, rows, n, dx, st);
    else if (dtype == 1) bwd<__bf16>(x, eight_bits, dy, rows, n, dx, st);
    else bwd<float>(x, eight_bits, dy, rows, n, dx, st);
    return check_launch("geglu_train_backward");
}

}  // extern "C"
