// groupnorm_train.hip — GroupNorm (+ SiLU) on channels-last maps with every gradient: input, gamma, beta and the per-(sample, channel)
// vector `pre` added ahead of the norm; fp16, bf16 and float32 activations; the backward's copy of the input as it is or in 8 bits
// (act8.h). What a prior block needs when it trains; groupnorm.hip is the frozen fp16 form.
//   u = x + pre, xh = (u - mean) rstd, z = xh gamma + beta, y = silu(z) or z
//   dz = dy silu'(z), dbeta = sum dz, dgamma = sum dz xh, g = dz gamma, dx = rstd (g - mean(g) - xh mean(g xh)), dpre = sum over pixels of dx
// Memory bound: forward two reads and a write of the map (+ half a write of codes), backward two reads of x and dy and a write. With the
// 8-bit input the backward's reads of x halve.
//   forward   k_stats     per (sample, pixel slab): sums of d and d^2 per group, d = u - pivot, pivot = the group's first value: the
//                         difference E[d^2] - E[d]^2 stays accurate for a map whose mean is far from zero
//             k_finish    per (sample, group): slab partials combined in double -> mean, rstd
//             k_apply     y, and the 8-bit form of x
//   backward  k_bwd_stats per (sample, slab): sums of dz, dz xh (and xh, for dpre) per channel
//             k_bwd_finish  per (sample, group): over slabs, in double -> channel sums, the two means, and dpre from the same sums:
//                           sum over pixels of dx = rstd (gamma S_dz - n m1 - m2 S_xh)
//             k_bwd_apply dx; its first threads add the channel sums over samples: dgamma, dbeta
// No atomics: partials are combined in a fixed order, results are bit-reproducible.
#include "act8.h"

using namespace sdfx;

namespace {

constexpr uint32_t kMaxGroups = 64;
constexpr uint32_t kMaxThreads = 320;        // C / 8 <= 320 vectors per pixel
constexpr uint32_t kTrip = 4;                // pixels whose loads a thread issues together

struct Shape {
    uint32_t N, HW, C, G;
    uint32_t cpg, cvs;       // channels per group, 8-channel vectors per pixel
    uint32_t ppi, threads;   // pixels a workgroup covers at once; ppi * cvs rounded up to whole waves
    uint32_t slabs, P;       // workgroups per sample, pixels per slab
    float eps;
    int pf32;                // gamma / beta (and their gradients) are float32
};

bool make_shape(uint32_t N, uint32_t HW, uint32_t C, uint32_t G, Shape& s) {
    if (N == 0 || HW == 0 || C == 0 || G == 0 || G > kMaxGroups || C % G || C % 8 || C / 8 > kMaxThreads) return false;
    s.N = N; s.HW = HW; s.C = C; s.G = G;
    s.cpg = C / G; s.cvs = C / 8;
    s.ppi = s.cvs >= 256 ? 1u : 256u / s.cvs;
    s.threads = ((s.ppi * s.cvs + 63u) / 64u) * 64u;
    // whole trips; about 1024 workgroups on the largest maps (four a CU), one trip each on small ones
    const uint32_t trip = s.ppi * kTrip;
    const uint32_t most = max(1024u / N, 1u);
    uint32_t slabs = div_up(HW, trip);
    if (slabs > most) slabs = most;
    s.P = div_up(div_up(HW, slabs), trip) * trip;
    s.slabs = div_up(HW, s.P);
    s.eps = 0.f; s.pf32 = 0;
    return true;
}

// this thread's pixel within an iteration and its vector of the pixel; false for the idle tail of the last wave
__device__ __forceinline__ bool my_place(const Shape& s, uint32_t& pp, uint32_t& cv) {
    pp = threadIdx.x / s.cvs;
    cv = threadIdx.x - pp * s.cvs;
    return threadIdx.x < s.ppi * s.cvs;
}
template <typename T> __device__ __forceinline__ float pivot_of(const T* x, const T* pre, const Shape& s, uint32_t n, uint32_t g) {
    const float p = pre ? (float)pre[(size_t)n * s.C + g * s.cpg] : 0.f;
    return (float)x[(size_t)n * s.HW * s.C + g * s.cpg] + p;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// ---- forward --------------------------------------------------------------------------------------------------------------------
// partial[n][g][which][slab]
template <typename T>
__global__ __launch_bounds__(kMaxThreads) void k_stats(const T* __restrict__ x, const T* __restrict__ pre, Shape s, float* __restrict__ partial) {
    extern __shared__ float part[];          // [2][ppi][C], then [2][C]
    const uint32_t n = blockIdx.x / s.slabs, slab = blockIdx.x - n * s.slabs;
    uint32_t pp, cv;
    if (my_place(s, pp, cv)) {
        float e[8], sum[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sq[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t c = cv * 8 + i;
            e[i] = (pre ? (float)pre[(size_t)n * s.C + c] : 0.f) - pivot_of(x, pre, s, n, c / s.cpg);
        }
        const uint32_t p1 = min((slab + 1) * s.P, s.HW);
        const T* base = x + (size_t)n * s.HW * s.C + cv * 8;
        for (uint32_t p = slab * s.P + pp; p < p1; p += kTrip * s.ppi) {
            Raw8<T> v[kTrip];
#pragma unroll
            for (uint32_t u = 0; u < kTrip; u++) v[u] = load8(base + (size_t)min(p + u * s.ppi, p1 - 1) * s.C);
#pragma unroll
            for (uint32_t u = 0; u < kTrip; u++) {
                if (p + u * s.ppi >= p1) break;
                float f[8];
                widen(v[u], f);
#pragma unroll
                for (int i = 0; i < 8; i++) { const float d = f[i] + e[i]; sum[i] += d; sq[i] = __builtin_fmaf(d, d, sq[i]); }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            part[(size_t)pp * s.C + cv * 8 + i] = sum[i];
            part[(size_t)(s.ppi + pp) * s.C + cv * 8 + i] = sq[i];
        }
    }
    __syncthreads();
    float* chan = part + 2 * s.ppi * s.C;
    for (uint32_t k = threadIdx.x; k < 2 * s.C; k += s.threads) {
        const uint32_t which = k >= s.C, c = k - which * s.C;
        float a = 0.f;
        for (uint32_t p = 0; p < s.ppi; p++) a += part[(size_t)(which * s.ppi + p) * s.C + c];
        chan[k] = a;
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < 2 * s.G; k += s.threads) {
        const uint32_t which = k >= s.G, g = k - which * s.G;
        float a = 0.f;
        for (uint32_t c = 0; c < s.cpg; c++) a += chan[which * s.C + g * s.cpg + c];
        partial[(((size_t)n * s.G + g) * 2 + which) * s.slabs + slab] = a;
    }
}

// one wave per (sample, group)
template <typename T>
__global__ __launch_bounds__(64) void k_finish(const T* __restrict__ x, const T* __restrict__ pre, const float* __restrict__ partial, Shape s,
                                             float* __restrict__ mean_rstd) {
    const uint32_t n = blockIdx.x / s.G, g = blockIdx.x - n * s.G;
    const float* p = partial + (size_t)blockIdx.x * 2 * s.slabs;
    double a = 0.0, b = 0.0;
    for (uint32_t w = threadIdx.x; w < s.slabs; w += 64) { a += (double)p[w]; b += (double)p[s.slabs + w]; }
    a = wave_sum(a); b = wave_sum(b);
    if (threadIdx.x == 0) {
        const double cnt = (double)s.HW * s.cpg;
        a /= cnt; b /= cnt;
        double var = b - a * a;
        var = var > 0.0 || var != var ? var : 0.0;                 // (a NaN stays one)
        mean_rstd[(size_t)blockIdx.x * 2] = (float)((double)pivot_of(x, pre, s, n, g) + a);
        mean_rstd[(size_t)blockIdx.x * 2 + 1] = (float)(1.0 / sqrt(var + (double)s.eps));
    }
}

template <typename T, bool ACT, bool Q8>
__global__ __launch_bounds__(kMaxThreads) void k_apply(const T* __restrict__ x, const T* __restrict__ pre, Shape s, const float* __restrict__ mean_rstd,
                                                        const void* __restrict__ gamma, const void* __restrict__ beta, T* __restrict__ y,
                                                        u2n* __restrict__ codes, uint8_t* __restrict__ scales) {
    const uint32_t n = blockIdx.x / s.slabs, slab = blockIdx.x - n * s.slabs;
    uint32_t pp, cv;
    if (!my_place(s, pp, cv)) return;
    float mean[8], a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t c = cv * 8 + i, g = c / s.cpg;
        const float* mr = mean_rstd + ((size_t)n * s.G + g) * 2;
        mean[i] = mr[0] - (pre ? (float)pre[(size_t)n * s.C + c] : 0.f);
        a[i] = mr[1] * load_param<T>(gamma, c, s.pf32);
        b[i] = load_param<T>(beta, c, s.pf32);
    }
    const uint32_t p1 = min((slab + 1) * s.P, s.HW);
    const size_t at0 = (size_t)n * s.HW * s.cvs + cv;
    for (uint32_t p = slab * s.P + pp; p < p1; p += kTrip * s.ppi) {
        Raw8<T> v[kTrip];
#pragma unroll
        for (uint32_t u = 0; u < kTrip; u++) v[u] = load8(x + (at0 + (size_t)min(p + u * s.ppi, p1 - 1) * s.cvs) * 8);
#pragma unroll
        for (uint32_t u = 0; u < kTrip; u++) {
            if (p + u * s.ppi >= p1) break;
            const size_t at = at0 + (size_t)(p + u * s.ppi) * s.cvs;
            float f[8];
            widen(v[u], f);
            if (Q8) {
                uint32_t sc;
                codes[at] = encode8(f, sc);
                if ((cv & 3u) == 0) scales[at >> 2] = (uint8_t)sc;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float z = __builtin_fmaf(f[i] - mean[i], a[i], b[i]);
                f[i] = ACT ? z * fast_sigmoid(z) : z;
            }
            store8(y + at * 8, f);
        }
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------------
template <bool ACT> __device__ __forceinline__ float dz_of(float xh, float dy, float gamma, float beta) {
    if (!ACT) return dy;
    const float z = __builtin_fmaf(xh, gamma, beta), sg = fast_sigmoid(z);
    return dy * sg * __builtin_fmaf(z, 1.0f - sg, 1.0f);
}

// partial[n][which][c][slab], which: sum dz, sum dz xh and (with pre) sum xh
template <typename T, bool ACT, bool Q8>
__global__ __launch_bounds__(kMaxThreads) void k_bwd_stats(const void* __restrict__ x, const uint8_t* __restrict__ scales, const T* __restrict__ pre,
                                                            const T* __restrict__ dy, Shape s, const float* __restrict__ mean_rstd,
                                                            const void* __restrict__ gamma, const void* __restrict__ beta, float* __restrict__ partial) {
    extern __shared__ float part[];          // [3][ppi][C]
    const uint32_t n = blockIdx.x / s.slabs, slab = blockIdx.x - n * s.slabs;
    const uint32_t K = pre ? 3u : 2u;
    uint32_t pp, cv;
    if (my_place(s, pp, cv)) {
        float mean[8], rstd[8], ga[8], be[8], s1[8], s2[8], s3[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t c = cv * 8 + i, g = c / s.cpg;
            const float* mr = mean_rstd + ((size_t)n * s.G + g) * 2;
            mean[i] = mr[0] - (pre ? (float)pre[(size_t)n * s.C + c] : 0.f);
            rstd[i] = mr[1];
            ga[i] = load_param<T>(gamma, c, s.pf32);
            be[i] = load_param<T>(beta, c, s.pf32);
            s1[i] = s2[i] = s3[i] = 0.f;
        }
        const uint32_t p1 = min((slab + 1) * s.P, s.HW);
        const size_t at0 = (size_t)n * s.HW * s.cvs + cv;
        for (uint32_t p = slab * s.P + pp; p < p1; p += kTrip * s.ppi) {
            Saved<T, Q8> vx[kTrip];
            Raw8<T> vd[kTrip];
#pragma unroll
            for (uint32_t u = 0; u < kTrip; u++) {
                const size_t at = at0 + (size_t)min(p + u * s.ppi, p1 - 1) * s.cvs;
                vx[u] = load_saved<T, Q8>(x, scales, at);
                vd[u] = load8(dy + at * 8);
            }
#pragma unroll
            for (uint32_t u = 0; u < kTrip; u++) {
                if (p + u * s.ppi >= p1) break;
                float fx[8], fd[8];
                widen_saved(vx[u], fx);
                widen(vd[u], fd);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float xh = (fx[i] - mean[i]) * rstd[i], dz = dz_of<ACT>(xh, fd[i], ga[i], be[i]);
                    s1[i] += dz;
                    s2[i] = __builtin_fmaf(dz, xh, s2[i]);
                    s3[i] += xh;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const size_t c = cv * 8 + i;
            part[(size_t)pp * s.C + c] = s1[i];
            part[(size_t)(s.ppi + pp) * s.C + c] = s2[i];
            if (pre) part[(size_t)(2 * s.ppi + pp) * s.C + c] = s3[i];
        }
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < K * s.C; k += s.threads) {
        const uint32_t which = k / s.C, c = k - which * s.C;
        float a = 0.f;
        for (uint32_t p = 0; p < s.ppi; p++) a += part[(size_t)(which * s.ppi + p) * s.C + c];
        partial[(((size_t)n * K + which) * s.C + c) * s.slabs + slab] = a;
    }
}

// One workgroup per (sample, group), one wave per (which, channel) in turn: means[n][g][2], the channel sums chan[n][2][C] and dpre.
constexpr uint32_t kFinishThreads = 512;
template <typename T>
__global__ __launch_bounds__(kFinishThreads) void k_bwd_finish(const float* __restrict__ partial, Shape s, const float* __restrict__ mean_rstd,
                                                              const T* __restrict__ pre, const void* __restrict__ gamma, float* __restrict__ means,
                                                              double* __restrict__ chan, T* __restrict__ dpre) {
    extern __shared__ double sums[];          // [K][cpg]
    __shared__ double mom[2];
    const uint32_t n = blockIdx.x / s.G, g = blockIdx.x - n * s.G, K = pre ? 3u : 2u, items = K * s.cpg;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t k = wave; k < items; k += kFinishThreads / 64) {
        const uint32_t which = k / s.cpg, c = g * s.cpg + (k - which * s.cpg);
        const float* p = partial + (((size_t)n * K + which) * s.C + c) * s.slabs;
        double a = 0.0;
        for (uint32_t w = lane; w < s.slabs; w += 64) a += (double)p[w];
        a = wave_sum(a);
        if (lane == 0) {
            sums[k] = a;
            if (which < 2) chan[((size_t)n * 2 + which) * s.C + c] = a;
        }
    }
    __syncthreads();
    if (wave < 2) {                           // m1 = mean(g), m2 = mean(g xh)
        double m = 0.0;
        for (uint32_t c = lane; c < s.cpg; c += 64) m += sums[wave * s.cpg + c] * (double)load_param<T>(gamma, g * s.cpg + c, s.pf32);
        m = wave_sum(m) / ((double)s.HW * s.cpg);
        if (lane == 0) {
            mom[wave] = m;
            means[(size_t)blockIdx.x * 2 + wave] = (float)m;
        }
    }
    if (!dpre) return;
    __syncthreads();
    const double rstd = (double)mean_rstd[(size_t)blockIdx.x * 2 + 1];
    for (uint32_t k = threadIdx.x; k < s.cpg; k += kFinishThreads) {
        const uint32_t c = g * s.cpg + k;
        const double ga = (double)load_param<T>(gamma, c, s.pf32);
        dpre[(size_t)n * s.C + c] = (T)(float)(rstd * (ga * sums[k] - (double)s.HW * mom[0] - mom[1] * sums[2 * s.cpg + k]));
    }
}

// dx, and (the first threads of the grid) dgamma / dbeta: the channel sums over samples in order. dx / dgamma / dbeta may be null.
template <typename T, bool ACT, bool Q8>
__global__ __launch_bounds__(kMaxThreads) void k_bwd_apply(const void* __restrict__ x, const uint8_t* __restrict__ scales, const T* __restrict__ pre,
                                                            const T* __restrict__ dy, Shape s, const float* __restrict__ mean_rstd,
                                                            const float* __restrict__ means, const double* __restrict__ chan,
                                                            const void* __restrict__ gamma, const void* __restrict__ beta, T* __restrict__ dx,
                                                            void* __restrict__ dgamma, void* __restrict__ dbeta) {
    if (dgamma || dbeta) {
        for (uint32_t c = blockIdx.x * blockDim.x + threadIdx.x; c < s.C; c += gridDim.x * blockDim.x) {
            double b = 0.0, g = 0.0;
            for (uint32_t n = 0; n < s.N; n++) { b += chan[(size_t)n * 2 * s.C + c]; g += chan[((size_t)n * 2 + 1) * s.C + c]; }
            if (dbeta) store_param<T>(dbeta, c, s.pf32, b);
            if (dgamma) store_param<T>(dgamma, c, s.pf32, g);
        }
    }
    if (!dx) return;
    const uint32_t n = blockIdx.x / s.slabs, slab = blockIdx.x - n * s.slabs;
    uint32_t pp, cv;
    if (!my_place(s, pp, cv)) return;
    float mean[8], rstd[8], ga[8], be[8], m1[8], m2[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t c = cv * 8 + i, g = c / s.cpg;
        const size_t k = ((size_t)n * s.G + g) * 2;
        mean[i] = mean_rstd[k] - (pre ? (float)pre[(size_t)n * s.C + c] : 0.f);
        rstd[i] = mean_rstd[k + 1];
        ga[i] = load_param<T>(gamma, c, s.pf32);
        be[i] = load_param<T>(beta, c, s.pf32);
        m1[i] = means[k]; m2[i] = means[k + 1];
    }
    const uint32_t p1 = min((slab + 1) * s.P, s.HW);
    const size_t at0 = (size_t)n * s.HW * s.cvs + cv;
    for (uint32_t p = slab * s.P + pp; p < p1; p += kTrip * s.ppi) {
        Saved<T, Q8> vx[kTrip];
        Raw8<T> vd[kTrip];
#pragma unroll
        for (uint32_t u = 0; u < kTrip; u++) {
            const size_t at = at0 + (size_t)min(p + u * s.ppi, p1 - 1) * s.cvs;
            vx[u] = load_saved<T, Q8>(x, scales, at);
            vd[u] = load8(dy + at * 8);
        }
#pragma unroll
        for (uint32_t u = 0; u < kTrip; u++) {
            if (p + u * s.ppi >= p1) break;
            float fx[8], fd[8];
            widen_saved(vx[u], fx);
            widen(vd[u], fd);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float xh = (fx[i] - mean[i]) * rstd[i], dz = dz_of<ACT>(xh, fd[i], ga[i], be[i]);
                fx[i] = rstd[i] * (__builtin_fmaf(dz, ga[i], -m1[i]) - xh * m2[i]);
            }
            store8(dx + (at0 + (size_t)(p + u * s.ppi) * s.cvs) * 8, fx);
        }
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
uint64_t partial_floats(const Shape& s) { return (uint64_t)s.N * 3 * s.C * s.slabs; }

template <typename T, bool ACT, bool Q8>
void forward(const void* x_, const void* pre_, const void* gamma, const void* beta, const Shape& s, void* y, uint8_t* saved, float* mean_rstd,
             float* scratch, hipStream_t st) {
    const T *x = static_cast<const T*>(x_), *pre = static_cast<const T*>(pre_);
    hipLaunchKernelGGL(k_stats<T>, dim3(s.N * s.slabs), dim3(s.threads), (2 * s.ppi + 2) * s.C * 4, st, x, pre, s, scratch);
    hipLaunchKernelGGL(k_finish<T>, dim3(s.N * s.G), dim3(64), 0, st, x, pre, scratch, s, mean_rstd);
    hipLaunchKernelGGL((k_apply<T, ACT, Q8>), dim3(s.N * s.slabs), dim3(s.threads), 0, st, x, pre, s, mean_rstd, gamma, beta, static_cast<T*>(y),
                       reinterpret_cast<u2n*>(saved), saved + (size_t)s.N * s.HW * s.C);
}
template <typename T, bool ACT, bool Q8>
void backward(const void* x, const void* pre_, const void* dy_, const void* gamma, const void* beta, const float* mean_rstd, const Shape& s,
              void* dx, void* dpre, void* dgamma, void* dbeta, float* scratch, hipStream_t st) {
    const T *pre = static_cast<const T*>(pre_), *dy = static_cast<const T*>(dy_);
    const uint8_t* scales = Q8 ? static_cast<const uint8_t*>(x) + (size_t)s.N * s.HW * s.C : nullptr;
    float* means = scratch + partial_floats(s);
    double* chan = reinterpret_cast<double*>(means + (size_t)s.N * s.G * 2);          // (partial_floats is a multiple of 8)
    const uint32_t K = pre ? 3 : 2;
    hipLaunchKernelGGL((k_bwd_stats<T, ACT, Q8>), dim3(s.N * s.slabs), dim3(s.threads), K * s.ppi * s.C * 4, st, x, scales, pre, dy, s, mean_rstd,
                       gamma, beta, scratch);
    hipLaunchKernelGGL(k_bwd_finish<T>, dim3(s.N * s.G), dim3(kFinishThreads), K * s.cpg * 8, st, scratch, s, mean_rstd, pre, gamma, means, chan,
                       static_cast<T*>(dpre));
    if (dx || dgamma || dbeta)
        hipLaunchKernelGGL((k_bwd_apply<T, ACT, Q8>), dim3(s.N * s.slabs), dim3(s.threads), 0, st, x, scales, pre, dy, s, mean_rstd, means, chan, gamma,
                           beta, static_cast<T*>(dx), dgamma, dbeta);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

#define SDFX_GN_DISPATCH(fn, ...)                                                                              \
    do {                                                                                                       \
        const int key = dtype * 4 + (silu ? 2 : 0) + (eight ? 1 : 0);                                          \
        switch (key) {                                                                                         \
            case 0: fn<_Float16, false, false>(__VA_ARGS__); break;                                            \
            case 1: fn<_Float16, false, true>(__VA_ARGS__); break;                                             \
            case 2: fn<_Float16, true, false>(__VA_ARGS__); break;                                             \
            case 3: fn<_Float16, true, true>(__VA_ARGS__); break;                                              \
            case 4: fn<__bf16, false, false>(__VA_ARGS__); break;                                              \
            case 5: fn<__bf16, false, true>(__VA_ARGS__); break;                                               \
            case 6: fn<__bf16, true, false>(__VA_ARGS__); break;                                               \
            case 7: fn<__bf16, true, true>(__VA_ARGS__); break;                                                \
            case 8: fn<float, false, false>(__VA_ARGS__); break;                                               \
            case 9: fn<float, false, true>(__VA_ARGS__); break;                                                \
            case 10: fn<float, true, false>(__VA_ARGS__); break;                                               \
            default: fn<float, true, true>(__VA_ARGS__); break;                                                \
        }                                                                                                      \
    } while (0)

}  // namespace

extern "C" {

uint64_t sdfx_group_norm_train_scratch_bytes(uint32_t N, uint32_t HW, uint32_t C, uint32_t G) {
    Shape s;
    if (!make_shape(N, HW, C, G, s)) return 0;
    return (partial_floats(s) + (uint64_t)N * G * 2) * sizeof(float) + (uint64_t)N * 2 * C * sizeof(double);
}

int sdfx_group_norm_train_forward(const void* x, const void* pre, const void* gamma, const void* beta, uint32_t N, uint32_t HW, uint32_t C, uint32_t G,
                                  float eps, int silu, int dtype, int params_f32, void* y, void* saved8, float* mean_rstd, float* scratch,
                                  sdfx_stream_t stream) {
    SDFX_REQUIRE(x && gamma && beta && y && mean_rstd && scratch, "group_norm_train_forward: null pointer");
    SDFX_REQUIRE(dtype >= 0 && dtype <= 2, "group_norm_train_forward: dtype %d (0 fp16, 1 bf16, 2 float32)", dtype);
    Shape s;
    SDFX_REQUIRE(make_shape(N, HW, C, G, s), "group_norm_train_forward: needs C %% 8 == 0, C %% G == 0, C <= %u, G <= %u (got N=%u HW=%u C=%u G=%u)",
                 kMaxThreads * 8, kMaxGroups, N, HW, C, G);
    SDFX_REQUIRE(!saved8 || C % 32 == 0, "group_norm_train_forward: the 8-bit form needs C %% 32 == 0 (got %u)", C);
    SDFX_REQUIRE(aligned16(x) && aligned16(y) && aligned16(saved8), "group_norm_train_forward: x / y / saved8 misaligned");
    SDFX_REQUIRE(eps >= 0.f, "group_norm_train_forward: negative eps");
    s.eps = eps; s.pf32 = params_f32 || dtype == 2;
    const bool eight = saved8 != nullptr;
    SDFX_GN_DISPATCH(forward, x, pre, gamma, beta, s, y, static_cast<uint8_t*>(saved8), mean_rstd, scratch, as_stream(stream));
    return check_launch("group_norm_train_forward");
}

int sdfx_group_norm_train_backward(const void* x, int eight_bits, const void* pre, const void* dy, const void* gamma, const void* beta,
                                   const float* mean_rstd, uint32_t N, uint32_t HW, uint32_t C, uint32_t G, int silu, int dtype, int params_f32, void* dx,
                                   void* dpre, void* dgamma, void* dbeta, float* scratch, sdfx_stream_t stream) {
    SDFX_REQUIRE(x && dy && gamma && beta && mean_rstd && scratch, "group_norm_train_backward: null pointer");
    SDFX_REQUIRE(dtype >= 0 && dtype <= 2, "group_norm_train_backward: dtype %d (0 fp16, 1 bf16, 2 float32)", dtype);
    Shape s;
    SDFX_REQUIRE(make_shape(N, HW, C, G, s), "group_norm_train_backward: needs C %% 8 == 0, C %% G == 0, C <= %u, G <= %u (got N=%u HW=%u C=%u G=%u)",
                 kMaxThreads * 8, kMaxGroups, N, HW, C, G);
    SDFX_REQUIRE(!eight_bits || C % 32 == 0, "group_norm_train_backward: the 8-bit form needs C %% 32 == 0 (got %u)", C);
    SDFX_REQUIRE(pre || !dpre, "group_norm_train_backward: dpre without pre");
    SDFX_REQUIRE(aligned16(x) && aligned16(dy) && aligned16(dx), "group_norm_train_backward: x / dy / dx misaligned");
    s.pf32 = params_f32 || dtype == 2;
    const bool eight = eight_bits != 0;
    SDFX_GN_DISPATCH(backward, x, pre, dy, gamma, beta, mean_rstd, s, dx, dpre, dgamma, dbeta, scratch, as_stream(stream));
    return check_launch("group_norm_train_backward");
}

}  // extern "C"
