// groupnorm_train.hip — GroupNorm (+ SiLU) on channels-last maps with every gradient: input, gamma, beta and the per-(sample, channel)
// vector `pre` added ahead of the norm; fp16, bf16 and float32 activations; the backward's copy of the input as it is or in 8 bits
// (act8.h). What a prior block needs when it trains; groupnorm.hip is the frozen fp16 form.
//   u = x + pre, xh = (u - mean) rstd, z = xh gamma + beta, y = silu(z) or z
// In float32 xh is (u - mean) rstd, an operation at a time; in 16 bits, whose own step hides it, an affine map of x (an operation less each way:
// mean rstd and the products with gamma round apart from x's).
//   dz = dy silu'(z), dbeta = sum dz, dgamma = sum dz xh, g = dz gamma, dx = rstd (g - mean(g) - xh mean(g xh)), dpre = sum over pixels of dx
// Memory bound: forward two reads and a write of the map (+ half a write of codes), backward two reads of x and dy and a write. With the
// 8-bit input the backward's reads of x halve.
//   forward   k_stats     per (sample, pixel slab): sums of d and d^2 per group, d = u - pivot, pivot = the group's first value, in double:
//                         E[d^2] - E[d]^2 loses (mean of d / deviation)^2 of 2^-53. That ratio is 0 for a constant map wherever it lies, and
//                         at most the root of the group's size where the first value is an outlier (whose own square is in the deviation).
//                         In float32 such an outlier cost 3 to 5 digits of rstd; double's fma runs at float32's rate here
//             k_finish    per (sample, group): slab partials combined in double -> mean, rstd. Up to kInlineSlabs slabs a sample every
//                         workgroup of k_apply combines them itself (one launch less; at most 64 KB out of L2 each)
//             k_apply     y, and the 8-bit form of x
//   backward  k_bwd_stats per (sample, slab): sums of dz, dz xh (and xh, for dpre) per channel
//                         and of g, g xh per group
//             k_bwd_finish  per (sample, group): the two means, in double; inline like k_finish
//             k_bwd_apply dx; then its waves take channels in turn: the sums over slabs and samples, in double -> dgamma, dbeta, and dpre
//                         from the same sums: sum over pixels of dx = rstd (gamma S_dz - n m1 - m2 S_xh)
// No atomics: partials are combined in a fixed order, results are bit-reproducible.
// Measured, 512 x 512 x 128 fp16 with 8-bit input: k_stats 17 us (3.8 TB/s; float32 sums took 16), k_apply 29 (5.9), k_bwd_stats 29 (3.5: it decodes and
// takes two transcendentals a value), k_bwd_apply 32 (5.2); each finish 7. Maps of the UNet's lower levels end at launches: 64 x 64 x 320,
// four kernels, 42 us in all, beside 81 us of host time for both ways.
#include "act8.h"

using namespace sdfx;

namespace {

constexpr uint32_t kMaxGroups = 64;
constexpr uint32_t kMaxThreads = 320;        // C / 8 <= 320 vectors per pixel
constexpr uint32_t kTrip = 4;                // pixels whose loads a thread issues together
constexpr uint32_t kInlineSlabs = 256;       // slabs a sample up to which every consumer combines them itself

struct Shape {
    uint32_t N, HW, C, G;
    uint32_t cpg, cvs;       // channels per group, 8-channel vectors per pixel
    uint32_t ppi, threads;   // pixels a workgroup covers at once; ppi * cvs rounded up to whole waves
    uint32_t slabs, P;       // workgroups per sample, pixels per slab
    float eps;
    int pf32;                // gamma / beta (and their gradients) are float32
    int inl;                 // the consumers combine the slabs' sums themselves
    uint32_t lanes;          // lanes that add a channel's slabs (a power of two)
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
    if ((uint64_t)N * s.slabs * kMaxThreads >= 1ull << 32) return false;               // (threads of a launch)
    s.inl = s.slabs <= kInlineSlabs;
    s.lanes = 1;
    while (s.lanes < 64 && s.lanes * 4 < s.slabs) s.lanes *= 2;
    return true;
}

// this thread's pixel within an iteration and its vector of the pixel; false for the idle tail of the last wave
__device__ __forceinline__ bool my_place(const Shape& s, uint32_t& pp, uint32_t& cv) {
    pp = threadIdx.x / s.cvs;
    cv = threadIdx.x - pp * s.cvs;
    return threadIdx.x < s.ppi * s.cvs;
}
// the groups of a thread's 8 channels, and a walk through them
struct GroupWalk {
    uint32_t g, r;
    __device__ __forceinline__ GroupWalk(const Shape& s, uint32_t c) : g(c / s.cpg), r(c - g * s.cpg) {}
    __device__ __forceinline__ void next(const Shape& s) { if (++r == s.cpg) { r = 0; g++; } }
};
template <typename T> __device__ __forceinline__ double pivot_of(const T* x, const T* pre, const Shape& s, uint32_t n, uint32_t g) {
    const double p = pre ? (double)(float)pre[(size_t)n * s.C + g * s.cpg] : 0.0;
    return (double)(float)x[(size_t)n * s.HW * s.C + g * s.cpg] + p;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// Slab partials of the groups' two sums: item k = 2 g + which of slab w at k * item + w * slab behind the sample's first. Combined inline they
// lie slab by slab (a workgroup reads whole rows), for the finish kernels item by item (a wave reads one item's).
struct Partials { uint32_t item, slab; };
__host__ __device__ inline Partials partials_of(const Shape& s) { return s.inl ? Partials{1u, 2u * s.G} : Partials{s.slabs, 1u}; }

// every workgroup's own combination: sums[2 G] in LDS (doubles), scr LDS doubles [threads]; the same order in every workgroup
template <typename P> __device__ __forceinline__ void combine_inline(const Shape& s, const P* __restrict__ partial, double* scr, double* sums) {
    const uint32_t K = 2 * s.G, J = s.threads >= K ? s.threads / K : 1u;
    for (uint32_t k0 = 0; k0 < K; k0 += s.threads) {                      // (one round unless the workgroup has fewer threads than items)
        const uint32_t j = threadIdx.x / (K < s.threads ? K : s.threads), k = k0 + threadIdx.x - j * (K < s.threads ? K : s.threads);
        double a = 0.0;
        if (j < J && k < K) {
            for (uint32_t w = j; w < s.slabs; w += 8 * J) {                // eight partials a trip, loaded together
                P v[8];
#pragma unroll
                for (uint32_t u = 0; u < 8; u++) v[u] = partial[(size_t)min(w + u * J, s.slabs - 1) * K + k];
#pragma unroll
                for (uint32_t u = 0; u < 8; u++)
                    if (w + u * J < s.slabs) a += (double)v[u];
            }
        }
        scr[threadIdx.x] = a;
        __syncthreads();
        if (j == 0 && k < K) {
            for (uint32_t i = 1; i < J; i++) a += scr[threadIdx.x + i * K];
            sums[k] = a;
        }
        __syncthreads();
    }
}
template <typename T>
__device__ __forceinline__ void moments(const Shape& s, const T* x, const T* pre, uint32_t n, uint32_t g, double a, double b, float& mean, float& rstd) {
    const double cnt = (double)s.HW * s.cpg;
    a /= cnt; b /= cnt;
    double var = b - a * a;
    var = var > 0.0 || var != var ? var : 0.0;                             // (a NaN stays one)
    mean = (float)(pivot_of(x, pre, s, n, g) + a);
    rstd = (float)(1.0 / sqrt(var + (double)s.eps));
}

// ---- forward --------------------------------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kMaxThreads) void k_stats(const T* __restrict__ x, const T* __restrict__ pre, Shape s, double* __restrict__ partial) {
    extern __shared__ double sums[];         // [2][ppi][C]; the sums over ppi end in the first of it
    const uint32_t n = blockIdx.x / s.slabs, slab = blockIdx.x - n * s.slabs;
    uint32_t pp, cv;
    if (my_place(s, pp, cv)) {
        float f0[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        double e[8], sum[8], sq[8];
        if (pre) widen(load8(pre + (size_t)n * s.C + cv * 8), f0);
        GroupWalk w(s, cv * 8);
        double pivot = pivot_of(x, pre, s, n, w.g);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            sum[i] = sq[i] = 0.0;
            e[i] = (double)f0[i] - pivot;
            const uint32_t g = w.g;
            w.next(s);
            if (i < 7 && w.g != g) pivot = pivot_of(x, pre, s, n, w.g);
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
                for (int i = 0; i < 8; i++) { const double d = (double)f[i] + e[i]; sum[i] += d; sq[i] = __builtin_fma(d, d, sq[i]); }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            sums[(size_t)pp * s.C + cv * 8 + i] = sum[i];
            sums[(size_t)(s.ppi + pp) * s.C + cv * 8 + i] = sq[i];
        }
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < 2 * s.C; k += s.threads) {           // (a thread reads and writes its own column)
        const uint32_t which = k >= s.C, c = k - which * s.C;
        double* col = sums + (size_t)which * s.ppi * s.C + c;
        double a = 0.0;
        for (uint32_t p = 0; p < s.ppi; p++) a += col[(size_t)p * s.C];
        col[0] = a;
    }
    __syncthreads();
    const Partials lay = partials_of(s);
    for (uint32_t k = threadIdx.x; k < 2 * s.G; k += s.threads) {
        const uint32_t which = k & 1u, g = k >> 1;
        double a = 0.0;
        for (uint32_t c = 0; c < s.cpg; c++) a += sums[(size_t)which * s.ppi * s.C + g * s.cpg + c];
        partial[(size_t)n * 2 * s.G * s.slabs + (size_t)k * lay.item + (size_t)slab * lay.slab] = a;
    }
}

// one wave per (sample, group)
template <typename T>
__global__ __launch_bounds__(64) void k_finish(const T* __restrict__ x, const T* __restrict__ pre, const double* __restrict__ partial, Shape s,
                                             float* __restrict__ mean_rstd) {
    const uint32_t n = blockIdx.x / s.G, g = blockIdx.x - n * s.G;
    const double* p = partial + (size_t)blockIdx.x * 2 * s.slabs;
    double a = 0.0, b = 0.0;
    for (uint32_t w = threadIdx.x; w < s.slabs; w += 64) { a += p[w]; b += p[s.slabs + w]; }
    a = wave_sum(a); b = wave_sum(b);
    if (threadIdx.x == 0) moments(s, x, pre, n, g, a, b, mean_rstd[(size_t)blockIdx.x * 2], mean_rstd[(size_t)blockIdx.x * 2 + 1]);
}

template <typename T, bool ACT, bool Q8>
__global__ __launch_bounds__(kMaxThreads) void k_apply(const T* __restrict__ x, const T* __restrict__ pre, Shape s, const double* __restrict__ partial,
                                                        float* __restrict__ mean_rstd, const void* __restrict__ gamma, const void* __restrict__ beta,
                                                        T* __restrict__ y, u2n* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ double scr[kMaxThreads], sums[2 * kMaxGroups];
    __shared__ float mom[2 * kMaxGroups];
    const uint32_t n = blockIdx.x / s.slabs, slab = blockIdx.x - n * s.slabs;
    if (s.inl) {
        combine_inline(s, partial + (size_t)n * 2 * s.G * s.slabs, scr, sums);
        for (uint32_t g = threadIdx.x; g < s.G; g += s.threads) {
            moments(s, x, pre, n, g, sums[2 * g], sums[2 * g + 1], mom[2 * g], mom[2 * g + 1]);
            if (slab == 0) { mean_rstd[((size_t)n * s.G + g) * 2] = mom[2 * g]; mean_rstd[((size_t)n * s.G + g) * 2 + 1] = mom[2 * g + 1]; }
        }
    } else
        for (uint32_t k = threadIdx.x; k < 2 * s.G; k += s.threads) mom[k] = mean_rstd[(size_t)n * s.G * 2 + k];
    __syncthreads();
    uint32_t pp, cv;
    if (!my_place(s, pp, cv)) return;
    constexpr bool kWhole = sizeof(T) == 4;
    float a[8], b[8], e[8] = {0, 0, 0, 0, 0, 0, 0, 0}, r[8];
    load_params<T>(gamma, cv * 8, s.pf32, a);
    load_params<T>(beta, cv * 8, s.pf32, b);
    if (pre) widen(load8(pre + (size_t)n * s.C + cv * 8), e);
    GroupWalk w(s, cv * 8);
#pragma unroll
    for (int i = 0; i < 8; i++, w.next(s)) {
        e[i] -= mom[2 * w.g];
        r[i] = mom[2 * w.g + 1];
        if (!kWhole) {                                                    // (x + e) r a + beta = x (a r) + b
            a[i] *= r[i];
            b[i] = __builtin_fmaf(e[i], a[i], b[i]);
        }
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
                const float z = __builtin_fmaf(kWhole ? (f[i] + e[i]) * r[i] : f[i], a[i], b[i]);
                f[i] = ACT ? z * sigmoid_of<T>(z) : z;
            }
            store8(y + at * 8, f);
        }
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------------
template <typename T, bool ACT> __device__ __forceinline__ float dz_of(float xh, float dy, float gamma, float beta) {
    if (!ACT) return dy;
    const float z = __builtin_fmaf(xh, gamma, beta), sg = sigmoid_of<T>(z);
    return dy * sg * __builtin_fmaf(z, 1.0f - sg, 1.0f);
}
// what a backward thread keeps of its 8 channels: xh = (x + m) r in float32, x r + m in 16 bits
struct Chan8 { float r[8], m[8], ga[8], be[8]; };
template <typename T> __device__ __forceinline__ float xh_of(const Chan8& k, int i, float x) {
    return sizeof(T) == 4 ? (x + k.m[i]) * k.r[i] : __builtin_fmaf(x, k.r[i], k.m[i]);
}
template <typename T>
__device__ __forceinline__ void load_chan(Chan8& k, const Shape& s, uint32_t n, uint32_t cv, const float* mean_rstd, const T* pre, const void* gamma, const void* beta) {
    float e[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    load_params<T>(gamma, cv * 8, s.pf32, k.ga);
    load_params<T>(beta, cv * 8, s.pf32, k.be);
    if (pre) widen(load8(pre + (size_t)n * s.C + cv * 8), e);
    GroupWalk w(s, cv * 8);
#pragma unroll
    for (int i = 0; i < 8; i++, w.next(s)) {
        const float* mr = mean_rstd + ((size_t)n * s.G + w.g) * 2;
        k.r[i] = mr[1];
        k.m[i] = sizeof(T) == 4 ? e[i] - mr[0] : (e[i] - mr[0]) * mr[1];
    }
}

// chan[n][which][c][slab], which: sum dz, sum dz xh and (PRE) sum xh; partial: the groups' sums of g = dz gamma and g xh
template <typename T, bool ACT, bool Q8, bool PRE>
__global__ __launch_bounds__(kMaxThreads) void k_bwd_stats(const void* __restrict__ x, const uint8_t* __restrict__ scales, const T* __restrict__ pre,
                                                            const T* __restrict__ dy, Shape s, const float* __restrict__ mean_rstd,
                                                            const void* __restrict__ gamma, const void* __restrict__ beta, float* __restrict__ partial,
                                                            float* __restrict__ chan) {
    extern __shared__ float part[];          // [K][ppi][C], then gamma [C], then [2][C]
    constexpr uint32_t K = PRE ? 3u : 2u;
    const uint32_t n = blockIdx.x / s.slabs, slab = blockIdx.x - n * s.slabs;
    uint32_t pp, cv;
    if (my_place(s, pp, cv)) {
        Chan8 k;
        load_chan(k, s, n, cv, mean_rstd, pre, gamma, beta);
        float s1[8] = {0, 0, 0, 0, 0, 0, 0, 0}, s2[8] = {0, 0, 0, 0, 0, 0, 0, 0}, s3[8] = {0, 0, 0, 0, 0, 0, 0, 0};
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
                    const float xh = xh_of<T>(k, i, fx[i]), dz = dz_of<T, ACT>(xh, fd[i], k.ga[i], k.be[i]);
                    s1[i] += dz;
                    s2[i] = __builtin_fmaf(dz, xh, s2[i]);
                    if (PRE) s3[i] += xh;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const size_t c = cv * 8 + i;
            part[(size_t)pp * s.C + c] = s1[i];
            part[(size_t)(s.ppi + pp) * s.C + c] = s2[i];
            if (PRE) part[(size_t)(2 * s.ppi + pp) * s.C + c] = s3[i];
            if (pp == 0) part[K * s.ppi * s.C + c] = k.ga[i];
        }
    }
    __syncthreads();
    const float* ga = part + K * s.ppi * s.C;
    float* weighted = part + (K * s.ppi + 1) * s.C;
    for (uint32_t k = threadIdx.x; k < K * s.C; k += s.threads) {
        const uint32_t which = k / s.C, c = k - which * s.C;
        float a = 0.f;
        for (uint32_t p = 0; p < s.ppi; p++) a += part[(size_t)(which * s.ppi + p) * s.C + c];
        chan[(((size_t)n * K + which) * s.C + c) * s.slabs + slab] = a;
        if (which < 2) weighted[k] = a * ga[c];
    }
    __syncthreads();
    const Partials lay = partials_of(s);
    for (uint32_t k = threadIdx.x; k < 2 * s.G; k += s.threads) {
        const uint32_t which = k & 1u, g = k >> 1;
        float a = 0.f;
        for (uint32_t c = 0; c < s.cpg; c++) a += weighted[which * s.C + g * s.cpg + c];
        partial[(size_t)n * 2 * s.G * s.slabs + (size_t)k * lay.item + (size_t)slab * lay.slab] = a;
    }
}

// one wave per (sample, group): the means of g and g xh
__global__ __launch_bounds__(64) void k_bwd_finish(const float* __restrict__ partial, Shape s, float* __restrict__ means) {
    const float* p = partial + (size_t)blockIdx.x * 2 * s.slabs;
    double a = 0.0, b = 0.0;
    for (uint32_t w = threadIdx.x; w < s.slabs; w += 64) { a += (double)p[w]; b += (double)p[s.slabs + w]; }
    a = wave_sum(a); b = wave_sum(b);
    const double cnt = (double)s.HW * s.cpg;
    if (threadIdx.x == 0) { means[(size_t)blockIdx.x * 2] = (float)(a / cnt); means[(size_t)blockIdx.x * 2 + 1] = (float)(b / cnt); }
}

template <typename T, bool ACT, bool Q8, bool PRE>
__global__ __launch_bounds__(kMaxThreads) void k_bwd_apply(const void* __restrict__ x, const uint8_t* __restrict__ scales, const T* __restrict__ pre,
                                                            const T* __restrict__ dy, Shape s, const float* __restrict__ mean_rstd,
                                                            const float* __restrict__ partial, const float* __restrict__ means,
                                                            const float* __restrict__ chan, const void* __restrict__ gamma, const void* __restrict__ beta,
                                                            T* __restrict__ dx, T* __restrict__ dpre, void* __restrict__ dgamma, void* __restrict__ dbeta) {
    __shared__ double scr[kMaxThreads], sums[2 * kMaxGroups];
    __shared__ float mom[2 * kMaxGroups];
    constexpr uint32_t K = PRE ? 3u : 2u;
    const uint32_t n = blockIdx.x / s.slabs, slab = blockIdx.x - n * s.slabs;
    if (s.inl) {
        combine_inline(s, partial + (size_t)n * 2 * s.G * s.slabs, scr, sums);
        const double cnt = (double)s.HW * s.cpg;
        for (uint32_t k = threadIdx.x; k < 2 * s.G; k += s.threads) mom[k] = (float)(sums[k] / cnt);
    } else
        for (uint32_t k = threadIdx.x; k < 2 * s.G; k += s.threads) mom[k] = means[(size_t)n * s.G * 2 + k];
    __syncthreads();
    uint32_t pp, cv;
    if (my_place(s, pp, cv) && dx) {
        Chan8 k;
        load_chan(k, s, n, cv, mean_rstd, pre, gamma, beta);
        float m1[8], m2[8];
        GroupWalk w(s, cv * 8);
#pragma unroll
        for (int i = 0; i < 8; i++, w.next(s)) { m1[i] = mom[2 * w.g]; m2[i] = mom[2 * w.g + 1]; }
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
                    const float xh = xh_of<T>(k, i, fx[i]), dz = dz_of<T, ACT>(xh, fd[i], k.ga[i], k.be[i]);
                    fx[i] = k.r[i] * (__builtin_fmaf(dz, k.ga[i], -m1[i]) - xh * m2[i]);
                }
                store8(dx + (at0 + (size_t)(p + u * s.ppi) * s.cvs) * 8, fx);
            }
        }
    }
    // The channels' gradients: L lanes to a channel (about four slabs a lane), the grid's lane groups in turn (dpre within the sample's
    // workgroups, dgamma / dbeta in the first sample's).
    const uint32_t L = s.lanes, sub = threadIdx.x & (L - 1u), per_wg = s.threads / L, first = slab * per_wg + threadIdx.x / L, stride = s.slabs * per_wg;
    auto total = [&](uint32_t nn, uint32_t which, uint32_t c) {
        const float* p = chan + (((size_t)nn * K + which) * s.C + c) * s.slabs;
        double a = 0.0;
        for (uint32_t w = sub; w < s.slabs; w += 4 * L) {
            float v[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) v[u] = p[min(w + u * L, s.slabs - 1)];
#pragma unroll
            for (uint32_t u = 0; u < 4; u++)
                if (w + u * L < s.slabs) a += (double)v[u];
        }
        for (uint32_t o = L / 2; o >= 1; o >>= 1) a += __shfl_xor(a, o, 64);
        return a;
    };
    if (PRE && dpre) {
        for (uint32_t c = first; c < s.C; c += stride) {
            const double a = total(n, 0, c), h = total(n, 2, c);
            const uint32_t g = c / s.cpg;
            const double rstd = (double)mean_rstd[((size_t)n * s.G + g) * 2 + 1], ga = (double)load_param<T>(gamma, c, s.pf32);
            if (sub == 0) dpre[(size_t)n * s.C + c] = (T)(float)(rstd * (ga * a - (double)s.HW * (double)mom[2 * g] - (double)mom[2 * g + 1] * h));
        }
    }
    if (n == 0 && (dgamma || dbeta)) {
        for (uint32_t c = first; c < s.C; c += stride) {
            double a = 0.0, b = 0.0;
            for (uint32_t nn = 0; nn < s.N; nn++) { a += total(nn, 0, c); b += total(nn, 1, c); }
            if (sub == 0) {
                if (dbeta) store_param<T>(dbeta, c, s.pf32, a);
                if (dgamma) store_param<T>(dgamma, c, s.pf32, b);
            }
        }
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
uint64_t group_floats(const Shape& s) { return (uint64_t)s.N * 2 * s.G * s.slabs; }      // (the forward's are doubles: within the backward's total, since G <= C)
uint64_t chan_floats(const Shape& s) { return (uint64_t)s.N * 3 * s.C * s.slabs; }

template <typename T, bool ACT, bool Q8>
void forward(const void* x_, const void* pre_, const void* gamma, const void* beta, const Shape& s, void* y, uint8_t* saved, float* mean_rstd,
             float* scratch, hipStream_t st) {
    double* partial = reinterpret_cast<double*>(scratch);
    const T *x = static_cast<const T*>(x_), *pre = static_cast<const T*>(pre_);
    hipLaunchKernelGGL(k_stats<T>, dim3(s.N * s.slabs), dim3(s.threads), 2 * s.ppi * s.C * 8, st, x, pre, s, partial);
    if (!s.inl) hipLaunchKernelGGL(k_finish<T>, dim3(s.N * s.G), dim3(64), 0, st, x, pre, partial, s, mean_rstd);
    hipLaunchKernelGGL((k_apply<T, ACT, Q8>), dim3(s.N * s.slabs), dim3(s.threads), 0, st, x, pre, s, partial, mean_rstd, gamma, beta, static_cast<T*>(y),
                       reinterpret_cast<u2n*>(saved), saved + (size_t)s.N * s.HW * s.C);
}
template <typename T, bool ACT, bool Q8, bool PRE>
void backward_pre(const void* x, const T* pre, const T* dy, const void* gamma, const void* beta, const float* mean_rstd, const Shape& s, T* dx, T* dpre,
                  void* dgamma, void* dbeta, float* scratch, hipStream_t st) {
    const uint8_t* scales = Q8 ? static_cast<const uint8_t*>(x) + (size_t)s.N * s.HW * s.C : nullptr;
    float *partial = scratch, *chan = partial + group_floats(s), *means = chan + chan_floats(s);
    const uint32_t K = PRE ? 3 : 2;
    hipLaunchKernelGGL((k_bwd_stats<T, ACT, Q8, PRE>), dim3(s.N * s.slabs), dim3(s.threads), (K * s.ppi + 3) * s.C * 4, st, x, scales, pre, dy, s,
                       mean_rstd, gamma, beta, partial, chan);
    if (!s.inl) hipLaunchKernelGGL(k_bwd_finish, dim3(s.N * s.G), dim3(64), 0, st, partial, s, means);
    hipLaunchKernelGGL((k_bwd_apply<T, ACT, Q8, PRE>), dim3(s.N * s.slabs), dim3(s.threads), 0, st, x, scales, pre, dy, s, mean_rstd, partial, means,
                       chan, gamma, beta, dx, dpre, dgamma, dbeta);
}
template <typename T, bool ACT, bool Q8>
void backward(const void* x, const void* pre, const void* dy, const void* gamma, const void* beta, const float* mean_rstd, const Shape& s,
              void* dx, void* dpre, void* dgamma, void* dbeta, float* scratch, hipStream_t st) {
    const T* dyp = static_cast<const T*>(dy);
    if (pre)
        backward_pre<T, ACT, Q8, true>(x, static_cast<const T*>(pre), dyp, gamma, beta, mean_rstd, s, static_cast<T*>(dx), static_cast<T*>(dpre), dgamma,
                                       dbeta, scratch, st);
    else
        backward_pre<T, ACT, Q8, false>(x, nullptr, dyp, gamma, beta, mean_rstd, s, static_cast<T*>(dx), nullptr, dgamma, dbeta, scratch, st);
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
    return (group_floats(s) + chan_floats(s) + (uint64_t)N * G * 2) * sizeof(float);
}

int sdfx_group_norm_train_forward(const void* x, const void* pre, const void* gamma, const void* beta, uint32_t N, uint32_t HW, uint32_t C, uint32_t G,
                                  float eps, int silu, int dtype, int params_f32, void* y, void* saved8, float* mean_rstd, float* scratch,
                                  sdfx_stream_t stream) {
    SDFX_REQUIRE(x && gamma && beta && y && mean_rstd && scratch, "group_norm_train_forward: null pointer");
    SDFX_REQUIRE(dtype >= 0 && dtype <= 2, "group_norm_train_forward: dtype %d (0 fp16, 1 bf16, 2 float32)", dtype);
    Shape s;
    SDFX_REQUIRE(make_shape(N, HW, C, G, s), "group_norm_train_forward: needs C %% 8 == 0, C %% G == 0, C <= %u, G <= %u and N < 2^23 (got N=%u HW=%u C=%u G=%u)",
                 kMaxThreads * 8, kMaxGroups, N, HW, C, G);
    SDFX_REQUIRE(!saved8 || C % 32 == 0, "group_norm_train_forward: the 8-bit form needs C %% 32 == 0 (got %u)", C);
    SDFX_REQUIRE(aligned16(x) && aligned16(y) && aligned16(saved8) && aligned16(pre) && aligned16(gamma) && aligned16(beta) &&
                 reinterpret_cast<uintptr_t>(scratch) % 8 == 0, "group_norm_train_forward: misaligned pointer");
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
    SDFX_REQUIRE(make_shape(N, HW, C, G, s), "group_norm_train_backward: needs C %% 8 == 0, C %% G == 0, C <= %u, G <= %u and N < 2^23 (got N=%u HW=%u C=%u G=%u)",
                 kMaxThreads * 8, kMaxGroups, N, HW, C, G);
    SDFX_REQUIRE(!eight_bits || C % 32 == 0, "group_norm_train_backward: the 8-bit form needs C %% 32 == 0 (got %u)", C);
    SDFX_REQUIRE(pre || !dpre, "group_norm_train_backward: dpre without pre");
    SDFX_REQUIRE(aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(pre) && aligned16(gamma) && aligned16(beta), "group_norm_train_backward: misaligned pointer");
    s.pf32 = params_f32 || dtype == 2;
    const bool eight = eight_bits != 0;
    SDFX_GN_DISPATCH(backward, x, pre, dy, gamma, beta, mean_rstd, s, dx, dpre, dgamma, dbeta, scratch, as_stream(stream));
    return check_launch("group_norm_train_backward");
}

}  // extern "C"
