// act8.h — eight consecutive channels of an activation as a thread holds them: loads / stores in the three activation types, and the
// 8-bit checkpoint form the training kernels keep their input in (groupnorm_train.hip, geglu_train.hip).
//
// 8-bit form of a row of C channels (C % 32 == 0): C codes, one signed byte each, and C / 32 scale bytes. A block of 32 consecutive
// channels shares the step 2^(floor(log2 max|x|) - 6), at least 2^-126; its scale byte is the step's biased exponent, and
// code = clamp(round-half-even(x / step), -127, 127): half a step off at most (one step where the largest magnitudes clamp), i.e.
// 2^-7 .. 2^-6 of the block's maximum. Steps are powers of two so that x / step and code * step are exact: the codes do not depend on
// how a division is rounded. A block that holds an infinity or a NaN gets scale byte 255 and codes 0: it decodes as NaN.
// Signed bytes with a shared exponent rather than e4m3: the 7 bits resolve 2^-7 of the maximum everywhere, e4m3's 3 mantissa bits
// 2^-4 of each value (rms 2.6 % against 0.7 % of the deviation of a normal block).
#pragma once

#include "sdfx_common.h"

namespace sdfx {

typedef float f2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef unsigned u4n __attribute__((ext_vector_type(4)));   // (native vectors: arrays of HIP's uint4 struct end up in scratch)
typedef unsigned u2n __attribute__((ext_vector_type(2)));

// raw<T>: the registers of 8 channels as they are loaded
template <typename T> struct Raw8 { u4n w; };
template <> struct Raw8<float> { u4n w, w2; };

template <typename T> __device__ __forceinline__ Raw8<T> load8(const T* p) {
    Raw8<T> r;
    r.w = *reinterpret_cast<const u4n*>(p);
    if constexpr (sizeof(T) == 4) r.w2 = *reinterpret_cast<const u4n*>(p + 4);
    return r;
}
__device__ __forceinline__ void widen(const Raw8<float>& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) { f[i] = __uint_as_float(r.w[i]); f[4 + i] = __uint_as_float(r.w2[i]); }
}
__device__ __forceinline__ void widen(const Raw8<_Float16>& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = r.w[i];
        const h2v h = *reinterpret_cast<const h2v*>(&u);
        f[2 * i] = (float)h[0]; f[2 * i + 1] = (float)h[1];
    }
}
__device__ __forceinline__ void widen(const Raw8<__bf16>& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(r.w[i] << 16); f[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u); }
}
// one rounding (to nearest even) per value
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    *reinterpret_cast<u4n*>(p) = u4n{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    *reinterpret_cast<u4n*>(p + 4) = u4n{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])};
}
__device__ __forceinline__ void store8(_Float16* p, const float (&f)[8]) {
    u4n w;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const h2v h = __builtin_convertvector(f2v{f[2 * i], f[2 * i + 1]}, h2v);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<u4n*>(p) = w;
}
__device__ __forceinline__ void store8(__bf16* p, const float (&f)[8]) {
    u4n w;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const b2v h = __builtin_convertvector(f2v{f[2 * i], f[2 * i + 1]}, b2v);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<u4n*>(p) = w;
}
// eight consecutive parameters of the activation's type or float32 (16-byte aligned)
template <typename T> __device__ __forceinline__ void load_params(const void* p, size_t c, bool f32, float (&f)[8]) {
    if (f32) widen(load8(static_cast<const float*>(p) + c), f);
    else widen(load8(static_cast<const T*>(p) + c), f);
}
// a parameter of the activation's type or float32
template <typename T> __device__ __forceinline__ float load_param(const void* p, size_t i, bool f32) {
    return f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}
template <typename T> __device__ __forceinline__ void store_param(void* p, size_t i, bool f32, double v) {
    if (f32) static_cast<float*>(p)[i] = (float)v;
    else static_cast<T*>(p)[i] = (T)(float)v;
}

// ---- 8-bit form: the four lanes of a quad hold the four vectors of a block ------------------------------------------------------
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));   // quad_perm [1, 0, 3, 2]
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));   // quad_perm [2, 3, 0, 1]
}
// codes of this lane's 8 channels; the block's scale byte in `scale` (the same in the quad's four lanes)
__device__ __forceinline__ u2n encode8(const float (&f)[8], uint32_t& scale) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);   // (as integers: a NaN is larger than an infinity)
    const uint32_t e = quad_max(m) >> 23;
    const bool bad = e == 255u;
    scale = bad ? 255u : (e > 7u ? e - 6u : 1u);
    const float inv = bad ? 0.f : __uint_as_float((254u - scale) << 23);
    u2n c;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float q = __builtin_rintf(f[4 * h + i] * inv);
            const int v = bad ? 0 : (int)fminf(fmaxf(q, -127.f), 127.f);
            w |= ((uint32_t)v & 255u) << (8 * i);
        }
        c[h] = w;
    }
    return c;
}
__device__ __forceinline__ void decode8(u2n c, uint32_t scale, float (&f)[8]) {
    const float step = __uint_as_float(scale << 23), low = -128.f * step;          // (scale 255: infinity, inf - inf = NaN)
    const u2n w = c ^ u2n{0x80808080u, 0x80808080u};          // code + 128: one conversion and one fma a value, both exact
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = __builtin_fmaf((float)((w[i >> 2] >> (8 * (i & 3))) & 255u), step, low);
}

// an input read back in the backward: the activation itself (Q8 false) or its 8-bit form
template <typename T, bool Q8> struct Saved { Raw8<T> r; };
template <typename T> struct Saved<T, true> { u2n c; uint32_t s; };
// vector `i` (8 channels) of a saved activation; `scales` only with Q8
template <typename T, bool Q8>
__device__ __forceinline__ Saved<T, Q8> load_saved(const void* x, const uint8_t* scales, size_t i) {
    Saved<T, Q8> v;
    if constexpr (Q8) {
        v.c = static_cast<const u2n*>(x)[i];
        v.s = scales[i >> 2];
    } else v.r = load8(static_cast<const T*>(x) + i * 8);
    return v;
}
template <typename T> __device__ __forceinline__ void widen_saved(const Saved<T, false>& v, float (&f)[8]) { widen(v.r, f); }
template <typename T> __device__ __forceinline__ void widen_saved(const Saved<T, true>& v, float (&f)[8]) { decode8(v.c, v.s, f); }

// sigmoid of an activation of type T. 16 bits: on the hardware's exp2 and reciprocal, |v| 2^-23 off, 4 instructions instead of some 30. float32: whole
template <typename T> __device__ __forceinline__ float sigmoid_of(float v) {
    if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-v));
    else return __builtin_amdgcn_rcpf(1.0f + __expf(-v));
}

}  // namespace sdfx
