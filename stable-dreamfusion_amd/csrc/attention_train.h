// attention_train.h — what the attention kernels with a gradient share: shapes, matrix-core fragments, tiles in LDS.
//   s = scale q k^T, p = softmax(s over the visible keys), o = p v;   delta = sum(do o), dp = do v^T, ds = p (dp - delta),
//   dq = scale ds k, dk = scale ds^T q, dv = p^T do
// (attention_train.hip: forward, joins, entry points; attention_train_dq.hip; attention_train_dkdv.hip)
//
// Every product runs transposed on v_mfma_f32_32x32x16 so that a lane owns one row of the softmax (forward, dq) or one key (dk / dv): the
// D fragment of lane (x = lane & 31, hi = lane >> 5) holds, in element r, row (r & 3) + 8 (r >> 2) + 4 hi of column x. Packed to 16 bits
// its elements 8 e .. 8 e + 7 are the B operand of K step e when the A operand takes its 16 rows in that same order, which two
// ds_read_b64_tr_b16 of a row-major tile deliver: probabilities never pass through LDS and no tile is stored transposed.
#pragma once

#include "sdfx_common.h"

namespace sdfx_attn {

using namespace sdfx;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef unsigned u2v __attribute__((ext_vector_type(2)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));   // (native vectors: arrays of HIP's uint4 struct end up in scratch)

struct Shape {
    uint32_t B, H, Hk, Nq, Nk, D;
    uint32_t group, rows;                 // query heads per key head; rows of one key head: group * Nq, row R = (head in group) * Nq + query
    uint64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;   // element strides (the channel stride is 1)
    const uint8_t* mask;                  // [B, Nk], 0 = the key is not seen; or null
    int causal, off;                      // query i sees keys <= i + off (off = Nk - Nq)
    float scale, c;                       // softmax scale; times log2(e)
    uint32_t tiles_x;                     // workgroups along rows (forward, dq) or keys (dk / dv)
    uint32_t splits;                      // workgroups along the other axis
    float few;                            // a row whose probabilities sum to less than this, of the largest, is one that few keys carry
    int exact;                            // few sums: every rounding of p and ds is made good (below, at marked)
};

// A launch takes fewer than 2^32 threads along x: workgroups beyond 2^22 go along y (many short windows: 2^24 heads of a few tokens).
constexpr uint32_t kGridXLog2 = 22;
inline dim3 flat_grid(uint64_t n) { return n >> kGridXLog2 ? dim3(1u << kGridXLog2, (uint32_t)((n + (1u << kGridXLog2) - 1) >> kGridXLog2)) : dim3((uint32_t)n); }
__device__ __forceinline__ uint32_t flat_block() { return (blockIdx.y << kGridXLog2) + blockIdx.x; }          // (to be checked against the launch's count)

template <typename T> struct Half;
template <> struct Half<_Float16> {
    typedef h8 v8; typedef h4 v4; typedef h2 v2;
    // Probabilities of a long flat row lie under fp16's normal range (2^-14), ds further down. The backward forms p * 2^15 and
    // ds * (2^15 g), g from the largest |do| |v| (see grad_scale): both in range, the power of two taken out of the float32 sums.
    static constexpr float kShift = 15.f;
    static constexpr bool kScaled = true;
};
template <> struct Half<__bf16> {
    typedef b8 v8; typedef b4 v4; typedef b2 v2;
    static constexpr float kShift = 0.f;
    static constexpr bool kScaled = false;
};
__device__ __forceinline__ f32x16 mma(h8 a, h8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(b8 a, b8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float max_halves(float x) {      // over lanes l and l ^ 32
    const uint32_t u = __float_as_uint(x);
    const u2v r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r.x, b = r.y;
    return fmaxf(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float sum_halves(float x) {
    const uint32_t u = __float_as_uint(x);
    const u2v r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r.x, b = r.y;
    return __uint_as_float(a) + __uint_as_float(b);
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; r++) z[r] = 0.f;
    return z;
}
// elements 8 e .. 8 e + 7 of a D fragment as the B operand of K step e
template <typename T> __device__ __forceinline__ typename Half<T>::v8 operand(const f32x16& p, int e) {
    typename Half<T>::v8 v;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const typename Half<T>::v2 h = __builtin_convertvector(f2{p[8 * e + 2 * j], p[8 * e + 2 * j + 1]}, typename Half<T>::v2);
        v[2 * j] = h[0]; v[2 * j + 1] = h[1];
    }
    return v;
}

// In front of a rarely needed block of selects (5 instructions a score): keeps it a branch, which the compiler would otherwise fold into straight code
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// ---- tiles of ROWS rows in LDS, row-major, an odd number of 16-byte chunks a row (16 rows of a ds_read_b128 start in 16 bank quads) ----
template <int DP, int ROWS, int TH> struct Tile {
    static constexpr int CH = DP / 8;
    static constexpr uint32_t PITCH = (uint32_t)(CH | 1) * 16u;
    static constexpr int ROWS_ = ROWS;
    static constexpr uint32_t BYTES = (uint32_t)ROWS * PITCH + 16u;      // (and a slot that nothing reads: see Stage)
    static constexpr int NCH = ROWS * CH;
    static constexpr int PT = (NCH + TH - 1) / TH;           // chunks per thread
};
// Channel blocks are 32 wide: the transposed reads of the last block of a row whose width is no multiple of 32 run up to 32 channels past
// it (their results are rows of the product that nothing stores): bytes to have behind the last tile.
constexpr uint32_t kTileSlack = 64;

// A thread's chunks of a tile: where each lies behind the tile's first row in memory (bytes; the first row's address is a scalar) and in LDS.
// Only the D / 8 chunks a row has are moved; a kernel that reads further clears LDS once. A thread without a chunk of its own reads the
// tile's last one and writes it to the 16 bytes behind the tile: no predicate and no branch around a load (scalar branches there cost
// 30 % of the dq kernel: the loads of a branch are waited for at its end).
template <typename L, int TH> struct Stage {
    uint32_t src[L::PT], dst[L::PT];
    __device__ __forceinline__ void init(uint32_t D, uint64_t sn, uint32_t tid) {
        const uint32_t chunks = D / 8, count = L::ROWS_ * chunks;
#pragma unroll
        for (int i = 0; i < L::PT; i++) {
            const uint32_t mine = tid + (uint32_t)i * TH, c = min(mine, count - 1u), row = c / chunks, ch = c - row * chunks;
            src[i] = row * (uint32_t)sn * 2u + ch * 16u;
            dst[i] = mine < count ? row * L::PITCH + ch * 16u : L::ROWS_ * L::PITCH;
        }
    }
    __device__ __forceinline__ uint32_t row_of(int i) const { return min(dst[i] / L::PITCH, (uint32_t)L::ROWS_ - 1u); }
    // `rows` of the tile exist (the others repeat the last)
    __device__ __forceinline__ void request(u4v (&r)[L::PT], const void* first, uint64_t sn, uint32_t rows) const {
        if (rows >= (uint32_t)L::ROWS_) {
#pragma unroll
            for (int i = 0; i < L::PT; i++) r[i] = *reinterpret_cast<const u4v*>(static_cast<const uint8_t*>(first) + src[i]);
        } else {
            keep_branch();
#pragma unroll
            for (int i = 0; i < L::PT; i++) {
                const uint32_t row = row_of(i), past = row >= rows ? row - (rows - 1u) : 0u;
                r[i] = *reinterpret_cast<const u4v*>(static_cast<const uint8_t*>(first) + (src[i] - past * (uint32_t)sn * 2u));
            }
        }
    }
    // into LDS; with `all` false, rows whose bit of `live` is clear as zeros (a masked key's values may be anything: 0 * NaN must not reach a product)
    __device__ __forceinline__ void put(uint8_t* tile, u4v (&r)[L::PT], bool all, uint64_t live) const {
        if (!all) {
            keep_branch();
#pragma unroll
            for (int i = 0; i < L::PT; i++)
                if (!((live >> row_of(i)) & 1u)) r[i] = u4v{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int i = 0; i < L::PT; i++) *reinterpret_cast<u4v*>(tile + dst[i]) = r[i];
    }
};
__device__ __forceinline__ void clear_lds(uint8_t* lds, uint32_t bytes, uint32_t tid, uint32_t th) {
    for (uint32_t i = tid; i < bytes / 16u; i += th) reinterpret_cast<u4v*>(lds)[i] = u4v{0u, 0u, 0u, 0u};
    __syncthreads();
}
// A operand, rows of the tile: lane (x, hi) row 32 blk + x, channels 16 ks + 8 hi .. + 7
template <typename T, typename L> __device__ __forceinline__ typename Half<T>::v8 row_operand(const uint8_t* tile, uint32_t blk, uint32_t ks, uint32_t x, uint32_t hi) {
    return *reinterpret_cast<const typename Half<T>::v8*>(tile + (32u * blk + x) * L::PITCH + ks * 32u + hi * 16u);
}
// A operand, the tile transposed: lane (x, hi) channel 32 dt + x; its 8 elements are rows 16 e + 4 hi + {0..3, 8..11}
typedef s4 __attribute__((address_space(3)))* lds_s4;
template <typename T, typename L> __device__ __forceinline__ typename Half<T>::v8 col_operand(const uint8_t* tile, uint32_t e, uint32_t dt, uint32_t lane) {
    const uint32_t l16 = lane & 15u, cb = (lane >> 4) & 1u, hi = lane >> 5;
    const uint8_t* p = tile + (16u * e + 4u * hi + (l16 >> 2)) * L::PITCH + (32u * dt + 16u * cb + 4u * (l16 & 3u)) * 2u;
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p));
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 8u * L::PITCH));
    const s8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Half<T>::v8, v);
}
// B operand straight from memory: lane (x, hi) row `p`, channels 16 ks + 8 hi .. + 7, zero from D on
template <typename T, int KS> __device__ __forceinline__ void row_fragments(typename Half<T>::v8 (&f)[KS], const void* p, uint32_t D, uint32_t hi) {
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        const uint32_t c0 = 16u * ks + 8u * hi;
        u4v w = u4v{0u, 0u, 0u, 0u};
        if (c0 < D) w = *reinterpret_cast<const u4v*>(static_cast<const uint16_t*>(p) + c0);
        f[ks] = __builtin_bit_cast(typename Half<T>::v8, w);
    }
}
// four consecutive channels
template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    const typename Half<T>::v2 x = __builtin_convertvector(f2{a, b}, typename Half<T>::v2), y = __builtin_convertvector(f2{c, d}, typename Half<T>::v2);
    *reinterpret_cast<typename Half<T>::v4*>(p) = typename Half<T>::v4{x[0], x[1], y[0], y[1]};
}

// ---- the power of two the fp16 backward scales ds by -------------------------------------------------------------------------------
// |dp - delta| <= 2 M, M = max |do row| max |v row| over the key head's rows (attention_train.hip: k_prep leaves the squares of
// block maxima): g = 2^-k with 2 M g <= 1, so |2^15 p g (dp - delta)| <= 2^15 whatever the loss scale, and gradients down to 2^-29 of
// that bound are normal numbers.
__device__ __forceinline__ float grad_scale(const float* rows2, uint32_t nr, const float* v2, uint32_t nv, uint32_t lane, float& vmax) {
    float a = 0.f, b = 0.f;
    for (uint32_t i = lane; i < nr; i += 64) a = fmaxf(a, rows2[i]);
    for (uint32_t i = lane; i < nv; i += 64) b = fmaxf(b, v2[i]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) { a = fmaxf(a, __shfl_xor(a, o, 64)); b = fmaxf(b, __shfl_xor(b, o, 64)); }
    vmax = sqrtf(b);
    const float m = sqrtf(a) * vmax;
    if (!(m > 0.f) || m > 1e37f) return 1.f;
    const uint32_t e = __float_as_uint(m) >> 23;
    return __uint_as_float((252u - min(e, 251u)) << 23);
}
constexpr uint32_t kPrepRows = 32;         // rows per workgroup of k_prep = rows per entry of the maxima
__host__ __device__ inline uint32_t prep_blocks(uint32_t n) { return (n + kPrepRows - 1) / kPrepRows; }

// what the backward's kernels get beside the shape
struct BwdArgs {
    const void *q, *k, *v, *dy;
    const float *lse, *delta, *rows2, *v2;
    const uint32_t* seen2;                 // [B][2]: the first two keys of a batch entry's mask that are seen, Nk where there is none (null: no mask)
    void *dq, *dk, *dv;                    // T [B, Nq, H, D], [B, Nk, Hk, D] (or null: not wanted)
    float *part, *part2;                   // splits > 1: float32 [splits][B Hk][rows or Nk][D] of dq, or of dk and dv
};
constexpr int kWidths[] = {48, 64, 80, 128, 160, 256};      // channels a kernel is built for; a head takes the next of them

// attention_train_dq.hip, attention_train_dkdv.hip: launch (shape's tiles_x / splits set for `waves` a workgroup)
void launch_dq(const BwdArgs& a, const Shape& s, int bf16, int waves, hipStream_t st);
void launch_dkdv(const BwdArgs& a, const Shape& s, int bf16, hipStream_t st);
// rows of the tile each stages: keys (forward, dq) or queries (dk / dv). One wave alone takes 32 and needs one buffer: its next tile waits in
// registers until it is done with the last (17 KB of LDS at 128 channels: eight such workgroups a CU).
constexpr int key_tile(int dp, int nw) { return dp <= 128 && nw == 4 ? 64 : 32; }
constexpr int buffers(int nw) { return nw == 4 ? 2 : 1; }
constexpr int query_tile(int dm) { return dm <= 80 ? 64 : 32; }
inline int padded(uint32_t D) {
    for (int w : kWidths)
        if (D <= (uint32_t)w) return w;
    return 0;
}

#define SDFX_ATTN_WIDTH(fn, T, nw, ...)                                   \
    do {                                                                  \
        switch (padded(s.D)) {                                            \
            case 48: fn<T, 48, nw>(__VA_ARGS__); break;                   \
            case 64: fn<T, 64, nw>(__VA_ARGS__); break;                   \
            case 80: fn<T, 80, nw>(__VA_ARGS__); break;                   \
            case 128: fn<T, 128, nw>(__VA_ARGS__); break;                 \
            case 160: fn<T, 160, nw>(__VA_ARGS__); break;                 \
            default: fn<T, 256, nw>(__VA_ARGS__); break;                  \
        }                                                                 \
    } while (0)

// operands of the second products requested ahead of the exponentials: where a lane's registers hold them
constexpr bool ahead(int dp) { return dp <= 64; }

// the tiles of `n` that split `i` of `splits` takes
__device__ __forceinline__ uint32_t split_at(uint32_t n, uint32_t i, uint32_t splits) { return splits == 1 ? (i ? n : 0u) : (uint32_t)((uint64_t)n * i / splits); }

// p and ds are rounded to the inputs' type for the second products. In sums over many rows and keys these roundings average out against that of the
// result: 1.41 times its own error alone. Two kinds of sums have little to average, and add a product with what the rounding left:
//  - a row that few keys carry: its probabilities sum to less than `few` = 4 of the largest. The terms of its dq cancel against each other
//    (bf16, causal 1010 x 24, scores with a deviation of 4: dq 2.6e-3 off where its own rounding is 1.7e-3; with the product 1.7e-3).
//    Marking rows below 16 gains nothing that shows and costs dq 14 us at 4096 x 40, this 4.
//  - at most 512 rows to a key head or at most 128 keys (`exact`: every row is marked, and dv takes the product too): sums of a
//    few, or of probabilities that all lie at one place between two powers of two, are up to 2.5 times as far off.
// The forward knows the sum, the backward only its logarithm, of which no bit can be spared (2^-22 of it were 2e-4 of a probability at 1000): the
// mark is the lowest bit of o_rest's first channel, 2^-23 of that value, and from k_prep on delta's.
__device__ __forceinline__ bool marked(float delta) { return __float_as_uint(delta) & 1u; }

// What rounding o to 16 bits left, in units of the float32's last place: 16 bits again (13 in fp16), and with them o is known exactly. (As a
// value of the inputs' type it was known to 17 bits in bf16.) Clamped below fp16's normal range, where o then is off by at most 2^-32.
template <typename T> __device__ __forceinline__ int o_rest(float f, T rounded) {
    const float r = (float)rounded;
    const int d = (int)(__float_as_uint(f) - __float_as_uint(r));
    return __builtin_fabsf(r) < INFINITY ? max(-32768, min(32767, d)) : 0;
}
template <typename T> __device__ __forceinline__ float o_whole(T rounded, short rest) { return __uint_as_float(__float_as_uint((float)rounded) + (uint32_t)(int)rest); }
template <typename T> __device__ __forceinline__ void store_rest4(short* p, const float (&f)[4], bool first, bool mark) {
    int d[4];
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] = o_rest<T>(f[i], (T)f[i]);
    if (first) d[0] = (d[0] & ~1) | (mark ? 1 : 0);
    *reinterpret_cast<s4*>(p) = s4{(short)d[0], (short)d[1], (short)d[2], (short)d[3]};
}

// A row that sees one key has no ds: dp and delta are the same number, and the bits in which they differ would be all of the gradient where no
// row has another. Which rows those are follows from the masks alone: with f1 < f2 the first two keys of the batch entry's mask, a row
// whose last key is `lim` sees none if lim < f1, one (f1) if f1 <= lim < f2, more otherwise.
// A row that one of several keys nearly carries keeps what p (dp - delta) gives, two float32 sums whose roundings are 2^-24 of |do| |v| each: with a
// second key 12 / 14 nats down its dq is 1.5 / 11 % off (dp summed against itself, as a plain form does, 0.5 / 3 %).
struct TwoSeen { int f1, f2; };
__device__ __forceinline__ TwoSeen two_seen(const BwdArgs& a, uint32_t b) {
    if (!a.seen2) return {0, 1};
    return {(int)a.seen2[2 * b], (int)a.seen2[2 * b + 1]};
}
// what rounding elements 8 e .. 8 e + 7 of a D fragment to `hi` left, as an operand
template <typename T> __device__ __forceinline__ typename Half<T>::v8 left_over(const f32x16& p, int e, const typename Half<T>::v8& hi) {
    typename Half<T>::v8 v;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const typename Half<T>::v2 h = __builtin_convertvector(f2{p[8 * e + 2 * j] - (float)hi[2 * j], p[8 * e + 2 * j + 1] - (float)hi[2 * j + 1]}, typename Half<T>::v2);
        v[2 * j] = h[0]; v[2 * j + 1] = h[1];
    }
    return v;
}

// the row a lane owns in the forward and in dq
struct Row {
    uint32_t R, head, qi;                  // row of the key head (clamped), query head, query
    bool on;
    int lim;                               // last key a causal row sees (may be negative)
};
__device__ __forceinline__ Row row_of(const Shape& s, uint32_t r, uint32_t hk) {
    Row w;
    w.on = r < s.rows;
    w.R = min(r, s.rows - 1u);
    const uint32_t g = w.R / s.Nq;
    w.qi = w.R - g * s.Nq;
    w.head = hk * s.group + g;
    w.lim = s.causal ? (int)w.qi + s.off : 0x7fffffff;
    return w;
}
// smallest and largest query among rows a .. b (rows of several heads: all queries)
__device__ __forceinline__ void query_range(const Shape& s, uint32_t a, uint32_t b, uint32_t& lo, uint32_t& hi) {
    const uint32_t ga = a / s.Nq, gb = b / s.Nq;
    lo = ga == gb ? a - ga * s.Nq : 0u;
    hi = ga == gb ? b - ga * s.Nq : s.Nq - 1u;
}
template <int KT> constexpr uint64_t all_keys() { return KT == 64 ? ~0ull : ((1ull << (KT & 63)) - 1ull); }
// Keys of a tile that exist (`left` from its first on) and are not masked, one bit each, the same in every wave. The mask's byte is loaded early
// (`row`: the batch entry's mask from the tile's first key on), the ballot taken later.
__device__ __forceinline__ uint8_t mask_byte(const uint8_t* row, uint32_t left, uint32_t lane) { return row[min(lane, left - 1u)]; }
template <int KT> __device__ __forceinline__ uint64_t live_keys(bool has_mask, uint8_t byte, uint32_t left, uint32_t lane) {
    if (!has_mask) return left >= (uint32_t)KT ? all_keys<KT>() : (1ull << left) - 1ull;
    return __ballot(lane < (uint32_t)KT && lane < left && byte != 0);
}
// -inf where the lane's row does not see the key: D element r of block st is key 32 st + (r & 3) + 8 (r >> 2) + 4 hi of the tile
__device__ __forceinline__ void hide(f32x16& sc, uint64_t live, int lim, int key0, int st, uint32_t hi) {
    const uint32_t bits = (uint32_t)(live >> (32 * st)) >> (4 * hi);
    const int last = lim - (key0 + 32 * st + 4 * (int)hi);
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int k = (r & 3) + 8 * (r >> 2);
        if (!((bits >> k) & 1u) || k > last) sc[r] = -INFINITY;
    }
}

}  // namespace sdfx_attn
