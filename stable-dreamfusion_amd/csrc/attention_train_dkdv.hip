// attention_train_dkdv.hip — dk = scale ds^T q and dv = p^T dy of attention's gradient (attention_train.h). A wave owns 32 keys: k and v in
// registers, tiles of queries (q and dy) shared by the workgroup's waves in LDS, double-buffered, over every query head that shares the key
// head. Per 32 queries: s = q k^T, dp = dy v^T, p, ds, then dv^T += dy^T p, dk^T += q^T ds. A masked key touches nothing but its own lane,
// whose result is written as zero.
// A lane's 16 scores belong to 16 queries, so their log-sum-exps and deltas cannot be lane scalars as in dq. Read from LDS they would take
// as many cycles there as the operands (8 of 30 reads a block); instead they ride in the products: a row carries 8 extra channels, q's
// with (shift - lse) / c and dy's with -delta as sums of 16-bit parts, k's and v's with the parts' weights, powers of two. s and dp come out
// of the matrix cores complete. Three parts: 24 bits in bf16, in fp16 as many as the
// weights' range allows, at least 22 (with two, ds of a row of 2 keys that one carries by 1e4 to 1 was 8e-4 off). Two things end
// this: fp16's weights at 2^28 (a small scale makes (shift - lse) / c large), and the products' sum, which keeps float32's bits of its largest
// term: 2^-22 of the log-sum-exp, 1.7e-4 of every probability at 1443. A tile with a row beyond 2^27 or 128 leaves these channels zero and
// takes shift - lse from LDS, added by an fma.
// Bound: as dq's (2 x 8 heads, 4096 x 4096 x 40, fp16: 163 us for four products, 527 TFLOP/s; matrix units busy 37 % of the
// cycles, vector units 46 %). A workgroup takes one key head's tile and
// all the rows of its query heads, so that shared heads need no atomics; few key tiles split the rows and join in float32.
#include "attention_train.h"

namespace sdfx_attn {
namespace {

// The extra channels: part i of a value is rounded at weight w 2^(-step i), the rest goes to part i + 1.
template <typename T> struct Parts;
template <> struct Parts<_Float16> { static constexpr int N = 3, STEP = 11; };
template <> struct Parts<__bf16> { static constexpr int N = 3, STEP = 8; };
template <typename T> __device__ __forceinline__ u4v split_parts(float v, float w) {       // v = sum of parts * (w 2^(-STEP i)), w a power of two
    typename Half<T>::v8 o = {};
    float rest = v * (1.f / w);
#pragma unroll
    for (int i = 0; i < Parts<T>::N; i++) {
        o[i] = (T)rest;
        rest = i == 0 && !(__builtin_fabsf(rest) < INFINITY) ? 0.f : (rest - (float)o[i]) * (float)(1 << Parts<T>::STEP);
    }
    return __builtin_bit_cast(u4v, o);
}
template <typename T> __device__ __forceinline__ u4v part_weights(float w) {
    typename Half<T>::v8 o = {};
#pragma unroll
    for (int i = 0; i < Parts<T>::N; i++) { o[i] = (T)w; w *= 1.f / (float)(1 << Parts<T>::STEP); }
    return __builtin_bit_cast(u4v, o);
}

// CS: workgroups that share a key tile's output channels (2 at 256 channels, where dk and dv of 32 keys and the operands would fill the register file)
// EX: dv too takes the product with what the rounding of p left (marked, attention_train.h)
template <typename T, int DM, int CS, bool EX>
__global__ __launch_bounds__(256, DM <= 64 ? 2 : 1) void k_dkdv(BwdArgs a, Shape s) {
    constexpr int NW = 4, DP = (DM + 8 + 15) / 16 * 16;                  // channels with the extra ones, in whole K steps
    constexpr int QT = query_tile(DM), KS = DP / 16, DT = (DM + 31) / 32 / CS, NB = QT / 32;
    typedef Tile<DP, QT, 64 * NW> L;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * L::BYTES + kTileSlack];
    __shared__ float far_stat[2][QT];
    uint8_t* const ldsY = lds;
    uint8_t* const ldsQ = lds + 2 * L::BYTES;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), x = lane & 31u, hi = lane >> 5;
    const uint32_t per_bh = s.tiles_x * s.splits;
    if (flat_block() >= per_bh * s.B * s.Hk * CS) return;
    const uint32_t all = xcd_contiguous(flat_block(), per_bh * s.B * s.Hk * CS), lid = all / CS, dt0 = (all - lid * CS) * DT;
    const uint32_t bh = lid / per_bh, rest = lid - bh * per_bh, split = rest / s.tiles_x, xt = rest - split * s.tiles_x;
    const uint32_t b = bh / s.Hk, hk = bh - b * s.Hk;
    const uint32_t wg_key = xt * NW * 32u, w0 = wg_key + wave * 32u, key = w0 + x, kc = min(key, s.Nk - 1u);
    const bool seen = key < s.Nk && (!s.mask || s.mask[(size_t)b * s.Nk + kc] != 0);
    const bool wave_on = __ballot(seen) != 0;
    // fp16: ds g (g from grad_scale, |ds g| <= 1) times 2^15 is what the second product takes. g is put into v (`gv`, so that dp comes out with it)
    // where that is exact: not below 1, at which small values would leave fp16's normal numbers and dp no longer cancel against delta (dk of
    // rows that one of two keys carries by 12 nats, dy of 64: 10 % off), and with the largest |v g| up to 2^12. What is left of g
    // (`gr`) takes a multiplication a score. Only where |dy| |v| passes 2^28 is gv under 1: delta's parts end at 2^31, and such a v has no
    // value that gv brings under 2^-33 of the row's largest.
    constexpr float shift = Half<T>::kShift;
    float gv = 1.f, gr = 1.f, md = 1.f;
    if (Half<T>::kScaled) {
        float vmax;
        const float g = grad_scale(a.rows2 + (size_t)bh * prep_blocks(s.rows), prep_blocks(s.rows), a.v2 + (size_t)bh * prep_blocks(s.Nk), prep_blocks(s.Nk), lane, vmax);
        const float v1 = __uint_as_float(__float_as_uint(fminf(fmaxf(vmax, 1e-30f), 1e30f)) & 0x7f800000u);       // a power of two, vmax in v1 .. 2 v1
        gv = fmaxf(fminf(g, 4096.f / v1), fminf(1.f, g * 0x1p29f));
        gr = g / gv;
        md = 0.5f / gr;                                                  // >= the largest |delta gv|
    }
    // weights of the parts: (shift - lse) / c reaches 2^28 in fp16
    const float ws = Half<T>::kScaled ? 4096.f : 1.f, wd = Half<T>::kScaled ? fminf(fmaxf(md, 1.f / 8192.f), 32768.f) : 1.f;
    const float inv_c = 1.f / s.c;

    typename Half<T>::v8 kf[KS], vf[KS];
    row_fragments<T, KS>(kf, static_cast<const T*>(a.k) + (size_t)b * s.k_sb + (size_t)kc * s.k_sn + (size_t)hk * s.k_sh, s.D, hi);
    row_fragments<T, KS>(vf, static_cast<const T*>(a.v) + (size_t)b * s.v_sb + (size_t)kc * s.v_sn + (size_t)hk * s.v_sh, s.D, hi);
    if (Half<T>::kScaled) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int i = 0; i < 8; i++) vf[ks][i] = (T)((float)vf[ks][i] * gv);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
        if (16u * ks + 8u * hi == s.D) {
            kf[ks] = __builtin_bit_cast(typename Half<T>::v8, part_weights<T>(ws));
            vf[ks] = __builtin_bit_cast(typename Half<T>::v8, part_weights<T>(wd));
        }
    // channels behind the extra ones are never staged: zero (0 * whatever LDS held must not be NaN)
    clear_lds(lds, sizeof lds, tid, 64 * NW);

    // Tiles: i of a head in the group, heads in turn; a causal workgroup starts each head at the first tile that sees one of its keys.
    const uint32_t per_head = (s.Nq + QT - 1) / QT;
    const int first_q = s.causal ? (int)wg_key - s.off : 0;              // the first query that sees key wg_key
    const uint32_t skip = first_q > 0 ? min((uint32_t)first_q / QT, per_head) : 0u, useful = per_head - skip;
    const uint32_t u0 = split_at(s.group * useful, split, s.splits);
    uint32_t todo = split_at(s.group * useful, split + 1, s.splits) - u0;
    // rows without a visible key (possible under a causal mask with a key mask or more queries than keys): their dy must not reach the sums
    const bool empties = s.causal && (s.mask || s.off < 0);

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) { dk[dt] = zero16(); dv[dt] = zero16(); }

    u4v rq[L::PT], ry[L::PT];
    Stage<L, 64 * NW> stq, sty;
    const uint64_t y_sn = (uint64_t)s.H * s.D;
    stq.init(s.D, s.q_sn, tid);
    sty.init(s.D, y_sn, tid);
    float r_lse = 0.f, r_delta = 0.f;
    // the next tile to request: its queries, and its rows' statistics (their ballot is uniform: every wave loads them)
    const uint32_t gi0 = useful ? u0 / useful : 0u;
    uint32_t head = hk * s.group + gi0, ni = skip + (u0 - gi0 * useful), nq0 = ni * QT;
    const T *qp, *yp;
    size_t stat_at;
    auto start = [&]() {                                                 // of tile `ni` of query head `head`
        qp = static_cast<const T*>(a.q) + (size_t)b * s.q_sb + (size_t)head * s.q_sh + (size_t)nq0 * s.q_sn;
        yp = static_cast<const T*>(a.dy) + ((size_t)b * s.Nq + nq0) * y_sn + (size_t)head * s.D;
        stat_at = ((size_t)b * s.H + head) * s.Nq + nq0;
    };
    auto ask = [&]() {
        const uint32_t left = s.Nq - nq0, in = min(lane, left - 1u);
        stq.request(rq, qp, s.q_sn, left);
        sty.request(ry, yp, y_sn, left);
        r_lse = lane < left ? a.lse[stat_at + in] : INFINITY;
        r_delta = a.delta[stat_at + in];
    };
    auto advance = [&]() {
        nq0 += QT;
        if (++ni == per_head) {
            ni = skip; nq0 = skip * QT; head++;
            start();
        } else {
            qp += (uint64_t)QT * s.q_sn; yp += (uint64_t)QT * y_sn; stat_at += QT;
        }
    };
    // Queries ahead of `lone_end` see one key at most (two_seen): staged as zeros with a log-sum-exp of 0 they have p = 1 there and, whatever
    // ds comes to, add nothing to dk: no branch in the products' loop.
    const TwoSeen two = two_seen(a, b);
    const int lone_end = s.causal ? two.f2 - s.off : two.f2 >= (int)s.Nk ? 0x7fffffff : 0;
    bool few = false, far = false;                                       // (some row of the tile)
    auto put = [&](uint32_t buf) {
        const uint32_t left = s.Nq - nq0;
        uint64_t live = left >= 64u ? ~0ull : (1ull << left) - 1ull;
        if (empties) live &= __ballot(r_lse != INFINITY);
        const bool whole = left >= (uint32_t)QT && !empties;
        if (!EX) few = __ballot(marked(r_delta)) != 0;
        const int lone = min(lone_end - (int)nq0, 64);                   // the tile's first so many rows
        const uint64_t lone_rows = lone <= 0 ? 0ull : lone == 64 ? ~0ull : (1ull << lone) - 1ull;
        if ((int)lane < lone && r_lse < INFINITY) r_lse = 0.f;           // (not a row that sees nothing, nor a NaN)
        const float stat = shift - r_lse;
        far = __ballot(lane < (uint32_t)QT && r_lse != INFINITY && (__builtin_fabsf(stat) > 128.f || __builtin_fabsf(stat * inv_c) > 0x1p27f)) != 0;
        stq.put(ldsQ + buf * L::BYTES, rq, whole && lone <= 0, live & ~lone_rows);
        sty.put(ldsY + buf * L::BYTES, ry, whole, live);
        if (lane < (uint32_t)QT) {                                       // the rows' extra channels, one tensor's by each of two waves
            if (wave == 0) {
                *reinterpret_cast<u4v*>(ldsQ + buf * L::BYTES + lane * L::PITCH + s.D * 2u) = split_parts<T>(far ? 0.f : stat * inv_c, ws);
                if (far) far_stat[buf][lane] = stat;
            }
            if (wave == 1) *reinterpret_cast<u4v*>(ldsY + buf * L::BYTES + lane * L::PITCH + s.D * 2u) = split_parts<T>(r_lse == INFINITY ? 0.f : -r_delta * gv, wd);
        }
    };

    uint32_t buf = 0;
    if (todo) { start(); ask(); put(0); }
    __syncthreads();
    for (; todo; todo--) {
        const uint8_t* qt = ldsQ + buf * L::BYTES;
        const uint8_t* yt = ldsY + buf * L::BYTES;
        const int q0 = (int)nq0;
        const float factor = far ? 1.f : s.c;
        if (todo > 1) { advance(); ask(); }
        if (wave_on && (!s.causal || q0 + QT - 1 + s.off >= (int)w0)) {
            const bool diagonal = s.causal && q0 + s.off < (int)w0 + 31;
            f32x16 sc[NB], dp[NB];
#pragma unroll
            for (int st = 0; st < NB; st++) sc[st] = dp[st] = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ks++)               // (the blocks' chains in turn: a product waits for the one before it in its chain)
#pragma unroll
                for (int st = 0; st < NB; st++) {
                    sc[st] = mma(row_operand<T, L>(qt, st, ks, x, hi), kf[ks], sc[st]);
                    dp[st] = mma(row_operand<T, L>(yt, st, ks, x, hi), vf[ks], dp[st]);
                }
#pragma unroll
            for (int st = 0; st < NB; st++) {
                // this block's transposed operands, requested ahead of its exponentials (the compiler would read each in front of its product and wait)
                typename Half<T>::v8 yo[2][DT], qo[2][DT];
                if (ahead(DM)) {
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int dt = 0; dt < DT; dt++) {
                            yo[e][dt] = col_operand<T, L>(yt, 2 * st + e, dt0 + dt, lane);
                            qo[e][dt] = col_operand<T, L>(qt, 2 * st + e, dt0 + dt, lane);
                        }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (far) {
                    keep_branch();
#pragma unroll
                    for (int r = 0; r < 16; r++) sc[st][r] = __builtin_fmaf(sc[st][r], s.c, far_stat[buf][32 * st + (r & 3) + 8 * (r >> 2) + 4 * (int)hi]);
                }
                if (diagonal) {                                          // query q0 + 32 st + 4 hi + i sees this key when it is not before it
                    keep_branch();
                    const int first = (int)key - s.off - q0 - 32 * st - 4 * (int)hi;
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if ((r & 3) + 8 * (r >> 2) < first) sc[st][r] = -INFINITY;
                }
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    sc[st][r] = __builtin_amdgcn_exp2f(sc[st][r] * factor);
                    dp[st][r] = sc[st][r] * dp[st][r];
                }
                if (Half<T>::kScaled && gr != 1.f) {
                    keep_branch();
#pragma unroll
                    for (int r = 0; r < 16; r++) dp[st][r] *= gr;
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const typename Half<T>::v8 pf = operand<T>(sc[st], e), df = operand<T>(dp[st], e);      // (p and ds rounded to the inputs' type)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) dv[dt] = mma(ahead(DM) ? yo[e][dt] : col_operand<T, L>(yt, 2 * st + e, dt0 + dt, lane), pf, dv[dt]);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) dk[dt] = mma(ahead(DM) ? qo[e][dt] : col_operand<T, L>(qt, 2 * st + e, dt0 + dt, lane), df, dk[dt]);
                    if (EX) {
                        const typename Half<T>::v8 lo = left_over<T>(sc[st], e, pf);
#pragma unroll
                        for (int dt = 0; dt < DT; dt++) dv[dt] = mma(ahead(DM) ? yo[e][dt] : col_operand<T, L>(yt, 2 * st + e, dt0 + dt, lane), lo, dv[dt]);
                    }
                    if (EX || few) {
                        if (!EX) keep_branch();
                        const typename Half<T>::v8 lo = left_over<T>(dp[st], e, df);
#pragma unroll
                        for (int dt = 0; dt < DT; dt++) dk[dt] = mma(ahead(DM) ? qo[e][dt] : col_operand<T, L>(qt, 2 * st + e, dt0 + dt, lane), lo, dk[dt]);
                    }
                }
            }
        }
        if (todo > 1) {
            buf ^= 1u;
            put(buf);
        }
        __syncthreads();
    }
    if (key >= s.Nk) return;
    const float fv = __builtin_amdgcn_exp2f(-shift), fk = s.scale * fv / gv / gr;
    const size_t at = (size_t)bh * s.Nk + key, pa = ((size_t)split * s.B * s.Hk * s.Nk + at) * s.D;
    const size_t oa = (((size_t)b * s.Nk + key) * s.Hk + hk) * s.D;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) {
            const uint32_t c0 = 32u * (dt0 + dt) + 8u * q4 + 4u * hi;
            if (c0 < s.D) {
                float wk[4], wv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    wk[i] = seen ? dk[dt][4 * q4 + i] * fk : 0.f;
                    wv[i] = seen ? dv[dt][4 * q4 + i] * fv : 0.f;
                }
                if (s.splits > 1) {
                    *reinterpret_cast<f4*>(a.part + pa + c0) = f4{wk[0], wk[1], wk[2], wk[3]};
                    *reinterpret_cast<f4*>(a.part2 + pa + c0) = f4{wv[0], wv[1], wv[2], wv[3]};
                } else {
                    store4(static_cast<T*>(a.dk) + oa + c0, wk[0], wk[1], wk[2], wk[3]);
                    store4(static_cast<T*>(a.dv) + oa + c0, wv[0], wv[1], wv[2], wv[3]);
                }
            }
        }
}

template <typename T, int DM> void go(const BwdArgs& a, const Shape& s, hipStream_t st) {
    constexpr int CS = DM == 256 ? 2 : 1;
    const dim3 grid = flat_grid((uint64_t)s.tiles_x * s.splits * s.B * s.Hk * CS);
    if (s.exact) hipLaunchKernelGGL((k_dkdv<T, DM, CS, true>), grid, dim3(256), 0, st, a, s);
    else hipLaunchKernelGGL((k_dkdv<T, DM, CS, false>), grid, dim3(256), 0, st, a, s);
}
template <typename T> void by_width(const BwdArgs& a, const Shape& s, hipStream_t st) {
    if (s.D <= 40) go<T, 40>(a, s, st);                // (40 and the 8 extra channels are three K steps)
    else if (s.D <= 64) go<T, 64>(a, s, st);
    else if (s.D <= 80) go<T, 80>(a, s, st);
    else if (s.D <= 128) go<T, 128>(a, s, st);
    else if (s.D <= 160) go<T, 160>(a, s, st);
    else go<T, 256>(a, s, st);
}

}  // namespace

void launch_dkdv(const BwdArgs& a, const Shape& s, int bf16, hipStream_t st) {
    if (bf16) by_width<__bf16>(a, s, st);
    else by_width<_Float16>(a, s, st);
}

}  // namespace sdfx_attn
