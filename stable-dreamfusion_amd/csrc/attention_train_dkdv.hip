// attention_train_dkdv.hip — dk = scale ds^T q and dv = p^T dy of attention's gradient (attention_train.h). A wave owns 32 keys: k and v in
// registers, tiles of queries (q, dy, their log-sum-exp and delta) shared by the workgroup's waves in LDS, double-buffered, over every
// query head that shares the key head. Per 32 queries: s = q k^T, dp = dy v^T, p, ds, then dv^T += dy^T p, dk^T += q^T ds. A masked key
// touches nothing but its own lane, whose result is written as zero.
#include "attention_train.h"

namespace sdfx_attn {
namespace {

template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, DP <= 64 ? 2 : 1) void k_dkdv(BwdArgs a, Shape s) {
    constexpr int QT = query_tile(DP), KS = DP / 16, DT = (DP + 31) / 32, NB = QT / 32;
    typedef Tile<DP, QT, 64 * NW> L;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * L::BYTES + kTileSlack];
    __shared__ __attribute__((aligned(16))) float stat[2][2][QT];       // [buffer][shift - lse, -delta g][query]
    uint8_t* const ldsY = lds;
    uint8_t* const ldsQ = lds + 2 * L::BYTES;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, x = lane & 31u, hi = lane >> 5;
    const uint32_t per_bh = s.tiles_x * s.splits;
    const uint32_t lid = xcd_contiguous(blockIdx.x, per_bh * s.B * s.Hk);
    const uint32_t bh = lid / per_bh, rest = lid - bh * per_bh, split = rest / s.tiles_x, xt = rest - split * s.tiles_x;
    const uint32_t b = bh / s.Hk, hk = bh - b * s.Hk;
    const uint32_t wg_key = xt * NW * 32u, w0 = wg_key + wave * 32u, key = w0 + x, kc = min(key, s.Nk - 1u);
    const bool seen = key < s.Nk && (!s.mask || s.mask[(size_t)b * s.Nk + kc] != 0);
    const bool wave_on = __ballot(seen) != 0;

    typename Half<T>::v8 kf[KS], vf[KS];
    row_fragments<T, KS>(kf, static_cast<const T*>(a.k) + (size_t)b * s.k_sb + (size_t)kc * s.k_sn + (size_t)hk * s.k_sh, s.D, hi);
    row_fragments<T, KS>(vf, static_cast<const T*>(a.v) + (size_t)b * s.v_sb + (size_t)kc * s.v_sn + (size_t)hk * s.v_sh, s.D, hi);
    float g = 1.f;
    if (Half<T>::kScaled) g = grad_scale(a.rows2 + (size_t)bh * prep_blocks(s.rows), prep_blocks(s.rows), a.v2 + (size_t)bh * prep_blocks(s.Nk), prep_blocks(s.Nk), lane);

    // tiles: t = head in group * per_head + tile of queries; a causal workgroup starts each head at the first tile that sees its keys
    const uint32_t per_head = (s.Nq + QT - 1) / QT;
    const int first_q = s.causal ? (int)wg_key - s.off : 0;              // the first query that sees key wg_key
    const uint32_t skip = first_q > 0 ? min((uint32_t)first_q / QT, per_head) : 0u;
    const uint32_t t_end = min((split + 1) * s.per_split, s.group * per_head);
    auto advance = [&](uint32_t t) -> uint32_t {                                     // the first tile from t on that is not skipped
        if (skip >= per_head) return t_end;
        while (t < t_end) {
            const uint32_t i = t % per_head;
            if (i >= skip) break;
            t += skip - i;
        }
        return min(t, t_end);
    };
    // rows without a visible key (possible under a causal mask with a key mask or more queries than keys): their dy must not reach the sums
    const bool empties = s.causal && (s.mask || s.off < 0);

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) { dk[dt] = zero16(); dv[dt] = zero16(); }

    u4v rq[L::PT], ry[L::PT];
    float r_lse = 0.f, r_delta = 0.f;
    auto ask = [&](uint32_t t) {
        const uint32_t gi = t / per_head, q0 = (t - gi * per_head) * QT, head = hk * s.group + gi;
        request<L>(rq, static_cast<const T*>(a.q) + (size_t)b * s.q_sb + (size_t)head * s.q_sh, s.q_sn, q0, s.Nq, s.D, tid, 64 * NW);
        request<L>(ry, static_cast<const T*>(a.dy) + (size_t)b * s.Nq * s.H * s.D + (size_t)head * s.D, (uint64_t)s.H * s.D, q0, s.Nq, s.D, tid, 64 * NW);
        const size_t at = (size_t)bh * s.rows + (size_t)gi * s.Nq + min(q0 + lane, s.Nq - 1u);
        r_lse = lane < (uint32_t)QT && q0 + lane < s.Nq ? a.lse[at] : INFINITY;       // (every wave: the empty rows' ballot is uniform)
        r_delta = a.delta[at];
    };
    auto put = [&](uint32_t t, uint32_t buf) {
        const uint32_t q0 = (t % per_head) * QT, left = s.Nq - q0;
        uint64_t live = left >= 64u ? ~0ull : (1ull << left) - 1ull;
        if (empties) live &= __ballot(r_lse != INFINITY);
        stash<L>(ldsQ + buf * L::BYTES, rq, live, tid, 64 * NW);
        stash<L>(ldsY + buf * L::BYTES, ry, live, tid, 64 * NW);
        if (wave == 0 && lane < (uint32_t)QT) {
            stat[buf][0][lane] = Half<T>::kShift - r_lse;
            stat[buf][1][lane] = r_lse == INFINITY ? 0.f : -r_delta * g;
        }
    };

    uint32_t t = advance(split * s.per_split), buf = 0;
    if (t < t_end) { ask(t); put(t, 0); }
    __syncthreads();
    while (t < t_end) {
        const uint32_t next = advance(t + 1);
        if (next < t_end) ask(next);
        const uint8_t* qt = ldsQ + buf * L::BYTES;
        const uint8_t* yt = ldsY + buf * L::BYTES;
        const int q0 = (int)((t % per_head) * QT);
        if (wave_on && (!s.causal || q0 + QT - 1 + s.off >= (int)w0)) {
            const bool diagonal = s.causal && q0 + s.off < (int)w0 + 31;
#pragma unroll
            for (int st = 0; st < NB; st++) {
                f32x16 sc = zero16(), dp = zero16();
#pragma unroll
                for (int ks = 0; ks < KS; ks++) sc = mma(row_operand<T, L>(qt, st, ks, x, hi), kf[ks], sc);
#pragma unroll
                for (int ks = 0; ks < KS; ks++) dp = mma(row_operand<T, L>(yt, st, ks, x, hi), vf[ks], dp);
                if (diagonal) {                                          // query q0 + 32 st + 4 hi + i sees this key when it is not before it
                    const int first = (int)key - s.off - q0 - 32 * st - 4 * (int)hi;
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if ((r & 3) + 8 * (r >> 2) < first) sc[r] = -INFINITY;
                }
#pragma unroll
                for (int q4 = 0; q4 < 4; q4++) {
                    const f4 nl = *reinterpret_cast<const f4*>(&stat[buf][0][32 * st + 8 * q4 + 4 * hi]);
                    const f4 nd = *reinterpret_cast<const f4*>(&stat[buf][1][32 * st + 8 * q4 + 4 * hi]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = 4 * q4 + i;
                        sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], s.c, nl[i]));
                        dp[r] = sc[r] * __builtin_fmaf(dp[r], g, nd[i]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const typename Half<T>::v8 pf = operand<T>(sc, e), df = operand<T>(dp, e);      // (p and ds rounded to the inputs' type)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) dv[dt] = mma(col_operand<T, L>(yt, 2 * st + e, dt, lane), pf, dv[dt]);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) dk[dt] = mma(col_operand<T, L>(qt, 2 * st + e, dt, lane), df, dk[dt]);
                }
            }
        }
        if (next < t_end) put(next, buf ^ 1u);
        __syncthreads();
        t = next;
        buf ^= 1u;
    }
    if (key >= s.Nk) return;
    const float fv = Half<T>::kScaled ? 1.f / 32768.f : 1.f, fk = s.scale * fv / g;
    const size_t at = (size_t)bh * s.Nk + key, pa = ((size_t)split * s.B * s.Hk * s.Nk + at) * s.D;
    const size_t oa = (((size_t)b * s.Nk + key) * s.Hk + hk) * s.D;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) {
            const uint32_t c0 = 32u * dt + 8u * q4 + 4u * hi;
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

template <typename T, int DP, int NW> void go(const BwdArgs& a, const Shape& s, hipStream_t st) {
    hipLaunchKernelGGL((k_dkdv<T, DP, NW>), dim3(s.tiles_x * s.splits * s.B * s.Hk), dim3(64 * NW), 0, st, a, s);
}

}  // namespace

void launch_dkdv(const BwdArgs& a, const Shape& s, int bf16, int waves, hipStream_t st) { SDFX_ATTN_DISPATCH(go, a, s, st); }

}  // namespace sdfx_attn
