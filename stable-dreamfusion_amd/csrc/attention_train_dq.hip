// attention_train_dq.hip — dq = scale ds k of attention's gradient (attention_train.h). A wave owns 32 rows: q and dy in registers, the key /
// value tiles shared by the workgroup's waves in LDS, double-buffered. Per 32 keys: s^T = k q^T and dp^T = v dy^T, p = exp2(s c - lse) with the
// forward's log-sum-exp, ds = p (dp - delta) with the lane's own delta, dq^T += k^T ds^T. One pass, no row statistics to find.
// Bound: instruction issue of vector and matrix units together (2 x 8 heads, 4096 x 4096 x 40, fp16: 114 us for three products, 565 TFLOP/s; matrix units
// busy 38 % of the cycles, vector units 46 %).
// A branch around each tile's loads, to leave out its share of a masked end, cost 30 %: they are unconditional with clamped rows.
#include "attention_train.h"

namespace sdfx_attn {
namespace {

template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, DP <= 80 ? 2 : 1) void k_dq(BwdArgs a, Shape s) {
    constexpr int KT = key_tile(DP, NW), NBUF = buffers(NW), KS = DP / 16, DT = (DP + 31) / 32, NB = KT / 32;
    typedef Tile<DP, KT, 64 * NW> L;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * NBUF * L::BYTES + kTileSlack];
    uint8_t* const ldsV = lds;
    uint8_t* const ldsK = lds + NBUF * L::BYTES;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), x = lane & 31u, hi = lane >> 5;
    const uint32_t per_bh = s.tiles_x * s.splits;
    if (flat_block() >= per_bh * s.B * s.Hk) return;
    const uint32_t lid = xcd_contiguous(flat_block(), per_bh * s.B * s.Hk);
    const uint32_t bh = lid / per_bh, rest = lid - bh * per_bh, split = rest / s.tiles_x, xt = rest - split * s.tiles_x;
    const uint32_t b = bh / s.Hk, hk = bh - b * s.Hk;
    const uint32_t r0 = xt * NW * 32u, w0 = r0 + wave * 32u;
    const Row row = row_of(s, w0 + x, hk);
    const T* kb = static_cast<const T*>(a.k) + (size_t)b * s.k_sb + (size_t)hk * s.k_sh;
    const T* vb = static_cast<const T*>(a.v) + (size_t)b * s.v_sb + (size_t)hk * s.v_sh;

    typename Half<T>::v8 qf[KS], yf[KS];
    row_fragments<T, KS>(qf, static_cast<const T*>(a.q) + (size_t)b * s.q_sb + (size_t)row.qi * s.q_sn + (size_t)row.head * s.q_sh, s.D, hi);
    row_fragments<T, KS>(yf, static_cast<const T*>(a.dy) + (((size_t)b * s.Nq + row.qi) * s.H + row.head) * s.D, s.D, hi);
    const size_t at = (size_t)bh * s.rows + row.R;
    const float lse = a.lse[at], delta = a.delta[at];
    const bool few = __ballot(row.on && marked(delta)) != 0;            // (some row of the wave)
    float g = 1.f, vmax;
    if (Half<T>::kScaled) g = grad_scale(a.rows2 + (size_t)bh * prep_blocks(s.rows), prep_blocks(s.rows), a.v2 + (size_t)bh * prep_blocks(s.Nk), prep_blocks(s.Nk), lane, vmax);
    const TwoSeen two = two_seen(a, b);
    const int last = min(row.lim, (int)s.Nk - 1);
    const bool alone = last >= two.f1 && last < two.f2;
    // ds = p (dp - delta) g: g joins the exponent (p is used for nothing else), -delta starts dp's sum on the matrix cores
    const float nlse = alone ? -INFINITY : Half<T>::kShift + (Half<T>::kScaled ? __builtin_amdgcn_logf(g) : 0.f) - lse, ndelta = -delta;
    f32x16 dp0;
#pragma unroll
    for (int r = 0; r < 16; r++) dp0[r] = ndelta;

    uint32_t kend = s.Nk;
    int wave_lo = 0x7fffffff, wave_hi = 0x7fffffff;
    if (s.causal) {
        uint32_t lo, hi_q;
        query_range(s, r0, min(r0 + NW * 32u, s.rows) - 1u, lo, hi_q);
        kend = (uint32_t)max(0, min((int)s.Nk, (int)hi_q + s.off + 1));
        query_range(s, min(w0, s.rows - 1u), min(w0 + 32u, s.rows) - 1u, lo, hi_q);
        wave_lo = (int)lo + s.off; wave_hi = (int)hi_q + s.off;
    }
    const uint32_t tiles = (kend + KT - 1) / KT, t0 = split_at(tiles, split, s.splits), t1 = split_at(tiles, split + 1, s.splits);

    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt] = zero16();
    if (t0 < t1) {
        u4v rk[L::PT], rv[L::PT];
        Stage<L, 64 * NW> stk, stv;
        stk.init(s.D, s.k_sn, tid);
        stv.init(s.D, s.v_sn, tid);
        if (DP != s.D) clear_lds(lds, sizeof lds, tid, 64 * NW);
        // the next tile to request: its rows, the keys left from it on, its part of the mask
        const T *kp = kb + (size_t)t0 * KT * s.k_sn, *vp = vb + (size_t)t0 * KT * s.v_sn;
        const uint64_t k_step = (uint64_t)KT * s.k_sn, v_step = (uint64_t)KT * s.v_sn;
        const bool has_mask = s.mask != nullptr;
        const uint8_t* mp = has_mask ? s.mask + (size_t)b * s.Nk + t0 * KT : nullptr;
        uint32_t left = s.Nk - t0 * KT;
        uint8_t byte = 1;
        auto ask = [&]() {
            stk.request(rk, kp, s.k_sn, left);
            stv.request(rv, vp, s.v_sn, left);
            if (has_mask) byte = mask_byte(mp, left, lane);
        };
        ask();
        uint64_t live = live_keys<KT>(has_mask, byte, left, lane);
        stk.put(ldsK, rk, live == all_keys<KT>(), live);
        stv.put(ldsV, rv, live == all_keys<KT>(), live);
        __syncthreads();
        uint32_t buf = 0;
        int key0 = (int)(t0 * KT);
        for (uint32_t j = t0; j < t1; j++, key0 += KT) {
            if (j + 1 < t1) {
                kp += k_step; vp += v_step; mp += KT; left -= KT;
                ask();
            }
            const uint8_t* kt = ldsK + buf * L::BYTES;
            const uint8_t* vt = ldsV + buf * L::BYTES;
            if (live != 0 && key0 <= wave_hi) {
                const bool masked = live != all_keys<KT>() || key0 + KT - 1 > wave_lo;
                f32x16 sc[NB], dp[NB];
#pragma unroll
                for (int st = 0; st < NB; st++) { sc[st] = zero16(); dp[st] = dp0; }
#pragma unroll
                for (int ks = 0; ks < KS; ks++)           // (the blocks' chains in turn: a product waits for the one before it in its chain)
#pragma unroll
                    for (int st = 0; st < NB; st++) {
                        sc[st] = mma(row_operand<T, L>(kt, st, ks, x, hi), qf[ks], sc[st]);
                        dp[st] = mma(row_operand<T, L>(vt, st, ks, x, hi), yf[ks], dp[st]);
                    }
#pragma unroll
                for (int st = 0; st < NB; st++) {
                    // the transposed key operands, requested ahead of the exponentials (the compiler would read each in front of its product and wait)
                    typename Half<T>::v8 ko[2][DT];
                    if (ahead(DP)) {
#pragma unroll
                        for (int e = 0; e < 2; e++)
#pragma unroll
                            for (int dt = 0; dt < DT; dt++) ko[e][dt] = col_operand<T, L>(kt, 2 * st + e, dt, lane);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (masked) {
                        keep_branch();
                        hide(sc[st], live, row.lim, key0, st, hi);
                    }
                    __builtin_amdgcn_s_setprio(1);        // (a wave at its exponentials ahead of one that feeds the matrix cores: the two overlap)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[st][r], s.c, nlse));
                        sc[st][r] = p * dp[st][r];
                    }
                    __builtin_amdgcn_s_setprio(0);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const typename Half<T>::v8 f = operand<T>(sc[st], e);            // (ds rounded to the inputs' type)
#pragma unroll
                        for (int dt = 0; dt < DT; dt++) acc[dt] = mma(ahead(DP) ? ko[e][dt] : col_operand<T, L>(kt, 2 * st + e, dt, lane), f, acc[dt]);
                        if (few) {
                            keep_branch();
                            const typename Half<T>::v8 lo = left_over<T>(sc[st], e, f);
#pragma unroll
                            for (int dt = 0; dt < DT; dt++) acc[dt] = mma(ahead(DP) ? ko[e][dt] : col_operand<T, L>(kt, 2 * st + e, dt, lane), lo, acc[dt]);
                        }
                    }
                }
            }
            if (NBUF == 1) __syncthreads();
            if (j + 1 < t1) {
                if (NBUF == 2) buf ^= 1u;
                live = live_keys<KT>(has_mask, byte, left, lane);
                stk.put(ldsK + buf * L::BYTES, rk, live == all_keys<KT>(), live);
                stv.put(ldsV + buf * L::BYTES, rv, live == all_keys<KT>(), live);
            }
            __syncthreads();
        }
    }
    if (!row.on) return;
    const bool empty = lse == INFINITY;                       // a row that sees nothing has no gradient, whatever its dy holds
    const float f = s.scale * (Half<T>::kScaled ? 1.f / 32768.f : 1.f) / g;
    float* pp = s.splits > 1 ? a.part + ((size_t)split * s.B * s.Hk * s.rows + at) * s.D : nullptr;
    T* op = static_cast<T*>(a.dq) + (((size_t)b * s.Nq + row.qi) * s.H + row.head) * s.D;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) {
            const uint32_t c0 = 32u * dt + 8u * q4 + 4u * hi;
            if (c0 < s.D) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = empty ? 0.f : acc[dt][4 * q4 + i] * f;
                if (pp) *reinterpret_cast<f4*>(pp + c0) = f4{w[0], w[1], w[2], w[3]};
                else store4(op + c0, w[0], w[1], w[2], w[3]);
            }
        }
}

template <typename T, int DP, int NW> void go(const BwdArgs& a, const Shape& s, hipStream_t st) {
    hipLaunchKernelGGL((k_dq<T, DP, NW>), flat_grid((uint64_t)s.tiles_x * s.splits * s.B * s.Hk), dim3(64 * NW), 0, st, a, s);
}
template <typename T, int DP, int NW> void go_one(const BwdArgs& a, const Shape& s, hipStream_t st) { go<T, DP < 160 ? DP : 160, NW>(a, s, st); }

}  // namespace

void launch_dq(const BwdArgs& a, const Shape& s, int bf16, int waves, hipStream_t st) {
    if (bf16 && waves == 4) SDFX_ATTN_WIDTH(go, __bf16, 4, a, s, st);
    else if (bf16) SDFX_ATTN_WIDTH(go_one, __bf16, 1, a, s, st);
    else if (waves == 4) SDFX_ATTN_WIDTH(go, _Float16, 4, a, s, st);
    else SDFX_ATTN_WIDTH(go_one, _Float16, 1, a, s, st);
}

}  // namespace sdfx_attn
