// attention_train.hip — softmax attention that keeps what its gradient needs: the forward (one pass over the keys with the running
// maximum and sum), the small kernels around the gradient's two, the joins of split axes, and the entry points. See attention_train.h.
#include "attention_train.h"

using namespace sdfx_attn;

namespace {

// ---- forward ----------------------------------------------------------------------------------------------------------------------
// A wave owns 32 rows (of the query heads that share a key head), a workgroup of NW waves shares the key / value tiles, double-buffered
// in LDS with the loads of tile j + 1 in flight while tile j is used. splits > 1 (few rows, a long key axis): a workgroup takes a range of
// the tiles and leaves its unnormalised output, maximum and sum for k_join_o.
// Bound: narrow heads by a wave's own instructions (2 x 8 heads, 4096 x 4096 x 40, fp16: 107 us, 401 TFLOP/s; matrix units busy 29 % of the cycles, vector units 61 %. A score has 160 operations of
// products and an exponential, a maximum, a sum and a conversion; vector and matrix cycles of a wave add up to its time, two waves a SIMD
// overlap little of them: prodding the compiler's order towards that (scheduling groups, priorities) gained nothing, more waves lost to their
// fragments' reloads). One query by memory (4 x 16 heads on 4 x 4 caches of 16384 x 128: 27 us for 134 MB, 5.0 TB/s; a 2 GiB copy: 4.9).
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, DP <= 80 ? 2 : 1) void k_fwd(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                   T* __restrict__ o, short* __restrict__ o_lo, float* __restrict__ lse, float* __restrict__ part,
                                                   float* __restrict__ part_ml, Shape s) {
    constexpr int KT = key_tile(DP, NW), NBUF = buffers(NW), KS = DP / 16, DT = (DP + 31) / 32, NB = KT / 32;
    typedef Tile<DP, KT, 64 * NW> L;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * NBUF * L::BYTES + kTileSlack];
    uint8_t* const ldsK = lds;
    uint8_t* const ldsV = lds + NBUF * L::BYTES;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), x = lane & 31u, hi = lane >> 5;
    const uint32_t per_bh = s.tiles_x * s.splits;
    if (flat_block() >= per_bh * s.B * s.Hk) return;
    const uint32_t lid = xcd_contiguous(flat_block(), per_bh * s.B * s.Hk);
    const uint32_t bh = lid / per_bh, rest = lid - bh * per_bh, split = rest / s.tiles_x, xt = rest - split * s.tiles_x;
    const uint32_t b = bh / s.Hk, hk = bh - b * s.Hk;
    const uint32_t r0 = xt * NW * 32u, w0 = r0 + wave * 32u;
    const Row row = row_of(s, w0 + x, hk);
    const T* kb = k + (size_t)b * s.k_sb + (size_t)hk * s.k_sh;
    const T* vb = v + (size_t)b * s.v_sb + (size_t)hk * s.v_sh;

    typename Half<T>::v8 qf[KS];
    row_fragments<T, KS>(qf, q + (size_t)b * s.q_sb + (size_t)row.qi * s.q_sn + (size_t)row.head * s.q_sh, s.D, hi);

    // keys this workgroup needs, and the causal bounds of this wave's rows
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
    float m_run = -1e30f, l_run = 0.f;
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
                f32x16 sc[NB];
#pragma unroll
                for (int st = 0; st < NB; st++) {
                    sc[st] = zero16();
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) sc[st] = mma(row_operand<T, L>(kt, st, ks, x, hi), qf[ks], sc[st]);
                }
                if (live != all_keys<KT>() || key0 + KT - 1 > wave_lo) {
                    keep_branch();
#pragma unroll
                    for (int st = 0; st < NB; st++) hide(sc[st], live, row.lim, key0, st, hi);
                }
                // the value operands, requested ahead of the softmax (the compiler would read each in front of its product and wait)
                typename Half<T>::v8 vo[2 * NB][DT];
                if (ahead(DP)) {
#pragma unroll
                    for (int e = 0; e < 2 * NB; e++)
#pragma unroll
                        for (int dt = 0; dt < DT; dt++) vo[e][dt] = col_operand<T, L>(vt, e, dt, lane);
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(1);            // (a wave in its softmax ahead of one that feeds the matrix cores: the two overlap)
                float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    mx = fmaxf(mx, sc[0][r]);
                    if (NB == 2) mx1 = fmaxf(mx1, sc[NB - 1][r]);
                }
                mx = fmaxf(mx, mx1);
                mx = max_halves(mx) * s.c;
                if (__ballot(mx > m_run)) {               // (some row has a new maximum: rare after the first tiles)
                    const float m_new = fmaxf(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
                    m_run = m_new;
                    l_run *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int r = 0; r < 16; r++) acc[dt][r] *= alpha;
                }
                float sum0 = 0.f, sum1 = 0.f;
                typename Half<T>::v8 pf[2 * NB];
#pragma unroll
                for (int st = 0; st < NB; st++) {
#pragma unroll
                    for (int r = 0; r < 16; r += 2) {
                        sc[st][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[st][r], s.c, -m_run));
                        sc[st][r + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[st][r + 1], s.c, -m_run));
                        sum0 += sc[st][r]; sum1 += sc[st][r + 1];
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        pf[2 * st + e] = operand<T>(sc[st], e);          // (the probabilities' rounding: half a unit of each, as the inputs')
#pragma unroll
                        for (int dt = 0; dt < DT; dt++) acc[dt] = mma(ahead(DP) ? vo[2 * st + e][dt] : col_operand<T, L>(vt, 2 * st + e, dt, lane), pf[2 * st + e], acc[dt]);
                    }
                }
                l_run += sum0 + sum1;
                // What that rounding left, where few keys carry a row: it shows in o, and the backward's delta is taken from o: the rounding of n
                // equal probabilities is 1 / sqrt(n) of ds's own (4 of them, 2 a lane: half of it). In a long flat row only the first tiles
                // take this (4096 x 40: 1 us; a bound of 16 cost 10). With or without a gradient to come: the same o.
                if (__ballot(l_run < 0.5f * s.few)) {
                    keep_branch();
#pragma unroll
                    for (int st = 0; st < NB; st++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const typename Half<T>::v8 lo = left_over<T>(sc[st], e, pf[2 * st + e]);
#pragma unroll
                            for (int dt = 0; dt < DT; dt++) acc[dt] = mma(ahead(DP) ? vo[2 * st + e][dt] : col_operand<T, L>(vt, 2 * st + e, dt, lane), lo, acc[dt]);
                        }
                }
                __builtin_amdgcn_s_setprio(0);
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
    const float l = sum_halves(l_run);
    if (!row.on) return;
    const size_t at = (size_t)bh * s.rows + row.R;                 // = (b, head, query) of [B, H, Nq]
    if (s.splits > 1) {
        const size_t pa = (size_t)split * s.B * s.Hk * s.rows + at;
        if (hi == 0) { part_ml[2 * pa] = m_run; part_ml[2 * pa + 1] = l; }
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint32_t c0 = 32u * dt + 8u * g + 4u * hi;
                if (c0 < s.D) *reinterpret_cast<f4*>(part + pa * s.D + c0) = f4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
            }
        return;
    }
    // a row that sees nothing: zero, and a log-sum-exp of +inf, at which the backward's exp2(s - lse) is 0
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    if (lse && hi == 0) lse[at] = l > 0.f ? m_run + __builtin_amdgcn_logf(l) : (l == l ? INFINITY : l);
    const bool mark = l > 0.f && l < s.few;
    T* op = o + (((size_t)b * s.Nq + row.qi) * s.H + row.head) * s.D;
    short* lp = o_lo ? o_lo + (((size_t)b * s.Nq + row.qi) * s.H + row.head) * s.D : nullptr;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const uint32_t c0 = 32u * dt + 8u * g + 4u * hi;
            if (c0 < s.D) {
                float f[4];
#pragma unroll
                for (int i = 0; i < 4; i++) f[i] = acc[dt][4 * g + i] * inv;
                store4(op + c0, f[0], f[1], f[2], f[3]);
                if (lp) store_rest4<T>(lp + c0, f, c0 == 0, mark);
            }
        }
}

// o of the splits of each row: D / 4 channel quads x `parts` ranges of the splits are the threads of a row, the ranges added in order through LDS
template <typename T>
__global__ __launch_bounds__(256) void k_join_o(const float* __restrict__ part, const float* __restrict__ ml, Shape s, uint32_t parts, T* __restrict__ o,
                                               short* __restrict__ o_lo, float* __restrict__ lse) {
    __shared__ f4 red[256];
    __shared__ float redl[256], redm[256];
    const uint32_t quads = s.D / 4, per = quads * parts, rows_here = 256u / per;
    const uint64_t total = (uint64_t)s.B * s.H * s.Nq;
    const uint32_t local = threadIdx.x / per, in_row = threadIdx.x - local * per, pt = in_row / quads, c0 = (in_row - pt * quads) * 4;
    const uint64_t r = (uint64_t)blockIdx.x * rows_here + local;
    const bool on = local < rows_here && r < total;
    float m = -1e30f, l = 0.f;
    f4 a = {0.f, 0.f, 0.f, 0.f};
    if (on) {
        const uint32_t n = (s.splits + parts - 1) / parts, i1 = min((pt + 1) * n, s.splits);
        for (uint32_t i = pt * n; i < i1; i += 4) {               // four splits a trip, loaded together; the sum follows their maximum
            float mi[4], li[4];
            f4 p[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) {
                const uint64_t at = min(i + u, i1 - 1u) * total + r;
                mi[u] = ml[2 * at];
                li[u] = i + u < i1 ? ml[2 * at + 1] : 0.f;
                p[u] = *reinterpret_cast<const f4*>(part + at * s.D + c0);
            }
            const float mn = fmaxf(fmaxf(fmaxf(mi[0], mi[1]), fmaxf(mi[2], mi[3])), m), alpha = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
            a = a * alpha;
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) {
                const float w = li[u] == 0.f ? 0.f : __builtin_amdgcn_exp2f(mi[u] - mn);                          // (0: nothing seen in this range)
                l = __builtin_fmaf(w, li[u], l);
#pragma unroll
                for (int j = 0; j < 4; j++) a[j] = __builtin_fmaf(w, p[u][j], a[j]);
            }
        }
    }
    red[threadIdx.x] = a;
    redl[threadIdx.x] = l;
    redm[threadIdx.x] = m;
    __syncthreads();
    if (!on || pt) return;
    for (uint32_t i = 1; i < parts; i++) m = fmaxf(m, redm[threadIdx.x + i * quads]);
    l = 0.f;
    a = f4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t i = 0; i < parts; i++) {
        const float w = __builtin_amdgcn_exp2f(redm[threadIdx.x + i * quads] - m);
        a += red[threadIdx.x + i * quads] * w;
        l = __builtin_fmaf(redl[threadIdx.x + i * quads], w, l);
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    const uint32_t bh = (uint32_t)(r / s.Nq), qi = (uint32_t)(r - (uint64_t)bh * s.Nq), b = bh / s.H, h = bh - b * s.H;
    const size_t at = (((size_t)b * s.Nq + qi) * s.H + h) * s.D + c0;
    if (lse && c0 == 0) lse[r] = l > 0.f ? m + __builtin_amdgcn_logf(l) : (l == l ? INFINITY : l);
    const float f[4] = {a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv};
    store4(o + at, f[0], f[1], f[2], f[3]);
    if (o_lo) store_rest4<T>(o_lo + at, f, c0 == 0, l > 0.f && l < s.few);
}

// out[b, n, h, :] = sum over splits of part[split][b, h, n, :], in order, for each of the gradients that were split (blockIdx.y)
struct JoinSum { const float* part; void* out; uint32_t splits, H, N; };
struct JoinSums { JoinSum of[3]; };
template <typename T>
__global__ __launch_bounds__(256) void k_join_sum(JoinSums js, uint32_t B, uint32_t D) {
    const JoinSum j = js.of[blockIdx.y];
    const uint32_t per = D / 4;
    const uint64_t total = (uint64_t)B * j.H * j.N, id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= total * per) return;
    const uint64_t r = id / per;
    const uint32_t c0 = (uint32_t)(id - r * per) * 4;
    f4 a = {0.f, 0.f, 0.f, 0.f};
    const float* p = j.part + r * D + c0;
    const uint64_t step = total * D;
    for (uint32_t i = 0; i < j.splits; i += 8) {                  // eight splits a trip, loaded together; added in order
        f4 v[8];
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) v[u] = *reinterpret_cast<const f4*>(p + min(i + u, j.splits - 1u) * step);
#pragma unroll
        for (uint32_t u = 0; u < 8; u++)
            if (i + u < j.splits) a += v[u];
    }
    const uint32_t bh = (uint32_t)(r / j.N), n = (uint32_t)(r - (uint64_t)bh * j.N), b = bh / j.H, h = bh - b * j.H;
    store4(static_cast<T*>(j.out) + (((size_t)b * j.N + n) * j.H + h) * D + c0, a[0], a[1], a[2], a[3]);
}

// ---- ahead of the gradient's kernels ---------------------------------------------------------------------------------------------
// delta[b, h, i] = sum over channels of dy o, o as the forward had it ahead of its rounding (o_rest), without which ds = p (dp - delta) of a
// peaked row loses the digits the subtraction cancels (bf16, scores with a deviation of 4: dq 5.8e-3 off instead of 2.4e-3). Also the
// block maxima of |dy row|^2 and |v row|^2 that grad_scale reads (fp16), and with a mask each batch entry's first two keys (two_seen).
// LR lanes a row.
__device__ __forceinline__ void find_two(const uint8_t* __restrict__ mask, uint32_t Nk, uint32_t* lds, uint32_t* __restrict__ two) {
    if (threadIdx.x < 2) lds[threadIdx.x] = Nk;
    uint32_t f1 = Nk, f2 = Nk;                                    // of the keys this thread has looked at
    for (uint32_t k0 = 0; k0 < Nk; k0 += 256 * 16) {              // sixteen a trip, loaded together; every thread leaves after the trip that found two
        uint8_t m[16];
#pragma unroll
        for (uint32_t u = 0; u < 16; u++) m[u] = mask[min(k0 + u * 256 + threadIdx.x, Nk - 1u)];
#pragma unroll
        for (uint32_t u = 0; u < 16; u++) {
            const uint32_t k = k0 + u * 256 + threadIdx.x;
            if (k >= Nk || !m[u]) continue;
            if (f1 == Nk) f1 = k;
            else if (f2 == Nk) f2 = k;
        }
        if (__syncthreads_count(f1 < Nk) + __syncthreads_count(f2 < Nk) >= 2) break;
    }
    __syncthreads();
    atomicMin(&lds[0], f1);
    __syncthreads();
    atomicMin(&lds[1], f1 == lds[0] ? f2 : f1);
    __syncthreads();
    if (threadIdx.x < 2) two[threadIdx.x] = lds[threadIdx.x];
}
template <typename T, int LR>
__global__ __launch_bounds__(256) void k_prep(const T* __restrict__ v, const T* __restrict__ o, const short* __restrict__ o_lo, const T* __restrict__ dy,
                                             const float* __restrict__ lse, Shape s, float* __restrict__ delta, float* __restrict__ rows2, float* __restrict__ v2,
                                             uint32_t* __restrict__ seen2) {
    __shared__ float red[256 / LR];
    __shared__ uint32_t two[2];
    const uint32_t nr = prep_blocks(s.rows), nv = prep_blocks(s.Nk), bh_n = s.B * s.Hk;
    const uint32_t masks = s.mask ? s.B : 0u;          // the first workgroups take a mask each (a chain of latencies: last, it cost 4 us)
    if (flat_block() < masks) {
        find_two(s.mask + (size_t)flat_block() * s.Nk, s.Nk, two, seen2 + 2 * flat_block());
        return;
    }
    const uint32_t block = flat_block() - masks;
    if (block >= bh_n * (nr + (Half<T>::kScaled ? nv : 0))) return;
    const bool of_v = block >= bh_n * nr;
    const uint32_t id = of_v ? block - bh_n * nr : block, per = of_v ? nv : nr;
    const uint32_t bh = id / per, blk = id - bh * per, b = bh / s.Hk, hk = bh - b * s.Hk;
    const uint32_t lr = threadIdx.x % LR, c0 = lr * 8u;
    const uint32_t n = of_v ? s.Nk : s.rows, end = min((blk + 1) * kPrepRows, n);
    float most = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < (kPrepRows * LR + 255) / 256; i++) {
        const uint32_t r = blk * kPrepRows + threadIdx.x / LR + i * (256 / LR);
        if (r >= end) continue;
        float d = 0.f, q = 0.f;
        size_t at = 0;
        uint32_t mark = 0;
        if (of_v) {
            if ((!s.mask || s.mask[(size_t)b * s.Nk + r]) && c0 < s.D) {
                const typename Half<T>::v8 a = *reinterpret_cast<const typename Half<T>::v8*>(v + (size_t)b * s.v_sb + (size_t)r * s.v_sn + (size_t)hk * s.v_sh + c0);
#pragma unroll
                for (int i = 0; i < 8; i++) q = __builtin_fmaf((float)a[i], (float)a[i], q);
            }
        } else {
            const uint32_t g = r / s.Nq, qi = r - g * s.Nq;
            at = (((size_t)b * s.Nq + qi) * s.H + hk * s.group + g) * s.D + c0;
            if (c0 < s.D) {
                const typename Half<T>::v8 y = *reinterpret_cast<const typename Half<T>::v8*>(dy + at), a = *reinterpret_cast<const typename Half<T>::v8*>(o + at);
                const s8 l = *reinterpret_cast<const s8*>(o_lo + at);
                mark = (uint32_t)l[0] & 1u;                       // (the row's in the lane of its first channel)
                const bool on = lse[(size_t)bh * s.rows + r] != INFINITY;          // (the dy of a row that sees nothing may be anything)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float f = (float)y[i];
                    d = __builtin_fmaf(f, o_whole<T>(a[i], l[i]), d);
                    q = __builtin_fmaf(f, f, q);
                }
                if (!on) d = q = 0.f;
            }
        }
#pragma unroll
        for (int w = LR / 2; w >= 1; w >>= 1) { d += __shfl_xor(d, w, 64); q += __shfl_xor(q, w, 64); }
        if (!of_v && lr == 0) delta[(size_t)bh * s.rows + r] = __uint_as_float((__float_as_uint(d) & ~1u) | mark);
        most = fmaxf(most, q);
    }
    if (!Half<T>::kScaled) return;
    if (lr == 0) red[threadIdx.x / LR] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t i = 1; i < 256 / LR; i++) most = fmaxf(most, red[i]);
        (of_v ? v2 : rows2)[(size_t)bh * per + blk] = most;
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------------------------
// Workgroups of 4 waves share their tiles; 32 rows or fewer (a few queries against a long cache) take one wave each. Where that leaves CUs
// without work the other axis is split, two tiles at least to a workgroup: a split costs float32 partials and a launch that adds them (2 x 12
// causal rows of 1001 x 64 make 192 workgroups: forward 31 us whole, 19 + 7 in three splits).
constexpr uint32_t kCus = 256;
void plan(Shape& s, uint32_t along, uint32_t other_tiles, int waves) {
    s.tiles_x = div_up(along, 32u * waves);
    const uint64_t base = (uint64_t)s.tiles_x * s.B * s.Hk, want = waves == 4 ? 2 * kCus : 8 * kCus;
    uint64_t splits = 2 * base >= want ? 1 : (want + base - 1) / base;
    const uint64_t most = other_tiles / 2 ? other_tiles / 2 : 1;
    if (splits > most) splits = most;
    s.splits = (uint32_t)splits;
}
void plan_rows(Shape& s, int& waves) {          // forward, dq
    const int dp = padded(s.D);
    waves = s.rows <= 32 && dp <= 160 ? 1 : 4;
    plan(s, s.rows, div_up(s.Nk, key_tile(dp, waves)), waves);
}
void plan_keys(Shape& s) { plan(s, s.Nk, s.group * div_up(s.Nq, query_tile((int)s.D)), 4); }

template <typename T, int DP, int NW>
void launch_fwd(const void* q, const void* k, const void* v, void* o, void* o_lo, float* lse, float* part, float* ml, const Shape& s, hipStream_t st) {
    hipLaunchKernelGGL((k_fwd<T, DP, NW>), flat_grid((uint64_t)s.tiles_x * s.splits * s.B * s.Hk), dim3(64 * NW), 0, st, static_cast<const T*>(q), static_cast<const T*>(k),
                       static_cast<const T*>(v), static_cast<T*>(o), static_cast<short*>(o_lo), lse, part, ml, s);
}
// (one wave alone: head widths up to 160; see plan_rows)
template <typename T, int DP, int NW>
void launch_one(const void* q, const void* k, const void* v, void* o, void* o_lo, float* lse, float* part, float* ml, const Shape& s, hipStream_t st) {
    launch_fwd<T, DP < 160 ? DP : 160, NW>(q, k, v, o, o_lo, lse, part, ml, s, st);
}
template <typename T> void join_o(const float* part, const float* ml, const Shape& s, void* o, void* o_lo, float* lse, hipStream_t st) {
    const uint32_t quads = s.D / 4;
    uint32_t parts = 256 / quads, most = (s.splits + 3) / 4;               // four splits to a thread
    if (parts > most) parts = most;
    const uint32_t rows_here = 256 / (quads * parts);
    const uint64_t n = (uint64_t)s.B * s.H * s.Nq;
    hipLaunchKernelGGL(k_join_o<T>, dim3((uint32_t)((n + rows_here - 1) / rows_here)), dim3(256), 0, st, part, ml, s, parts, static_cast<T*>(o),
                       static_cast<short*>(o_lo), lse);
}
template <typename T> void prep(const void* v, const void* o, const void* o_lo, const void* dy, const float* lse, const Shape& s, float* delta, float* rows2, float* v2, uint32_t* seen2, hipStream_t st) {
    const dim3 grid = flat_grid((uint64_t)s.B * s.Hk * (prep_blocks(s.rows) + (Half<T>::kScaled ? prep_blocks(s.Nk) : 0)) + (s.mask ? s.B : 0));
    const T *vp = static_cast<const T*>(v), *op = static_cast<const T*>(o), *yp = static_cast<const T*>(dy);
    const short* lp = static_cast<const short*>(o_lo);
    if (s.D <= 64) hipLaunchKernelGGL((k_prep<T, 8>), grid, dim3(256), 0, st, vp, op, lp, yp, lse, s, delta, rows2, v2, seen2);
    else if (s.D <= 128) hipLaunchKernelGGL((k_prep<T, 16>), grid, dim3(256), 0, st, vp, op, lp, yp, lse, s, delta, rows2, v2, seen2);
    else hipLaunchKernelGGL((k_prep<T, 32>), grid, dim3(256), 0, st, vp, op, lp, yp, lse, s, delta, rows2, v2, seen2);
}

const char* shape_error(uint32_t B, uint32_t H, uint32_t Hk, uint32_t Nq, uint32_t Nk, uint32_t D) {
    if (!B || !H || !Hk || !Nq || !Nk) return "empty problem";
    if (H % Hk) return "the key heads do not divide the query heads";
    if (D == 0 || D % 8 || D > 256) return "the head width must be a multiple of 8 up to 256";
    if (Nq >= 0x40000000u || Nk >= 0x40000000u || (uint64_t)(H / Hk) * Nq >= 0x40000000u) return "more than 2^30 queries or keys";
    if ((uint64_t)B * H * ((uint64_t)Nq + Nk) >= 0x40000000ull) return "more than 2^30 rows";
    if ((uint64_t)H * D >= (1u << 24)) return "more than 2^24 channels";
    return nullptr;
}
void fill(Shape& s, uint32_t B, uint32_t H, uint32_t Hk, uint32_t Nq, uint32_t Nk, uint32_t D) {
    memset(&s, 0, sizeof s);
    s.B = B; s.H = H; s.Hk = Hk; s.Nq = Nq; s.Nk = Nk; s.D = D;
    s.group = H / Hk; s.rows = s.group * Nq;
    s.exact = s.rows <= 512 || Nk <= 128;
    s.few = s.exact ? INFINITY : 4.f;
}
void fill_call(Shape& s, const uint64_t* qs, const uint64_t* ks, const uint64_t* vs, const void* mask, float scale, int causal) {
    s.q_sb = qs[0]; s.q_sn = qs[1]; s.q_sh = qs[2];
    s.k_sb = ks[0]; s.k_sn = ks[1]; s.k_sh = ks[2];
    s.v_sb = vs[0]; s.v_sn = vs[1]; s.v_sh = vs[2];
    s.mask = static_cast<const uint8_t*>(mask);
    s.causal = causal != 0;
    s.off = (int)s.Nk - (int)s.Nq;
    s.scale = scale;
    s.c = scale * 1.4426950408889634f;
}
bool strides_ok(const uint64_t* a, const uint64_t* b, const uint64_t* c) {
    uint64_t all = 0;
    for (int i = 0; i < 3; i++) all |= a[i] | b[i] | c[i];
    const uint64_t token = a[1] | b[1] | c[1];          // (offsets inside a tile of 64 rows are 32-bit)
    return all % 8 == 0 && token < (1ull << 24);
}
uint64_t up16(uint64_t floats) { return (floats + 3) / 4 * 4; }
struct BwdLayout { uint64_t rows2, v2, seen2, pq, pk, pv, total; };   // float offsets behind delta
BwdLayout bwd_layout(const Shape& s0) {
    Shape a = s0, b = s0;
    int waves;
    plan_rows(a, waves);
    plan_keys(b);
    const uint64_t heads = (uint64_t)s0.B * s0.Hk;
    BwdLayout l;
    l.rows2 = up16(heads * s0.rows);
    l.v2 = l.rows2 + up16(heads * prep_blocks(s0.rows));
    l.seen2 = l.v2 + up16(heads * prep_blocks(s0.Nk));
    l.pq = l.seen2 + up16(2ull * s0.B);
    l.pk = l.pq + (a.splits > 1 ? a.splits * heads * s0.rows * s0.D : 0);
    const uint64_t one = b.splits > 1 ? b.splits * heads * s0.Nk * s0.D : 0;
    l.pv = l.pk + one;
    l.total = l.pv + one;
    return l;
}

}  // namespace

extern "C" {

uint64_t sdfx_attention_train_scratch_bytes(uint32_t B, uint32_t H, uint32_t Hk, uint32_t Nq, uint32_t Nk, uint32_t D, int backward) {
    if (shape_error(B, H, Hk, Nq, Nk, D)) return 0;
    Shape s;
    fill(s, B, H, Hk, Nq, Nk, D);
    if (backward) return bwd_layout(s).total * 4;
    int waves;
    plan_rows(s, waves);
    return s.splits > 1 ? ((uint64_t)s.splits * B * s.Hk * s.rows * (D + 2)) * 4 : 0;
}

int sdfx_attention_train_forward(const void* q, const void* k, const void* v, const void* key_mask, uint32_t B, uint32_t H, uint32_t Hk, uint32_t Nq,
                                 uint32_t Nk, uint32_t D, const uint64_t* q_strides, const uint64_t* k_strides, const uint64_t* v_strides, float scale,
                                 int causal, int bf16, void* o, void* o_lo, float* lse, float* scratch, sdfx_stream_t stream) {
    SDFX_REQUIRE(q && k && v && o && q_strides && k_strides && v_strides, "attention_train_forward: null pointer");
    const char* e = shape_error(B, H, Hk, Nq, Nk, D);
    SDFX_REQUIRE(!e, "attention_train_forward: %s (B=%u H=%u Hk=%u Nq=%u Nk=%u D=%u)", e, B, H, Hk, Nq, Nk, D);
    SDFX_REQUIRE(scale >= 1e-30f && scale <= 1e30f, "attention_train_forward: the scale must lie in 1e-30 .. 1e30");
    SDFX_REQUIRE(strides_ok(q_strides, k_strides, v_strides) && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                 reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(o_lo) | reinterpret_cast<uintptr_t>(scratch)) % 16) == 0,
                 "attention_train_forward: rows must be 16-byte aligned, token strides below 2^24");
    Shape s;
    fill(s, B, H, Hk, Nq, Nk, D);
    fill_call(s, q_strides, k_strides, v_strides, key_mask, scale, causal);
    int waves;
    plan_rows(s, waves);
    SDFX_REQUIRE(s.splits == 1 || scratch, "attention_train_forward: this shape needs scratch");
    float* ml = s.splits > 1 ? scratch + (uint64_t)s.splits * B * s.Hk * s.rows * D : nullptr;
    hipStream_t st = as_stream(stream);
    if (bf16 && waves == 4) SDFX_ATTN_WIDTH(launch_fwd, __bf16, 4, q, k, v, o, o_lo, lse, scratch, ml, s, st);
    else if (bf16) SDFX_ATTN_WIDTH(launch_one, __bf16, 1, q, k, v, o, o_lo, lse, scratch, ml, s, st);
    else if (waves == 4) SDFX_ATTN_WIDTH(launch_fwd, _Float16, 4, q, k, v, o, o_lo, lse, scratch, ml, s, st);
    else SDFX_ATTN_WIDTH(launch_one, _Float16, 1, q, k, v, o, o_lo, lse, scratch, ml, s, st);
    if (s.splits > 1) {
        if (bf16) join_o<__bf16>(scratch, ml, s, o, o_lo, lse, st);
        else join_o<_Float16>(scratch, ml, s, o, o_lo, lse, st);
    }
    return check_launch("attention_train_forward");
}

int sdfx_attention_train_backward(const void* q, const void* k, const void* v, const void* key_mask, const void* o, const void* o_lo, const float* lse,
                                  const void* dy, uint32_t B, uint32_t H, uint32_t Hk, uint32_t Nq, uint32_t Nk, uint32_t D, const uint64_t* q_strides,
                                  const uint64_t* k_strides, const uint64_t* v_strides, float scale, int causal, int bf16, void* dq, void* dk, void* dv,
                                  float* scratch, sdfx_stream_t stream) {
    SDFX_REQUIRE(q && k && v && o && o_lo && lse && dy && scratch && q_strides && k_strides && v_strides, "attention_train_backward: null pointer");
    SDFX_REQUIRE(!dk == !dv, "attention_train_backward: dk and dv come together");
    const char* e = shape_error(B, H, Hk, Nq, Nk, D);
    SDFX_REQUIRE(!e, "attention_train_backward: %s (B=%u H=%u Hk=%u Nq=%u Nk=%u D=%u)", e, B, H, Hk, Nq, Nk, D);
    SDFX_REQUIRE(scale >= 1e-30f && scale <= 1e30f, "attention_train_backward: the scale must lie in 1e-30 .. 1e30");
    SDFX_REQUIRE(strides_ok(q_strides, k_strides, v_strides) && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                 reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(o_lo) | reinterpret_cast<uintptr_t>(dy) |
                 reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) | reinterpret_cast<uintptr_t>(scratch)) % 16) == 0,
                 "attention_train_backward: rows must be 16-byte aligned, token strides below 2^24");
    Shape s;
    fill(s, B, H, Hk, Nq, Nk, D);
    fill_call(s, q_strides, k_strides, v_strides, key_mask, scale, causal);
    const BwdLayout l = bwd_layout(s);
    hipStream_t st = as_stream(stream);
    BwdArgs a;
    a.q = q; a.k = k; a.v = v; a.dy = dy; a.lse = lse;
    a.delta = scratch; a.rows2 = scratch + l.rows2; a.v2 = scratch + l.v2;
    a.dq = dq; a.dk = dk; a.dv = dv;
    uint32_t* seen2 = reinterpret_cast<uint32_t*>(scratch + l.seen2);
    a.seen2 = s.mask ? seen2 : nullptr;
    if (bf16) prep<__bf16>(v, o, o_lo, dy, lse, s, scratch, scratch + l.rows2, scratch + l.v2, seen2, st);
    else prep<_Float16>(v, o, o_lo, dy, lse, s, scratch, scratch + l.rows2, scratch + l.v2, seen2, st);
    JoinSums js;
    uint32_t joins = 0;
    uint64_t most = 0;
    auto join = [&](const float* part, void* out, uint32_t splits, uint32_t heads, uint32_t n) {
        if (splits == 1) return;
        js.of[joins++] = {part, out, splits, heads, n};
        if ((uint64_t)heads * n > most) most = (uint64_t)heads * n;
    };
    if (dk) {
        Shape t = s;
        plan_keys(t);
        a.part = scratch + l.pk; a.part2 = scratch + l.pv;
        launch_dkdv(a, t, bf16, st);
        join(a.part, dk, t.splits, Hk, Nk);
        join(a.part2, dv, t.splits, Hk, Nk);
    }
    if (dq) {
        Shape t = s;
        int waves;
        plan_rows(t, waves);
        a.part = scratch + l.pq; a.part2 = nullptr;
        launch_dq(a, t, bf16, waves, st);
        join(a.part, dq, t.splits, H, Nq);
    }
    if (joins) {
        const dim3 grid((uint32_t)((most * B * (D / 4) + 255) / 256), joins);
        if (bf16) hipLaunchKernelGGL(k_join_sum<__bf16>, grid, dim3(256), 0, st, js, B, D);
        else hipLaunchKernelGGL(k_join_sum<_Float16>, grid, dim3(256), 0, st, js, B, D);
    }
    return check_launch("attention_train_backward");
}

}  // extern "C"
