"""Calls of the training operators (csrc/attention_train*.hip, groupnorm_train.hip, geglu_train.hip) at the edge of what their documentation
allows, against float64."""
import math

import pytest
import torch

import train_ops_ref as ref
from sdfx_nerf.attention import attention
from sdfx_nerf.groupnorm import geglu, group_norm_act

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rn(dev, *shape, seed=0, dtype=F16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev)


# ---- group norm -----------------------------------------------------------------------------------------------------------------
def _moments(x, G, eps, pre=None):
    """mean and rstd [N, G] as csrc/groupnorm_train.hip writes them, and in float64."""
    import _sdfx as S
    N, C, H, W = x.shape
    w = torch.ones(C, dtype=x.dtype, device=x.device)
    y, got = torch.empty_like(x), torch.empty(N, G, 2, device=x.device)
    scratch = torch.empty(S.lib().sdfx_group_norm_train_scratch_bytes(N, H * W, C, G) // 8 + 1, dtype=torch.float64, device=x.device)
    S.call("sdfx_group_norm_train_forward", S.ptr(x), S.ptr(pre), S.ptr(w), S.ptr(w), N, H * W, C, G, eps, 0, {F16: 0, BF16: 1, F32: 2}[x.dtype], 0,
           S.ptr(y), None, S.ptr(got), S.ptr(scratch), S.stream())
    u = x.cpu().double() + (0 if pre is None else pre.cpu().double()[:, :, None, None])
    r = u.reshape(N, G, -1)
    return got.cpu().double(), r.mean(-1), (r.var(-1, unbiased=False) + eps).rsqrt()


@pytest.mark.parametrize("first", [0.0, 30.0, 300.0, -3e4])
@pytest.mark.parametrize("dtype,N,C,H,W,G,pre", [(F32, 2, 64, 64, 64, 8, False), (F32, 1, 32, 256, 256, 8, True), (F16, 1, 128, 96, 64, 32, True),
                                                 (BF16, 2, 320, 16, 16, 32, False), (F32, 1, 8, 300, 400, 1, False)])
def test_group_norm_statistics_do_not_hang_on_a_groups_first_value(dev, dtype, N, C, H, W, G, pre, first):
    """Mean and rstd to the last rounding of float32 (half a step, one more for eps as a float32 and for the roundings of double): the mean
    relative to itself or, where it is small, to the deviation."""
    x = _rn(dev, N, C, H, W, seed=1, dtype=F32)
    if first:
        x[:, ::C // G, 0, 0] = first
    x = x.to(dtype).contiguous(memory_format=torch.channels_last)
    p = _rn(dev, N, C, seed=2, dtype=dtype) if pre else None
    got, mean, rstd = _moments(x, G, 1e-5, p)
    assert float(((got[..., 1] - rstd).abs() / rstd).max()) <= 2.0 ** -23
    assert float(((got[..., 0] - mean).abs() - 2.0 ** -23 * mean.abs() - 2.0 ** -40 / rstd).max()) <= 0


@pytest.mark.parametrize("value", [0.0, 3.0, -1e6])
def test_group_norm_of_a_constant_map(dev, value):
    """No variance at all: rstd is eps ** -0.5 wherever the map lies, y is the bias and dx that of a map whose deviations are zero."""
    x = torch.full((2, 32, 9, 11), value, device=dev).contiguous(memory_format=torch.channels_last)
    got, mean, rstd = _moments(x, 4, 1e-5)
    assert torch.equal(got[..., 0], mean) and float(((got[..., 1] - rstd).abs() / rstd).max()) <= 2.0 ** -23


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("dtype,first", [(F32, 300.0), (F16, 3e4)])
def test_group_norm_and_its_gradient_beside_an_outlier(dev, dtype, first, checkpoint):
    x = _rn(dev, 2, 64, 48, 40, seed=1, dtype=F32)
    x[:, ::8, 0, 0] = first
    x = x.to(dtype).contiguous(memory_format=torch.channels_last)
    w, b, dy = _rn(dev, 64, seed=3, dtype=dtype), _rn(dev, 64, seed=4, dtype=dtype), _rn(dev, 2, 64, 48, 40, seed=5, dtype=dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = group_norm_act(leaves[0], 8, leaves[1], leaves[2], checkpoint=checkpoint)
    got = dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, leaves, dy)), y=y.detach())
    for n, (want, bound) in ref.group_norm(x, 8, w, b, dy, eight=checkpoint == "int8").items():
        ref.check(n, got[n], want, bound)


# ---- attention ------------------------------------------------------------------------------------------------------------------
def _heads(dev, B, H, N, d, seed, dtype, scale=1.0):
    return _rn(dev, B, N, H * d, seed=seed, dtype=dtype, scale=scale).view(B, N, H, d).transpose(1, 2)


def _attend(q, k, v, dy, mask=None, causal=False, scale=None):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = attention(q, k, v, mask, causal, scale)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), dy)]


def _compare(got, want, bound):
    for n, g, w, b in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(n, g, w, b)


@pytest.mark.parametrize("H,Hk,Nq,Nk,d,spread", [(4, 4, 300, 200, 64, 1.0), (4, 2, 40, 2, 40, 3.0), (2, 2, 600, 700, 128, 1.0), (2, 1, 90, 33, 160, 2.0)])
def test_fp16_attention_gradients_follow_a_loss_scale(dev, H, Hk, Nq, Nk, d, spread):
    """dy times a power of two gives the gradients times it where both are normal numbers: dv bit for bit (it knows no scale), dq and dk but for
    what float32 rounds on the way, 2^-21 of a probability, which moves one in 2^10 of the half-precision roundings of ds by 2^-11: 2^-16 of
    the 2-norm, allowed 2^-14."""
    q, k = (_heads(dev, 1, h, n, d, i, F16, spread) for i, (h, n) in enumerate(((H, Nq), (Hk, Nk)), 1))
    v, dy = _heads(dev, 1, Hk, Nk, d, 3, F16), _rn(dev, 1, Nq, H * d, seed=4)
    dy = torch.where(dy.abs() < 2.0 ** -4, torch.zeros_like(dy), dy)            # (2^-8 of it is exact in fp16)
    want = _attend(q, k, v, dy)[1:]
    for e in (-8, -3, 5, 9):
        for n, g, w in zip(("dq", "dk", "dv"), _attend(q, k, v, dy * 2.0 ** e)[1:], want):
            a, b = g.double() * 2.0 ** -e, w.double()
            both = (b.abs() * min(1.0, 2.0 ** e) >= 2.0 ** -14) & (b.abs() * max(1.0, 2.0 ** e) < 65504)
            assert both.float().mean() > 0.02, (n, e)
            assert torch.equal(a[both], b[both]) if n == "dv" else float((a - b)[both].norm() / b[both].norm()) <= 2.0 ** -14, (n, e)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gap", [9.0, 12.0, 14.0])
def test_a_row_that_one_of_two_keys_nearly_carries_keeps_its_gradient(dev, dtype, gap):
    """512 rows of two keys, one of which has a share of e^-gap: dq and dk are what that share leaves, found as p (dp - delta). dp and delta are
    float32 sums of d = 64 products of size 1, each addition off by at most half a step of the running sum: with rms 0.29 steps at random, the
    running sum of j products having a size of sqrt(j), 0.29 * 2^-23 * sqrt(64 * 64 / 2) = 1.6e-6 in dp and no more in delta: 2.2e-6 beside
    share * |dp_1 - dp_2| = share * 11. At 14 nats (8e-7) that is a quarter of the dominant key's ds, half of which energy is in dq and dk: 0.18
    of their 2-norm, allowed 0.25; at 12 and 9 nats 0.03 and 0.01 with the type's own rounding, allowed 0.05."""
    B, H, d = 64, 8, 64
    q = _rn(dev, B, H, 1, d, seed=1, dtype=F32)
    q = q * (8 / q.norm(dim=-1, keepdim=True))
    k = torch.cat([q * (gap / 8), torch.zeros_like(q)], dim=2).to(dtype)
    k[:, :, 1] = _rn(dev, B, H, d, seed=2, dtype=dtype, scale=0.05)
    q, v, dy = q.to(dtype), _rn(dev, B, H, 2, d, seed=3, dtype=dtype), _rn(dev, B, 1, H * d, seed=4, dtype=dtype)
    dy = dy * 64                                                            # (fp16: results far above 2^-24)
    got, (want, _) = _attend(q, k, v, dy), ref.attention(q, k, v, dy)
    for n, g, w in list(zip(("o", "dq", "dk", "dv"), got, want))[1:3]:
        err = float((g.cpu().double() - w).norm() / w.norm())
        assert err <= (0.25 if gap == 14.0 else 0.05), (n, err)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,Hk,Nq,Nk,spread", [(2, 2, 1024, 300, 1.0), (4, 1, 700, 130, 3.0), (3, 3, 70, 90, 8.0), (2, 1, 5, 4000, 8.0), (1, 1, 9, 1, 12.0)])
def test_a_mask_that_leaves_one_key_leaves_no_gradient_of_q_and_k(dev, dtype, H, Hk, Nq, Nk, spread):
    """Exact zeros whatever the score (up to several hundred here) and the number of rows; a second batch entry sees two keys and has gradients."""
    B, d = 2, 64
    q, k = (_heads(dev, B, h, n, d, i, dtype, spread) for i, (h, n) in enumerate(((H, Nq), (Hk, Nk)), 1))
    v, dy = _heads(dev, B, Hk, Nk, d, 3, dtype), _rn(dev, B, Nq, H * d, seed=4, dtype=dtype)
    m = torch.zeros(B, Nk, dtype=torch.bool, device=dev)
    m[:, Nk // 2] = m[1, Nk - 1] = True
    o, dq, dk, dv = got = _attend(q, k, v, dy, m)
    assert not dq[0].any() and not dk[0].any() and dv[0].any()
    assert torch.equal(o[0], v[0, :, Nk // 2].repeat_interleave(H // Hk, 0).reshape(1, -1).expand(Nq, -1))
    if Nk > 1:
        assert dq[1].any() and dk[1].any()
    if spread < 8:
        _compare(got, *ref.attention(q, k, v, dy, m))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,Hk,Nq,Nk,first,second", [(2, 2, 1024, 1024, 100, 600), (4, 2, 300, 900, 640, 800), (1, 1, 700, 200, 0, 150), (2, 1, 90, 90, 33, 90),
                                                     (1, 1, 900, 900, 0, 1)])
def test_causal_rows_between_the_first_and_the_second_key_have_no_gradient_of_q_and_k(dev, dtype, H, Hk, Nq, Nk, first, second):
    """Rows that see key `first` alone get dq = 0 and add nothing to its dk: with dy zero elsewhere dk is zero throughout."""
    d, off = 40, Nk - Nq
    q, k = (_heads(dev, 1, h, n, d, i, dtype, 3.0) for i, (h, n) in enumerate(((H, Nq), (Hk, Nk)), 1))
    v, dy = _heads(dev, 1, Hk, Nk, d, 3, dtype), _rn(dev, 1, Nq, H * d, seed=4, dtype=dtype)
    m = (torch.arange(Nk, device=dev)[None] == first) | (torch.arange(Nk, device=dev)[None] >= second)
    last = torch.arange(Nq, device=dev) + off
    lone = (last >= first) & (last < second)
    got = _attend(q, k, v, dy, m, True)
    assert not got[1][:, :, lone].any()
    _compare(got, *ref.attention(q, k, v, dy, m, True))
    only = dy * lone[None, :, None]
    o, dq, dk, dv = _attend(q, k, v, only, m, True)
    assert not dq.any() and not dk.any() and dv.any() == lone.any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,Hk,Nq,Nk,causal", [(2, 2, 64, 64, False), (2, 1, 700, 1000, False), (1, 1, 600, 600, True)])
@pytest.mark.parametrize("scale,size", [(1e-8, 1.0), (2e-7, 1.0), (1e-29, 1.0), (3e-8, 3000.0), (1e-40, 1.0)])
def test_attention_scales_of_any_smallness(dev, dtype, H, Hk, Nq, Nk, causal, scale, size):
    """Nearly equal probabilities, and large q and k whose product a small scale brings to scores of 17 (the key whose k is the query)."""
    d = 64
    k = _heads(dev, 1, Hk, Nk, d, 2, dtype, size)
    at = torch.randint(0, min(Nq, Nk), (Nq,), generator=torch.Generator().manual_seed(1)).to(dev)
    q = k.repeat_interleave(H // Hk, 1)[:, :, at].contiguous() if size > 1 else _heads(dev, 1, H, Nq, d, 1, dtype)
    v, dy = _heads(dev, 1, Hk, Nk, d, 3, dtype, 4.0), _rn(dev, 1, Nq, H * d, seed=4, dtype=dtype, scale=32.0)
    got = _attend(q, k, v, dy, None, causal, scale)
    _compare(got, *ref.attention(q, k, v, dy, None, causal, scale))
    assert got[3].any() and (size == 1.0 or (got[1].any() and got[2].any()))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_recomputes_probabilities_that_sum_to_one(dev, dtype):
    """Scores about 1000, spread by 1, one query a head, dy = 1: dv is p, whose sum over 4000 keys averages dv's roundings away. Each is off by at most
    u = 2^-11 or 2^-8 of itself, rms 0.42 u (uniform within a step, mantissas between 1 and 2); weights e^N(0, 1) make 4000 keys worth 4000 / e
    equal ones: 0.42 u / 38, and 3.5 times that over 256 heads, 2e-5 or 1.5e-4. The other part is float32's half step of the log-sum-exp, 6.1e-5 at
    1443, times log(2): 4.2e-5. Together 6e-5 or 1.9e-4, allowed 1e-4 and 2e-4."""
    B, H, Nk, d = 16, 16, 4000, 64
    q, k = _heads(dev, B, H, 1, d, 1, dtype), _heads(dev, B, H, Nk, d, 2, dtype)
    q[..., 0], k[..., 0] = 64.0, 125.0
    v, dy = _heads(dev, B, H, Nk, d, 3, dtype), torch.ones(B, 1, H * d, device=dev, dtype=dtype)
    dv = _attend(q, k, v, dy)[3]
    assert float((dv[..., 0].double().sum(-1) - 1).abs().max()) <= (1e-4 if dtype == F16 else 2e-4)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_saves_what_rounding_o_left_exactly(dev, dtype):
    """o and o_lo give the float32 output again, the log-sum-exp is whole. Probabilities enter the product in two parts, 2^-17 of them off in bf16, less in
    fp16, with float32's sums within 2^-15 of p |v|; rounding o alone is 2^-12 / 2^-9 of o off. Whole and split key axes."""
    import _sdfx as S
    import ctypes
    for Nq, Nk in ((300, 200), (3, 5000)):
        B, H, d = 1, 2, 40
        q, k, v = (_rn(dev, B, H, n, d, seed=i, dtype=dtype) for i, n in enumerate((Nq, Nk, Nk), 1))
        o = torch.empty(B, Nq, H, d, dtype=dtype, device=dev)
        lo, lse = torch.empty(B, Nq, H, d, dtype=torch.int16, device=dev), torch.empty(B, H, Nq, device=dev)
        scratch = torch.empty(max(1, S.lib().sdfx_attention_train_scratch_bytes(B, H, H, Nq, Nk, d, 0)), dtype=torch.uint8, device=dev)
        st = lambda t: (ctypes.c_uint64 * 3)(t.stride(0), t.stride(2), t.stride(1))
        S.call("sdfx_attention_train_forward", S.ptr(q), S.ptr(k), S.ptr(v), None, B, H, H, Nq, Nk, d, st(q), st(k), st(v), d ** -0.5, 0, int(dtype == BF16),
               S.ptr(o), S.ptr(lo), S.ptr(lse), S.ptr(scratch), S.stream())
        whole = ((o.float().view(torch.int32) + lo.int()).view(torch.float32)).cpu().double()
        qd, kd, vd = (t.cpu().double() for t in (q, k, v))
        s = qd @ kd.transpose(-1, -2) * d ** -0.5
        p = torch.softmax(s, -1)
        want, size = ((p @ t).transpose(1, 2) for t in (vd, vd.abs()))
        assert float(((whole - want).abs() - 2.0 ** -15 * size).max()) <= 0
        assert float((torch.logsumexp(s, -1) / math.log(2) - lse.cpu().double()).abs().max()) <= 1e-5


# ---- hooks on saved tensors -----------------------------------------------------------------------------------------------------
def _saving_calls(dev):
    C = 64
    x = _rn(dev, 2, C, 6, 7, seed=1).contiguous(memory_format=torch.channels_last)
    w, b, pre = (_rn(dev, *s, seed=i, dtype=t) for i, (s, t) in enumerate([((C,), F32), ((C,), F32), ((2, C), F16)], 2))
    q, m = _heads(dev, 2, 4, 33, 40, 5, F16), torch.arange(33, device=dev)[None].expand(2, 33) < 30
    rows = x.permute(0, 2, 3, 1).reshape(-1, C)
    return [((x, w, b, pre), lambda x, w, b, p: group_norm_act(x, 8, w, b, pre=p)), ((x, w, b), lambda x, w, b: group_norm_act(x, 8, w, b, checkpoint="int8")),
            ((q, q * 0.5, q + 1), lambda q, k, v: attention(q, k, v, m)), ((rows,), lambda x: geglu(x, "int8")), ((rows,), lambda x: geglu(x, "full"))]


@pytest.mark.parametrize("how", ["apart", "reversed", "misaligned"])
def test_saved_tensors_may_come_back_in_any_layout(dev, how):
    def unpack(t):
        if how == "apart":                                  # every second element of a wider tensor
            return torch.stack([t, torch.zeros_like(t)], -1)[..., 0]
        if how == "reversed":                               # axes in the opposite order in memory
            return t.permute(*range(t.dim() - 1, -1, -1)).contiguous().permute(*range(t.dim() - 1, -1, -1))
        return torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)
    for args, f in _saving_calls(dev):
        leaves = [t.detach().requires_grad_(True) for t in args]
        y = f(*leaves)
        want = torch.autograd.grad(y, leaves, torch.ones_like(y))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = f(*leaves)
        for a, c in zip(torch.autograd.grad(y, leaves, torch.ones_like(y)), want):
            assert torch.equal(a, c)


@pytest.mark.parametrize("how", ["shorter", "wider type", "on the host"])
def test_saved_tensors_that_come_back_as_others_are_refused(dev, how):
    unpack = {"shorter": lambda t: t[..., :-1], "wider type": lambda t: t.double(), "on the host": lambda t: t.cpu()}[how]
    for args, f in _saving_calls(dev):
        leaves = [t.detach().requires_grad_(True) for t in args]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = f(*leaves)
        with pytest.raises(RuntimeError, match="hook on saved tensors"):
            torch.autograd.grad(y, leaves, torch.ones_like(y))


# ---- many short rows ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,H,N,masked", [(2 ** 21, 8, 4, False), (2 ** 23, 8, 1, True)])
def test_attention_of_more_heads_than_a_launch_has_threads(dev, B, H, N, masked):
    """2^24 heads of 4 tokens, 2^26 of one: the first, middle and last batch entries bit for bit as a call of their own gives them."""
    d = 8
    g = torch.Generator(device=dev).manual_seed(1)
    q, k, v, dy = (torch.empty(B, N, H * d, dtype=F16, device=dev).normal_(generator=g) for _ in range(4))
    heads = lambda t: t.view(-1, N, H, d).transpose(1, 2)
    m = torch.rand(B, N, device=dev, generator=g) < 0.7 if masked else None
    got = _attend(heads(q), heads(k), heads(v), dy, m)
    for at in (0, B // 2 - 50, B - 100):
        cut = slice(at, at + 100)
        want = _attend(heads(q[cut]), heads(k[cut]), heads(v[cut]), dy[cut], None if m is None else m[cut])
        assert all(torch.equal(a[cut], c) for a, c in zip(got, want))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Nq,Nk", [(700, 300), (20, 9), (300, 700)])
def test_attention_rows_that_see_no_key_may_hold_anything(dev, dtype, Nq, Nk):
    """As the tensor operations do (tests/test_train_ops_edges.py): NaN and infinities in the queries and dy of such rows reach nothing."""
    H, Hk, d = 4, 2, 40
    q, k, v = _heads(dev, 2, H, Nq, d, 1, dtype), _heads(dev, 2, Hk, Nk, d, 2, dtype), _heads(dev, 2, Hk, Nk, d, 3, dtype)
    dy = _rn(dev, 2, Nq, H * d, seed=4, dtype=dtype)
    m = torch.ones(2, Nk, dtype=torch.bool, device=dev)
    m[0, :5] = m[1] = False
    n = max(0, Nq - Nk + 5)
    want = None
    for bad in (0.0, float("nan"), float("inf")):
        qb, dyb = q.clone(), dy.clone()
        qb[0, :, :n] = qb[1] = bad
        dyb[0, :n] = dyb[1] = bad
        got = _attend(qb, k, v, dyb, m, True)
        want = want or got
        assert all(torch.isfinite(t).all() for t in got) and all(torch.equal(a, b) for a, b in zip(got, want))
    _compare(got, *ref.attention(q, k, v, dy, m, True))


@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("shift,spread", [(0.0, 1.0), (3.0, 1.5), (-40.0, 1.0)])
def test_float32_group_norm_is_as_exact_as_its_formulas(dev, act, shift, spread):
    """The 2-norm of each error within 1.5 times that of the same formulas in float32, operation by operation, with mean and rstd rounded to float32
    (1.5: their sums run in another order)."""
    N, C, H, W, G = 2, 96, 37, 29, 8
    x = (_rn(dev, N, C, H, W, seed=1, dtype=F32) * spread + shift).contiguous(memory_format=torch.channels_last)
    w, b, dy = _rn(dev, C, seed=2, dtype=F32), _rn(dev, C, seed=3, dtype=F32) * 4, _rn(dev, N, C, H, W, seed=4, dtype=F32)
    leaf = x.detach().requires_grad_(True)
    y = group_norm_act(leaf, G, w, b, act=act)
    got = {"y": y.detach(), "dx": torch.autograd.grad(y, leaf, dy)[0]}

    def formulas(t):
        per = lambda u: u.reshape(N, G, -1)
        full = lambda u: u.expand(N, G, C // G * H * W).reshape(N, C, H, W)
        xc, wc, bc, d = (u.cpu().to(t) for u in (x, w[None, :, None, None], b[None, :, None, None], dy))
        mean = per(x.cpu().double()).mean(-1, keepdim=True)
        rstd = ((per(x.cpu().double()) - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt().to(t)
        xh = (xc - full(mean.to(t))) * full(rstd)
        z = xh * wc + bc
        sg = 1 / (1 + torch.exp(-z))
        dz = d * sg * (1 + z * (1 - sg)) if act else d
        g = dz * wc
        avg = lambda u: full(per(u.double()).mean(-1, keepdim=True).to(t))
        return {"y": z * sg if act else z, "dx": full(rstd) * (g - avg(g) - xh * avg(g * xh))}
    want, plain = formulas(torch.float64), formulas(F32)
    for n in want:
        own, base = (float((t[n].cpu().double() - want[n]).norm()) for t in (got, plain))
        assert own <= 1.5 * base, (n, own, base)


@pytest.mark.parametrize("Nq,Nk", [(300, 48), (40, 2048), (700, 900)])
@pytest.mark.parametrize("big", ["k", "q"])
def test_fp16_attention_keeps_the_digits_of_a_tiny_dy(dev, Nq, Nk, big):
    """dy of 2^-17 (fp16's subnormal numbers), v of 2^6, and k (or q) so large that dq (or dk) is a normal number all the same. p and ds are rounded once
    and the result once, sqrt(2) half steps at most in the 2-norm, and the sums: 3 allowed."""
    H, d = 2, 64
    size = {"q": 2.0 ** -10, "k": 2.0 ** 13} if big == "k" else {"q": 2.0 ** 13, "k": 2.0 ** -10}
    q, k, v = (_heads(dev, 1, H, n, d, i, F16, s) for i, (n, s) in enumerate(((Nq, size["q"]), (Nk, size["k"]), (Nk, 64.0)), 1))
    dy = _rn(dev, 1, Nq, H * d, seed=4, dtype=F32, scale=2.0 ** -17).to(F16)
    got, (want, _) = _attend(q, k, v, dy, scale=2.0 ** -6), ref.attention(q, k, v, dy, scale=2.0 ** -6)
    i = 1 if big == "k" else 2
    normal = want[i].abs() > 2.0 ** -13
    assert normal.float().mean() > 0.3
    err = float((got[i].cpu().double() - want[i])[normal].norm() / want[i][normal].norm())
    assert err <= 3 * ref.half_step(F16), err


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [8, 24, 40, 64, 72, 80, 104, 128, 160, 200, 256])
@pytest.mark.parametrize("Nq,Nk,causal,way", [(300, 200, False, "scale"), (600, 600, True, "scale"), (530, 700, True, "offset"), (33, 40, False, "offset")])
def test_attention_of_every_width_with_statistics_beyond_their_channels(dev, dtype, d, Nq, Nk, causal, way):
    """A scale of 1e-9, or scores of 140 +- 1 (202 in base 2: float32 rounds such scores, and so p, by 2e-5): dk and dv take the log-sum-exp from LDS."""
    H, Hk = 4, 2
    q, k, v = (_heads(dev, 2, h, n, d, i, dtype) for i, (h, n) in enumerate(((H, Nq), (Hk, Nk), (Hk, Nk)), 1))
    dy, m = _rn(dev, 2, Nq, H * d, seed=4, dtype=dtype), torch.rand(2, Nk, generator=torch.Generator().manual_seed(5)) < 0.8
    scale = 1e-9
    if way == "offset":
        q[..., 0], k[..., 0], scale = 16.0, 70.0, 0.125
    m = m.to(dev)
    _compare(_attend(q, k, v, dy, m, causal, scale), *ref.attention(q, k, v, dy, m, causal, scale))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("seen", [(), (8500,), (4095, 4096), (0, 8999), (255, 4111), (8998, 8999)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_few_seen_keys_anywhere_in_a_long_mask(dev, dtype, seen, causal):
    H, Nq, Nk, d = 2, 40, 9000, 40
    q, k, v = (_heads(dev, 2, H, n, d, i, dtype) for i, n in enumerate((Nq, Nk, Nk), 1))
    dy, m = _rn(dev, 2, Nq, H * d, seed=4, dtype=dtype), torch.zeros(2, Nk, dtype=torch.bool, device=dev)
    m[0, list(seen)] = True
    m[1, 5:9] = True
    got = _attend(q, k, v, dy, m, causal)
    _compare(got, *ref.attention(q, k, v, dy, m, causal))
    last = torch.arange(Nq) + Nk - Nq if causal else torch.full((Nq,), Nk - 1)
    sees = sum((last >= j).long() for j in seen) if seen else torch.zeros(Nq).long()
    assert torch.equal(got[1][0].cpu().float().abs().amax((0, 2)) > 0, sees > 1)
