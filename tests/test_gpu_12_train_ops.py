"""csrc/attention_train*.hip, groupnorm_train.hip and geglu_train.hip against float64 with elementwise bounds (tests/train_ops_ref.py)."""
import pytest
import torch

import train_ops_ref as ref
from sdfx_nerf.attention import attention
from sdfx_nerf.groupnorm import eight_bits, geglu, group_norm_act

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rn(dev, *shape, seed=0, dtype=F16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev)


def _heads(dev, B, H, N, d, seed, dtype, scale=1.0):
    """[B, H, N, d] as the transformer blocks form it: a projection's [B, N, H d] output viewed."""
    return _rn(dev, B, N, H * d, seed=seed, dtype=dtype, scale=scale).view(B, N, H, d).transpose(1, 2)


def _mask(dev, kind, B, Nk, seed=7):
    if kind == "none":
        return None
    g = torch.Generator().manual_seed(seed)
    if kind == "holes":
        return (torch.rand(B, Nk, generator=g) < 0.6).to(dev)
    n = torch.randint(1, Nk + 1, (B,), generator=g)
    if B > 1:
        n[0] = 0                                   # a batch entry without a key
    return (torch.arange(Nk)[None] < n[:, None]).to(dev)


def _attend(q, k, v, dy, mask=None, causal=False, scale=None):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = attention(q, k, v, mask, causal, scale)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), dy)]


def _compare(got, want, bound):
    for n, g, w, b in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(n, g, w, b)


@pytest.mark.parametrize("dtype,B,H,Hk,Nq,Nk,d,causal,mask,spread", [
    (F16, 1, 1, 1, 1, 1, 8, False, "none", 1.0),              # one score: p = 1, no gradient for q and k
    (F16, 1, 3, 1, 2, 31, 16, False, "none", 1.0),
    (BF16, 2, 8, 8, 64, 77, 160, False, "prompt", 1.0),
    (F16, 2, 4, 2, 33, 65, 40, True, "none", 2.0),            # more keys than queries
    (BF16, 1, 6, 2, 130, 100, 64, True, "holes", 1.0),        # more queries than keys: rows without a key
    (F16, 3, 2, 2, 100, 200, 80, False, "prompt", 1.0),
    (F16, 1, 2, 1, 257, 1000, 128, False, "none", 1.0),
    (BF16, 1, 2, 2, 70, 300, 256, False, "none", 1.0),
    (F16, 1, 2, 1, 40, 90, 200, True, "holes", 1.0),
    (F16, 1, 3, 1, 5, 4000, 72, False, "holes", 1.0),         # few queries: the key axis is split
    (BF16, 1, 2, 2, 3001, 20, 48, False, "none", 1.0),        # few keys: the query axis is split
    (F16, 2, 8, 8, 1024, 1024, 40, False, "none", 1.0),
    (BF16, 1, 4, 1, 1, 777, 128, False, "prompt", 2.0),
    (BF16, 2, 12, 4, 300, 300, 64, True, "none", 2.0),
    (F16, 1, 4, 4, 1100, 1100, 56, True, "prompt", 1.0),
    (BF16, 1, 8, 8, 1024, 77, 104, False, "prompt", 1.0),
    (F16, 4, 16, 16, 70, 500, 128, False, "none", 1.0),       # whole workgroups of four waves
    (BF16, 4, 16, 16, 130, 140, 256, True, "none", 1.0),
    (F16, 4, 16, 16, 130, 140, 160, False, "holes", 1.0),
])
def test_attention_and_its_gradient(dev, dtype, B, H, Hk, Nq, Nk, d, causal, mask, spread):
    q, k, v = _heads(dev, B, H, Nq, d, 1, dtype, spread), _heads(dev, B, Hk, Nk, d, 2, dtype, spread), _heads(dev, B, Hk, Nk, d, 3, dtype)
    dy, m = _rn(dev, B, Nq, H * d, seed=4, dtype=dtype), _mask(dev, mask, B, Nk)
    got = _attend(q, k, v, dy, m, causal)
    _compare(got, *ref.attention(q, k, v, dy, m, causal))
    again = _attend(q, k, v, dy, m, causal)
    assert all(torch.equal(a, b) for a, b in zip(got, again))                 # nothing depends on the order of workgroups
    with torch.no_grad():
        assert torch.equal(attention(q, k, v, m, causal), got[0])             # the same output when nothing is kept


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_masked_places_may_hold_anything(dev, dtype, causal):
    """Infinities and NaN in masked keys and values, and in the dy of rows without a key, reach nothing; masked keys get zero gradients."""
    B, H, N, d = 3, 2, 150, 40
    q, k, v, dy = (_heads(dev, B, H, N, d, i, dtype) for i in (1, 2, 3, 4))
    m = _mask(dev, "holes", B, N)
    m[:, 64:128] = False                          # a whole tile
    m[1] = False                                  # a batch entry
    m[2, :30] = False                             # with the causal mask: rows 0 .. 29 of entry 2 see nothing
    dy = dy.transpose(1, 2).reshape(B, N, H * d).clone()
    clean = _attend(q, k, v, dy, m, causal)
    hid = ~m[:, None, :, None].expand_as(k)
    k2, v2, dy2 = k.clone(), v.clone(), dy.clone()
    k2[hid] = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min], device=dev, dtype=dtype).repeat(int(hid.sum()) // 4)
    v2[hid] = float("nan")
    dy2[1] = float("nan")
    if causal:
        dy2[2, :30] = float("inf")
    got = _attend(q, k2, v2, dy2, m, causal)
    assert all(torch.isfinite(t).all() for t in got)
    assert not got[0][1].any() and not got[1][1].any() and not got[2][hid].any() and not got[3][hid].any()
    _compare(got, *ref.attention(q, k, v, dy, m, causal))
    assert torch.equal(got[0], clean[0])


def test_attention_strides_views_and_shared_context(dev):
    """q / k / v cut out of one stacked projection, a context expanded over the batch, an odd layout that is copied, a dy that is a view."""
    B, H, N, d = 2, 4, 50, 40
    qkv = _rn(dev, B, N, 3 * H * d, seed=1)
    q, k, v = (qkv[..., i * H * d:(i + 1) * H * d].unflatten(-1, (H, d)).transpose(1, 2) for i in range(3))
    dy = _rn(dev, B, N + 3, 2 * H * d, seed=2)[:, 3:, ::2]
    _compare(_attend(q, k, v, dy), *ref.attention(q, k, v, dy))
    ctx = _rn(dev, 1, H, 33, d, seed=3)
    k2 = ctx.expand(B, H, 33, d)
    _compare(_attend(q, k2, k2, dy), *ref.attention(q, k2, k2, dy))
    leaf = ctx.clone().requires_grad_(True)                                # the gradient of a broadcast context is the sum over the batch
    (g,) = torch.autograd.grad(attention(q, leaf.expand(B, H, 33, d), k2), leaf, dy)
    want, bound = ref.attention(q, k2, k2, dy)
    ref.check("ctx", g, want[2].sum(0, keepdim=True), bound[2].sum(0, keepdim=True) + ref.half_step(F16) * want[2].abs().sum(0, keepdim=True))
    odd = _rn(dev, B, H, d, N + 1, seed=4)[..., 1:].transpose(2, 3)          # channel stride N + 1
    _compare(_attend(odd, k, v, dy, scale=0.37), *ref.attention(odd, k, v, dy, scale=0.37))


def test_attention_wanted_gradients_only(dev):
    B, H, N, d = 1, 2, 60, 64
    q, k, v, dy = (_heads(dev, B, H, N, d, i, F16) for i in (1, 2, 3, 4))
    dy = dy.transpose(1, 2).reshape(B, N, H * d)
    full = _attend(q, k, v, dy)
    for which in ((0,), (1,), (2,), (1, 2)):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate((q, k, v))]
        o = attention(*leaves)
        for i, g in zip(which, torch.autograd.grad(o, [leaves[i] for i in which], dy)):
            assert torch.equal(g, full[1 + i])


@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 2.0 ** 12])
def test_attention_fp16_gradients_keep_their_digits_at_any_loss_scale(dev, size):
    """2048 keys with nearly equal probabilities (2^-11 each) and dy scaled: ds would leave fp16's normal range without its power of two. The
    relative error (2-norm) of every gradient stays at a few half steps wherever the gradient itself is a normal number."""
    B, H, N, d = 1, 2, 2048, 64
    q, k, v, dy = (_heads(dev, B, H, N, d, i, F16) for i in (1, 2, 3, 4))
    q = q * 0.25
    v = v * 8                                     # (gradients of q and k well above 2^-24)
    dy = (dy.transpose(1, 2).reshape(B, N, H * d) * size).to(F16)
    got = _attend(q, k, v, dy)
    want, _ = ref.attention(q, k, v, dy)
    for n, g, w in list(zip(("o", "dq", "dk", "dv"), got, want)):
        big = w.abs() > 2.0 ** -13
        if big.float().mean() > 0.1:
            err = float((g.cpu().double() - w)[big].norm() / w[big].norm())
            assert err <= 3 * ref.half_step(F16), (n, err)                   # p and ds rounded once, the result once: sqrt(2) half steps at most, and the sums


def test_attention_on_another_stream_and_two_at_once(dev):
    B, H, N, d = 1, 4, 700, 40
    q, k, v, dy = (_heads(dev, B, H, N, d, i, BF16) for i in (1, 2, 3, 4))
    dy = dy.transpose(1, 2).reshape(B, N, H * d).contiguous()
    want = _attend(q, k, v, dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([_attend(q, k, v, dy) for _ in range(3)])
    torch.cuda.synchronize()
    for one in got:
        for r in one:
            assert all(torch.equal(a, b) for a, b in zip(r, want))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("how", ["one_key", "mask", "first_row"])
def test_attention_a_row_of_one_visible_key_has_no_gradient(dev, dtype, how):
    """p = 1 whatever the score: dq and dk are zeros, not what dp - delta leaves, and dv is dy's sum over the rows."""
    B, H, N, d = 2, 3, 70, 72
    Nk = 1 if how == "one_key" else 90 if how == "mask" else N
    q, dy = (_heads(dev, B, H, N, d, i, dtype, 3.0) for i in (1, 4))
    k, v = (_heads(dev, B, H, Nk, d, i, dtype, 3.0) for i in (2, 3))
    dy = dy.transpose(1, 2).reshape(B, N, H * d).contiguous()
    m = None
    if how == "mask":
        m = torch.zeros(B, Nk, dtype=torch.bool, device=dev)
        m[0, 41] = m[1, 89] = True
    o, dq, dk, dv = got = _attend(q, k, v, dy, m, how == "first_row")
    _compare(got, *ref.attention(q, k, v, dy, m, how == "first_row"))
    if how == "first_row":
        assert not dq[:, :, 0].any() and dq[:, :, 1:].any()
        return
    j = [0, 0] if how == "one_key" else [41, 89]
    assert not dq.any() and not dk.any()
    for b in range(B):
        assert torch.equal(o[b], v[b, :, j[b]].reshape(1, -1).expand(N, -1))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,Hk,Nq,Nk,causal,spread", [(1, 1, 4, 100, False, 2.0), (2, 1, 40, 333, False, 1.0), (3, 3, 60, 60, True, 1.0),
                                                      (2, 2, 700, 12, False, 0.5), (4, 4, 1010, 1010, True, 2.0)])
def test_attention_short_sums_are_as_exact_as_their_type(dev, dtype, H, Hk, Nq, Nk, causal, spread):
    """Few rows, few keys or rows that few keys carry: the error (2-norm) of each result stays within 1.25 times that of rounding the float64
    result once (dv of many rows: 1.5). Left from p and ds are their second roundings, half steps of half steps: 2^-8 of a term, against
    a cancellation of their terms of up to 2^5 at these scores, in quadrature under 1 %; the remainder of 1.25 is for o + o_lo's last bits in delta."""
    d = 64
    q, k, v, dy = (_heads(dev, 1, h, n, d, i, dtype, s) for i, (h, n, s) in enumerate([(H, Nq, spread), (Hk, Nk, spread), (Hk, Nk, 1.0), (H, Nq, 1.0)], 1))
    dy = dy.transpose(1, 2).reshape(1, Nq, H * d).contiguous()
    got, (want, _) = _attend(q, k, v, dy, None, causal), ref.attention(q, k, v, dy, None, causal)
    short = Nq * (H // Hk) <= 512 or Nk <= 128
    for n, g, w in zip(("o", "dq", "dk", "dv"), got, want):
        own = float((w.to(dtype).double() - w).norm())
        assert float((g.cpu().double() - w).norm()) <= (1.25 if short or n in ("dq", "dk") else 1.5) * own, n


def test_attention_a_cache_that_spans_more_than_32_bits(dev):
    """Tokens 2^17 elements apart (one layer of a cache that holds many): 20 000 of them span 5.2 GB. The result of the dense copy, bit for bit."""
    H, Nk, d, step = 2, 20000, 64, 2 ** 17
    q, dy = _rn(dev, 1, 2 * H, 3, d, seed=1), _rn(dev, 1, 3, 2 * H * d, seed=2)
    k, v = _heads(dev, 1, H, Nk, d, 3, F16), _heads(dev, 1, H, Nk, d, 4, F16)
    cache = torch.empty(Nk * step, dtype=F16, device=dev)
    far = [torch.as_strided(cache, (1, H, Nk, d), (Nk * step, d, step, 1), 2 * H * d * i) for i in range(2)]
    for f, t in zip(far, (k, v)):
        f.copy_(t)
    m = torch.ones(1, Nk, dtype=torch.bool, device=dev)
    m[:, 100:300] = False
    want = _attend(q, k, v, dy, m, True)
    assert all(torch.equal(a, c) for a, c in zip(_attend(q, *far, dy, m, True), want))
    _compare(want, *ref.attention(q, k, v, dy, m, True))


def test_attention_misaligned_and_odd_axes_of_one(dev):
    """Dense tensors that start between two 16-byte addresses, an axis of one with an odd stride, a dy of stride 0, a mask that is a view."""
    B, H, N, d = 1, 1, 37, 24
    flat = _rn(dev, 3 * N * d + 3, seed=1)
    q, k, v = (flat[i + 1 + i * N * d:][:N * d].view(B, H, N, d) for i in range(3))
    odd = torch.as_strided(flat, (B, H, N, d), (7, 5, d, 1), 1)
    m = _mask(dev, "holes", N, 2 * B).t()[:B]
    for a in (q, odd):
        leaf = [t.detach().requires_grad_(True) for t in (a, k, v)]
        o = attention(*leaf, m)
        got = [o.detach(), *torch.autograd.grad(o.sum(), leaf)]
        _compare(got, *ref.attention(a, k, v, torch.ones(B, N, d, dtype=F16), m))


def test_differentiated_twice_is_refused_and_saved_tensors_may_move(dev):
    """create_graph gives first gradients whose own backward raises; a graph kept gives the same gradients again; tensors that hooks took to the
    host and back (in another layout) give the same gradients; an input changed in place behind the forward is noticed."""
    C = 64
    x4 = _rn(dev, 2, C, 6, 7, seed=1).contiguous(memory_format=torch.channels_last)
    w, b, pre = (_rn(dev, *s, seed=i, dtype=t) for i, (s, t) in enumerate([((C,), F32), ((C,), F32), ((2, C), F16)], 2))
    q = _heads(dev, 2, 4, 33, 40, 5, F16)
    cases = [((x4, w, b, pre), lambda x, w, b, p: group_norm_act(x, 8, w, b, pre=p)),
             ((x4, w, b), lambda x, w, b: group_norm_act(x, 8, w, b, checkpoint="int8")),
             ((q, q * 0.5, q + 1), lambda q, k, v: attention(q, k, v)),
             ((x4.permute(0, 2, 3, 1).reshape(-1, C),), lambda x: geglu(x, "int8")), ((x4.permute(0, 2, 3, 1).reshape(-1, C),), lambda x: geglu(x, "full"))]
    for args, f in cases:
        leaves = [t.detach().requires_grad_(True) for t in args]
        y = f(*leaves)
        want = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
        again = torch.autograd.grad(y, leaves, torch.ones_like(y), create_graph=True)
        assert all(torch.equal(a, c) for a, c in zip(want, again))
        with pytest.raises(RuntimeError, match="differentiate twice"):
            sum(t.float().sum() for t in again).backward()
        with torch.autograd.graph.save_on_cpu():
            y = f(*leaves)
        assert all(torch.equal(a, c) for a, c in zip(want, torch.autograd.grad(y, leaves, torch.ones_like(y))))
    x = x4.detach().clone(memory_format=torch.channels_last)
    w.requires_grad_(True)
    y = group_norm_act(x, 8, w, b)
    x.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


# ---- group norm -----------------------------------------------------------------------------------------------------------------
def _norm(x, G, w, b, dy, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    pre = kw.pop("pre", None)
    if pre is not None:
        pre = pre.detach().requires_grad_(True)
    y = group_norm_act(leaves[0], G, leaves[1], leaves[2], pre=pre, **kw)
    names = ["dx", "dweight", "dbias"] + ([] if pre is None else ["dpre"])
    return dict(zip(names, torch.autograd.grad(y, leaves + ([] if pre is None else [pre]), dy)), y=y.detach())


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("dtype,params,N,C,H,W,G,act,pre", [
    (F16, F16, 2, 320, 16, 16, 32, True, True),
    (F16, F32, 1, 128, 64, 48, 32, True, False),
    (BF16, BF16, 2, 1280, 8, 8, 32, True, True),
    (BF16, F32, 3, 96, 37, 5, 8, False, True),
    (F32, F32, 2, 64, 19, 23, 16, True, False),
    (F32, F32, 1, 32, 1, 16, 1, False, False),
    (F16, F16, 1, 2560, 4, 4, 32, True, False),          # the widest
    (F16, F32, 5, 32, 3, 7, 32, True, True),             # one channel a group
    (BF16, F32, 1, 64, 300, 301, 32, True, True),        # many slabs, a ragged end
    (F16, F16, 1, 1024, 5, 5, 1, True, True),            # one group
])
def test_group_norm_and_its_gradient(dev, dtype, params, N, C, H, W, G, act, pre, checkpoint):
    cl = lambda t: t.contiguous(memory_format=torch.channels_last)
    shift = _rn(dev, 1, C, 1, 1, seed=9, dtype=F32)
    x = cl((_rn(dev, N, C, H, W, seed=1, dtype=F32, scale=1.5) + shift).to(dtype))
    dy = cl(_rn(dev, N, C, H, W, seed=2, dtype=dtype))
    w, b = _rn(dev, C, seed=3, dtype=params), _rn(dev, C, seed=4, dtype=params)
    e = _rn(dev, N, C, seed=5, dtype=dtype) if pre else None
    got = _norm(x, G, w, b, dy, act=act, pre=e, checkpoint=checkpoint)
    assert got["y"].is_contiguous(memory_format=torch.channels_last) and got["y"].dtype == dtype and got["dweight"].dtype == params
    for n, (want, bound) in ref.group_norm(x, G, w, b, dy, act=act, pre=e, eight=checkpoint == "int8").items():
        ref.check(n, got[n], want, bound)
    again = _norm(x, G, w, b, dy, act=act, pre=e, checkpoint=checkpoint)
    assert all(torch.equal(got[n], again[n]) for n in got)
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, G, w, b, act=act, pre=e, checkpoint=checkpoint), got["y"])


def test_group_norm_far_mean_other_layouts_and_wanted_gradients(dev):
    x = (_rn(dev, 2, 32, 20, 20, seed=1, dtype=F32) * 0.5 + 60)             # the mean is 120 deviations away
    w, b, dy = _rn(dev, 32, seed=2, dtype=F32), _rn(dev, 32, seed=3, dtype=F32), _rn(dev, 2, 32, 20, 20, seed=4, dtype=F32)
    got = _norm(x, 4, w, b, dy)                                             # x and dy NCHW: copied
    for n, (want, bound) in ref.group_norm(x, 4, w, b, dy).items():
        ref.check(n, got[n], want, bound)
    off = _rn(dev, 2, 20, 20, 33, seed=5, dtype=F16)[..., 1:].permute(0, 3, 1, 2)      # neither dense nor aligned
    h = [t.half() for t in (w, b, dy)]
    got = _norm(off, 4, *h)
    for n, (want, bound) in ref.group_norm(off, 4, *h).items():
        ref.check(n, got[n], want, bound)
    xs, ws, bs = off.detach().requires_grad_(True), h[0].detach().requires_grad_(True), h[1]
    (g,) = torch.autograd.grad(group_norm_act(xs, 4, ws.detach(), bs), xs, h[2])
    (gw,) = torch.autograd.grad(group_norm_act(off, 4, ws, bs), ws, h[2])
    assert torch.equal(g, got["dx"]) and torch.equal(gw, got["dweight"])
    odd = _rn(dev, 2, 20, 4, 4, seed=6)                                     # 20 channels: the formulas in PyTorch ops
    ww = torch.ones(20, device=dev, dtype=F16)
    r = ref.group_norm(odd, 5, ww, ww, odd)
    got = _norm(odd, 5, ww, ww, odd)
    for n in r:
        ref.check(n, got[n], *r[n])


def test_eight_bit_input_with_infinities_poisons_its_block_and_group_only(dev):
    """A block with an infinity decodes as NaN: the map's group is NaN anyway, other samples stay exact."""
    x = _rn(dev, 2, 32, 4, 4, seed=1).contiguous(memory_format=torch.channels_last)
    w, b, dy = _rn(dev, 32, seed=2), _rn(dev, 32, seed=3), _rn(dev, 2, 32, 4, 4, seed=4)
    clean = _norm(x, 1, w, b, dy, checkpoint="int8")
    bad = x.clone()
    bad[1, 3, 2, 2] = float("inf")
    got = _norm(bad, 1, w, b, dy, checkpoint="int8")
    assert got["y"][1].isnan().any() and got["dx"][1].isnan().all() and torch.equal(got["dx"][0], clean["dx"][0])


# ---- GEGLU ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("dtype,lead,n", [(F16, (2, 333), 320), (BF16, (77,), 64), (F32, (5, 3), 96), (F16, (1,), 32), (BF16, (4099,), 1280), (F32, (), 32)])
def test_geglu_and_its_gradient(dev, dtype, lead, n, checkpoint):
    x, dy = _rn(dev, *lead, 2 * n, seed=1, dtype=dtype, scale=2.0), _rn(dev, *lead, n, seed=2, dtype=dtype)
    leaf = x.detach().requires_grad_(True)
    y = geglu(leaf, checkpoint)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    r = ref.geglu(x, dy, checkpoint == "int8")
    ref.check("y", y, *r["y"])
    ref.check("dx", dx, *r["dx"])
    with torch.no_grad():
        assert torch.equal(geglu(x, checkpoint), y)


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
def test_no_rows_and_no_pixels(dev, checkpoint):
    x = torch.zeros(3, 0, 128, dtype=F16, device=dev, requires_grad=True)
    y = geglu(x, checkpoint)
    y.sum().backward()
    assert y.shape == (3, 0, 64) and x.grad.shape == x.shape
    w = torch.ones(64, device=dev, requires_grad=True)
    m = torch.zeros(2, 64, 0, 5, dtype=F16, device=dev, requires_grad=True)
    group_norm_act(m, 8, w, w, checkpoint=checkpoint).sum().backward()
    assert m.grad.shape == m.shape and not w.grad.any()


def test_geglu_far_arguments_views_and_other_widths(dev):
    x = torch.tensor([[1.0, -1.0] * 8 + [0.0, -0.0, 40.0, -40.0, 6.0, -6.0, 300.0, -300.0] * 2], device=dev, dtype=F32)
    dy = torch.ones(1, 16, device=dev)
    leaf = x.clone().requires_grad_(True)
    y = geglu(leaf, "full")
    (dx,) = torch.autograd.grad(y, leaf, dy)
    r = ref.geglu(x, dy)
    ref.check("y", y, *r["y"])
    ref.check("dx", dx, *r["dx"])
    v = _rn(dev, 9, 300, seed=1)[:, 3:259]                                  # a view, off alignment
    d = _rn(dev, 9, 256, seed=2)[:, ::2]
    leaf = v.detach().requires_grad_(True)
    y = geglu(leaf, "full")
    (dx,) = torch.autograd.grad(y, leaf, d)
    r = ref.geglu(v, d)
    ref.check("y", y, *r["y"])
    ref.check("dx", dx, *r["dx"])
    leaf = _rn(dev, 9, 20, seed=3).requires_grad_(True)                     # 10 channels: the formulas in PyTorch ops
    y = geglu(leaf, "full")
    r = ref.geglu(leaf, torch.ones(9, 10))
    ref.check("y", y, *r["y"])
    ref.check("dx", torch.autograd.grad(y, leaf, torch.ones_like(y))[0], *r["dx"])


def test_the_kernels_eight_bit_form_is_the_documented_one(dev):
    """Codes and scale bytes as the forward writes them, decoded by the documented layout, against `eight_bits`."""
    import _sdfx as S
    x = _rn(dev, 65, 64, seed=1, dtype=F32) * torch.exp(8 * _rn(dev, 65, 1, seed=2, dtype=F32))
    x[3] = 0
    x[4, :32] *= 2.0 ** -130
    x[5, 7], x[6, 40] = float("nan"), -float("inf")
    y, saved = torch.empty(65, 32, device=dev), torch.empty(65 * 64 + 65 * 2, dtype=torch.uint8, device=dev)
    S.call("sdfx_geglu_train_forward", S.ptr(x), 65, 32, 2, S.ptr(y), S.ptr(saved), S.stream())
    saved = saved.cpu()                           # (2^n by torch.pow is exact on the CPU; on the GPU it is not)
    codes, scale = saved[:65 * 64].view(torch.int8).view(65, 2, 32).double(), saved[65 * 64:].view(65, 2, 1).double()
    step = torch.where(scale == 255, torch.full_like(scale, float("inf")), torch.pow(2.0, scale - 127))
    got, want = (codes * step).view(65, 64), eight_bits(x).double().cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# ---- together -------------------------------------------------------------------------------------------------------------------
def test_captured_and_replayed(dev):
    """Forward and backward of the three in one captured graph, replayed on new inputs with eager work in between: the eager results. Two
    such graphs replayed on two streams at once share no workspace."""
    B, H, N, d, C = 1, 4, 640, 40, 160
    w, b = _rn(dev, C, seed=1, dtype=F32), _rn(dev, C, seed=2, dtype=F32)

    def step(x, dy):
        leaf, ww = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        n = group_norm_act(leaf, 32, ww, b, checkpoint="int8").permute(0, 2, 3, 1).reshape(B, N, C)
        h = n.view(B, N, H, d).transpose(1, 2)
        out = geglu(attention(h, h[:, :, :77], h[:, :, :77]) + n, "int8" if (C // 2) % 32 == 0 else "full")
        return [out.detach(), *torch.autograd.grad(out, (leaf, ww), dy)]

    make = lambda s: (_rn(dev, B, C, 20, 32, seed=s).contiguous(memory_format=torch.channels_last), _rn(dev, B, N, C // 2, seed=s + 50))
    graphs = []
    for i in range(2):
        x, dy = make(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, dy)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x, dy)
        graphs.append((g, x, dy, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in range(1, 5):
        ins = [make(10 * s + i) for i in range(2)]
        want = [step(*t) for t in ins]
        for (g, x, dy, _), (nx, ny) in zip(graphs, ins):
            x.copy_(nx)
            dy.copy_(ny)
        torch.cuda.synchronize()
        for st, (g, *_) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (_, _, _, out), r in zip(graphs, want):
            assert all(torch.equal(a, c) for a, c in zip(out, r))


@pytest.mark.parametrize("dtype,checkpoint", [(F16, "full"), (F16, "int8"), (BF16, "int8")])
def test_prior_blocks_train_on_these_operators(dev, dtype, checkpoint):
    """A ResNet block and a transformer block of the UNet with every parameter trainable, a padded prompt: outputs and all gradients
    against the same blocks in float64 on the CPU with the same checkpoints. 2-norms: about 40 half-precision roundings on the way, half a step
    rms 0.3 u each (u = 2^-11 / 2^-8), adding at random: 2 u; sums of products with cancellation a few times that. 8-bit codes follow inputs
    that differ by those roundings: a code in 50 / 6 moves by a step of 2^-7 of its block's maximum."""
    import copy
    from sdfx_nerf.sd15_arch import ResBlock, TransformerBlock, use_training_ops
    torch.manual_seed(0)
    res, tr = ResBlock(64, 160, 96), TransformerBlock(160, 48, heads=4)
    for m in (res, tr):
        use_training_ops(m, checkpoint)
    near = [copy.deepcopy(m).to(dtype) for m in (res, tr)]
    far = [copy.deepcopy(m).double() for m in near]
    near = [m.to(dev).to(memory_format=torch.channels_last) for m in near]
    x, emb, ctx, dy = (_rn("cpu", *s, seed=i, dtype=dtype) for i, s in enumerate(((2, 64, 12, 8), (2, 96), (2, 20, 48), (2, 160, 12, 8))))
    mask = torch.arange(20)[None] < torch.tensor([[20], [9]])

    def step(blocks, cast):
        a = [cast(t).detach().requires_grad_(True) for t in (x, emb, ctx)]
        y = blocks[1](blocks[0](a[0], a[1]), a[2], mask.to(a[0].device))
        ps = [p for m in blocks for p in m.parameters()]
        return [y.detach(), *torch.autograd.grad(y, a + ps, cast(dy))]
    got = step(near, lambda t: t.to(dev).contiguous(memory_format=torch.channels_last) if t.dim() == 4 else t.to(dev))
    want = step(far, lambda t: t.double())
    u = ref.half_step(dtype)
    tol = 12 * u + (2 * 2.0 ** -7 if checkpoint == "int8" else 0)
    for i, (g, w) in enumerate(zip(got, want)):
        assert g.shape == w.shape and torch.isfinite(g).all()
        err = float((g.cpu().double() - w).norm() / w.norm().clamp(min=1e-30))
        assert err <= tol, (i, err, tol)
