"""CPU: the training operators' tensor-operation forms against float64 and finite differences, the 8-bit form, refusals in Python and at the C ABI."""
import ctypes

import pytest
import torch

import train_ops_ref as ref
from sdfx_nerf.attention import attention
from sdfx_nerf.groupnorm import GroupNormAct, eight_bits, geglu, group_norm_act


def _rn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


@pytest.mark.parametrize("H,Hk,Nq,Nk,causal,masked", [(4, 4, 5, 7, False, False), (4, 2, 6, 6, True, False), (6, 2, 5, 3, True, True), (2, 1, 1, 9, False, True)])
def test_attention_gradient_against_differences(H, Hk, Nq, Nk, causal, masked):
    q, k, v = (_rn(2, h, n, 8, seed=i, dtype=torch.float64).requires_grad_(True) for i, (h, n) in enumerate(((H, Nq), (Hk, Nk), (Hk, Nk))))
    m = None
    if masked:
        m = torch.rand(2, Nk, generator=torch.Generator().manual_seed(5)) < 0.6
        m[1] = False
    assert torch.autograd.gradcheck(lambda a, b, c: attention(a, b, c, m, causal, 0.3), (q, k, v))


def test_attention_float32_matches_the_reference_and_empty_rows_are_zero():
    q, k, v, dy = _rn(2, 4, 9, 16, seed=1), _rn(2, 2, 6, 16, seed=2), _rn(2, 2, 6, 16, seed=3), _rn(2, 9, 64, seed=4)
    m = torch.ones(2, 6, dtype=torch.bool)
    m[0, :2] = False
    m[1] = False
    k[~m[:, None, :, None].expand_as(k)] = float("nan")
    v[~m[:, None, :, None].expand_as(v)] = float("inf")
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    o = attention(q, k, v, m, True)
    got = [o, *torch.autograd.grad(o, (q, k, v), dy)]
    want, bound = ref.attention(q, k, v, dy, m, True)
    for n, g, w, b in zip(("o", "dq", "dk", "dv"), got, want, bound):
        ref.check(n, g, w, b)
    assert not o[1].any() and not got[2][1].any()           # a batch entry without a key; rows 0 .. 4 of the other see none either
    assert not o[0, :5].any()


@pytest.mark.parametrize("shapes", [((2, 4, 0, 8), (2, 4, 5, 8)), ((2, 4, 3, 8), (2, 4, 0, 8)), ((0, 4, 3, 8), (0, 4, 5, 8))])
def test_attention_lengths_of_zero(shapes):
    q, k = torch.randn(shapes[0], requires_grad=True), torch.randn(shapes[1], requires_grad=True)
    o = attention(q, k, k * 1.0)
    assert o.shape == (shapes[0][0], shapes[0][2], 32) and not o.any()
    o.sum().backward()
    assert q.grad.shape == q.shape and not q.grad.any() and not k.grad.any()
    with torch.no_grad():                         # nor does any value reach the zeros
        q.fill_(float("inf"))
        k.fill_(float("nan"))
        assert not attention(q, k, k).any()


def test_attention_refuses():
    q, k = torch.randn(2, 4, 3, 8), torch.randn(2, 4, 5, 8)
    m = torch.ones(2, 5, dtype=torch.bool)
    for bad in (lambda: attention(q[0], k, k), lambda: attention(q, k, k[:, :, :4]), lambda: attention(q, k[:, :3], k[:, :3]),
                lambda: attention(q, k.half(), k.half()), lambda: attention(q, k[..., :4], k[..., :4]), lambda: attention(q, k[:1], k[:1]),
                lambda: attention(q, k, k, m.float()), lambda: attention(q, k, k, m[:, :4]), lambda: attention(q, k, k, scale=0.0),
                lambda: attention(q, k, k, scale=-1.0), lambda: attention(q, k, k, scale=float("inf")), lambda: attention(q, k, k, scale=float("nan")),
                lambda: attention(q.long(), k.long(), k.long())):
        with pytest.raises(ValueError):
            bad()


def test_eight_bits_is_the_definition():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(200, 96, generator=g) * torch.exp(6 * torch.randn(200, 1, generator=g))
    x[3] = 0
    x[4, :32] = torch.tensor([1.0] + [2.0 ** -8] * 31)        # below half a step
    x[5, 0], x[6, 40] = float("inf"), float("nan")
    x[7, :32] = torch.linspace(-1.9999, 1.9999, 32)           # the largest clamp at 127 steps
    x[8] *= 2.0 ** -120
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        xt = x.to(dt)
        got, want = eight_bits(xt).double(), ref.eight_bits(xt).to(dt).double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        ok = torch.isfinite(xt.float().unflatten(-1, (-1, 32))).all(-1, keepdim=True)
        m = xt.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
        err = (got - xt.double()).unflatten(-1, (-1, 32)).abs()
        assert bool((torch.where(ok, err, torch.zeros(())) <= torch.where(ok, m * 2.0 ** -6, torch.zeros(())) + 2.0 ** -126).all())
    assert eight_bits(x)[5, :32].isnan().all() and eight_bits(x)[5, 32:].isfinite().all()


@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("with_pre", [True, False])
def test_group_norm_gradient_against_differences(act, with_pre):
    x, w, b = _rn(2, 8, 3, 2, seed=1, dtype=torch.float64), _rn(8, seed=2, dtype=torch.float64), _rn(8, seed=3, dtype=torch.float64)
    args = [t.requires_grad_(True) for t in ((x, w, b) + ((_rn(2, 8, seed=4, dtype=torch.float64),) if with_pre else ()))]
    assert torch.autograd.gradcheck(lambda *a: group_norm_act(a[0], 2, a[1], a[2], act=act, pre=a[3] if with_pre else None), args)


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("dtype,params", [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)])
def test_group_norm_matches_the_reference(dtype, params, checkpoint):
    x, pre, dy = _rn(2, 64, 5, 3, seed=1, dtype=dtype, scale=2.0), _rn(2, 64, seed=2, dtype=dtype), _rn(2, 64, 5, 3, seed=3, dtype=dtype)
    w, b = _rn(64, seed=4, dtype=params), _rn(64, seed=5, dtype=params)
    leaves = [t.requires_grad_(True) for t in (x, w, b, pre)]
    y = group_norm_act(x, 8, w, b, pre=pre, checkpoint=checkpoint)
    got = dict(zip(("dx", "dweight", "dbias", "dpre"), torch.autograd.grad(y, leaves, dy)), y=y)
    for n, (want, bound) in ref.group_norm(x, 8, w, b, dy, pre=pre, eight=checkpoint == "int8").items():
        ref.check(n, got[n], want, bound)


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
def test_geglu_matches_the_reference_and_differences(checkpoint):
    x, dy = _rn(3, 5, 128, seed=1, scale=2.0).requires_grad_(True), _rn(3, 5, 64, seed=2)
    y = geglu(x, checkpoint)
    (dx,) = torch.autograd.grad(y, x, dy)
    r = ref.geglu(x, dy, checkpoint == "int8")
    ref.check("y", y, *r["y"])
    ref.check("dx", dx, *r["dx"])
    assert torch.autograd.gradcheck(lambda t: geglu(t, "full"), (_rn(3, 6, seed=3, dtype=torch.float64).requires_grad_(True),))


def test_norm_and_geglu_refuse():
    x, w = torch.randn(2, 16, 3, 3), torch.ones(16)
    for bad in (lambda: group_norm_act(x[0], 4, w, w), lambda: group_norm_act(x, 3, w, w), lambda: group_norm_act(x, 0, w, w),
                lambda: group_norm_act(x, 4, w[:8], w), lambda: group_norm_act(x, 4, None, w), lambda: group_norm_act(x, 4, w.double(), w.double()),
                lambda: group_norm_act(x, 4, w.half(), w), lambda: group_norm_act(x, 4, w, w, pre=torch.zeros(2, 8)),
                lambda: group_norm_act(x, 4, w, w, pre=torch.zeros(2, 16).half()), lambda: group_norm_act(x, 4, w, w, checkpoint="int4"),
                lambda: group_norm_act(x, 4, w, w, checkpoint="int8"), lambda: group_norm_act(x, 4, w, w, eps=-1.0),
                lambda: group_norm_act(x, 4, w, w, eps=float("nan")), lambda: group_norm_act(x.long(), 4, w, w),
                lambda: geglu(x[0, 0], "int4"), lambda: geglu(torch.randn(3, 7), "full"), lambda: geglu(torch.randn(3, 32), "int8"),
                lambda: geglu(torch.randn(3, 0), "full")):
        with pytest.raises(ValueError):
            bad()


def test_empty_maps_and_rows():
    x, w, b = torch.randn(0, 16, 3, 3, requires_grad=True), torch.ones(16, requires_grad=True), torch.zeros(16, requires_grad=True)
    y = group_norm_act(x, 4, w, b)
    assert y.shape == x.shape
    y.sum().backward()
    assert not w.grad.any() and x.grad.shape == x.shape
    e = torch.randn(0, 16, requires_grad=True)
    geglu(e, "full").sum().backward()
    assert e.grad.shape == e.shape


def test_frozen_forms_are_unchanged_by_default():
    m = GroupNormAct(4, 16, act=True)
    x = torch.randn(2, 16, 3, 3)
    assert torch.equal(m(x), torch.nn.functional.silu(torch.nn.functional.group_norm(x, 4, m.weight, m.bias, m.eps)))
    a, g = x.chunk(2, dim=-1) if False else torch.randn(2, 8).chunk(2, dim=-1)
    assert torch.equal(geglu(torch.cat([a, g], -1)), a * torch.nn.functional.gelu(g))


def test_c_abi_refuses_before_any_launch():
    """Null pointers, misaligned pointers and shapes the kernels do not take are errors on the host; no GPU here."""
    import _sdfx as S
    lib = S.lib()
    P, odd, st = ctypes.c_void_p(4096), ctypes.c_void_p(4100), (ctypes.c_uint64 * 3)(8, 8, 8)

    def fwd(q=P, o=P, B=1, H=2, Hk=1, Nq=3, Nk=5, D=16, strides=st, scale=1.0, scratch=P):
        return lib.sdfx_attention_train_forward(q, P, P, None, B, H, Hk, Nq, Nk, D, strides, st, st, scale, 0, 0, o, None, None, scratch, None)
    bad = [dict(q=None), dict(o=None), dict(q=odd), dict(B=0), dict(Nq=0), dict(Nk=0), dict(H=3, Hk=2), dict(D=12), dict(D=264), dict(D=0), dict(scale=0.0),
           dict(scale=-1.0), dict(scale=float("nan")), dict(strides=(ctypes.c_uint64 * 3)(8, 4, 8)), dict(Nq=1 << 30), dict(B=1 << 20, Nk=1 << 12),
           dict(Nk=1 << 15, Nq=1, scratch=None)]
    for kw in bad:
        assert fwd(**kw) == -1, kw
        assert b"attention_train_forward" in lib.sdfx_last_error()
    assert lib.sdfx_attention_train_backward(P, P, P, None, P, P, P, P, 1, 1, 1, 3, 5, 16, st, st, st, 1.0, 0, 0, P, P, None, P, None) == -1
    assert lib.sdfx_attention_train_backward(P, P, P, None, P, None, P, P, 1, 1, 1, 3, 5, 16, st, st, st, 1.0, 0, 0, P, P, P, P, None) == -1
    assert lib.sdfx_attention_train_scratch_bytes(1, 2, 1, 3, 5, 12, 1) == 0

    def gn(x=P, y=P, N=1, HW=4, C=32, G=4, dtype=0, saved=None, eps=1e-5):
        return lib.sdfx_group_norm_train_forward(x, None, P, P, N, HW, C, G, eps, 1, dtype, 0, y, saved, P, P, None)
    for kw in (dict(x=None), dict(y=odd), dict(C=20, G=4), dict(C=32, G=5), dict(C=2568, G=8), dict(C=128, G=128), dict(N=0), dict(HW=0), dict(dtype=3),
               dict(C=40, saved=P), dict(eps=-1.0)):
        assert gn(**kw) == -1, kw
    assert lib.sdfx_group_norm_train_backward(P, 0, None, P, P, P, P, 1, 4, 32, 4, 1, 0, 0, P, P, None, None, P, None) == -1     # dpre without pre
    assert lib.sdfx_group_norm_train_backward(P, 1, None, P, P, P, P, 1, 4, 40, 4, 1, 0, 0, P, None, None, None, P, None) == -1
    assert lib.sdfx_geglu_train_forward(P, 4, 12, 0, P, None, None) == -1 and lib.sdfx_geglu_train_forward(P, 4, 40, 0, P, P, None) == -1
    assert lib.sdfx_geglu_train_forward(None, 4, 16, 0, P, None, None) == -1 and lib.sdfx_geglu_train_backward(P, 0, P, 4, 16, 5, P, None) == -1
    assert lib.sdfx_geglu_train_forward(P, 0, 16, 0, P, None, None) == 0          # no rows: nothing to do


# ---- the prior's blocks on these operators ------------------------------------------------------------------------------------------
def _small_unet(dtype):
    from sdfx_nerf.sd15_arch import UNetSD15
    torch.manual_seed(0)
    return UNetSD15(in_ch=4, out_ch=4, base=32, mult=(1, 2), ctx_dim=24, heads=4, res_per_level=1).to(dtype)


def test_a_unet_on_the_training_ops_has_the_gradients_of_the_plain_one():
    """float64, checkpoint "full": the same outputs and parameter gradients to rounding; the switch goes back; a context mask equals a
    shorter context."""
    from sdfx_nerf.sd15_arch import use_training_ops
    net = _small_unet(torch.float64)
    x, t, ctx = _rn(2, 4, 8, 8, seed=1, dtype=torch.float64), torch.tensor([3, 500]), _rn(2, 7, 24, seed=2, dtype=torch.float64)
    dy = _rn(2, 4, 8, 8, seed=3, dtype=torch.float64)
    ps = list(net.parameters())
    y0 = net(x, t, ctx)
    g0 = torch.autograd.grad(y0, ps, dy)
    y1 = use_training_ops(net, "full")(x, t, ctx)
    g1 = torch.autograd.grad(y1, ps, dy)
    assert torch.allclose(y0, y1, rtol=1e-10, atol=1e-12)
    for a, b in zip(g0, g1):
        assert float((a - b).norm()) <= 1e-9 * float(a.norm()) + 1e-12
    mask = torch.arange(7)[None].expand(2, 7) < 5
    assert torch.allclose(net(x, t, ctx, context_mask=mask), net(x, t, ctx[:, :5]), rtol=1e-10, atol=1e-12)
    assert torch.equal(use_training_ops(net, None)(x, t, ctx), y0)
    assert torch.allclose(net(x, t, ctx, context_mask=mask), net(x, t, ctx[:, :5]), rtol=1e-10, atol=1e-12)
    with pytest.raises(ValueError):
        use_training_ops(net, "int4")


def test_a_unet_with_8_bit_checkpoints_keeps_its_outputs_and_nearly_its_gradients():
    """The forward does not see the checkpoint. A gradient through one norm is off by the 8-bit input's error (rms of a step over a normal
    block's deviation below 1 %) times a factor of order one; the errors of the dozen norms and GEGLUs add up at random."""
    from sdfx_nerf.sd15_arch import use_training_ops
    net = _small_unet(torch.float32)
    x, t, ctx, dy = _rn(2, 4, 8, 8, seed=1), torch.tensor([3, 500]), _rn(2, 7, 24, seed=2), _rn(2, 4, 8, 8, seed=3)
    ps = list(net.parameters())
    y0 = use_training_ops(net, "full")(x, t, ctx)
    g0 = torch.cat([g.flatten() for g in torch.autograd.grad(y0, ps, dy)])
    y1 = use_training_ops(net, "int8")(x, t, ctx)
    g1 = torch.cat([g.flatten() for g in torch.autograd.grad(y1, ps, dy)])
    assert torch.equal(y0, y1)
    assert not torch.equal(g0, g1) and float((g0 - g1).norm()) <= 0.1 * float(g0.norm())
