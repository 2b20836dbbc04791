"""CPU: calls of the training operators that lie at the edge of what their documentation allows."""
import pytest
import torch

import train_ops_ref as ref
from sdfx_nerf.attention import attention


def _rn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


@pytest.mark.parametrize("training", [None, "full"])
@pytest.mark.parametrize("dim,heads", [(320, 1), (640, 2), (320, 2)])
def test_a_context_mask_hides_tokens_from_heads_of_any_width(dim, heads, training):
    """Masked tokens are as good as absent, whatever they hold; float64, so that only the order of sums differs."""
    from sdfx_nerf.sd15_arch import TransformerBlock, use_training_ops
    torch.manual_seed(0)
    block = use_training_ops(TransformerBlock(dim, 24, heads=heads).double(), training)
    x, ctx = _rn(2, dim, 3, 2, seed=1, dtype=torch.float64), _rn(2, 7, 24, seed=2, dtype=torch.float64)
    mask = torch.arange(7)[None].expand(2, 7) < 5
    far = ctx.clone()
    far[:, 5:] = 1e3
    want = block(x, ctx[:, :5])
    for c in (ctx, far):
        assert torch.allclose(block(x, c, mask), want, rtol=1e-10, atol=1e-12)
    assert not torch.allclose(block(x, ctx), want, rtol=1e-3)


@pytest.mark.parametrize("scale,taken", [(1e-30, True), (9e-31, False), (1e30, True), (1.1e30, False)])
def test_the_c_entries_refuse_scales_they_cannot_carry(scale, taken):
    """A call that is refused for its scale says so; one whose scale is taken is refused for what is checked next (misaligned rows). No launch."""
    import ctypes
    import _sdfx as S
    lib, P, odd, st = S.lib(), ctypes.c_void_p(4096), ctypes.c_void_p(4100), (ctypes.c_uint64 * 3)(8, 8, 8)
    assert lib.sdfx_attention_train_forward(odd, P, P, None, 1, 1, 1, 3, 5, 16, st, st, st, scale, 0, 0, P, None, None, P, None) == -1
    assert (b"scale" in lib.sdfx_last_error()) != taken
    assert lib.sdfx_attention_train_backward(odd, P, P, None, P, P, P, P, 1, 1, 1, 3, 5, 16, st, st, st, scale, 0, 0, P, P, P, P, None) == -1
    assert (b"scale" in lib.sdfx_last_error()) != taken


def test_a_row_that_sees_no_key_may_hold_anything():
    """NaN and infinities in the queries and dy of rows that see nothing reach no gradient; nor do those of masked keys (in tensor operations)."""
    q, k, v, dy = _rn(2, 2, 6, 8, seed=1), _rn(2, 2, 4, 8, seed=2), _rn(2, 2, 4, 8, seed=3), _rn(2, 6, 16, seed=4)
    m = torch.tensor([[True] * 4, [False] * 4])
    want = None
    for bad in (0.0, float("nan"), float("inf")):
        qb, dyb = q.clone(), dy.clone()
        qb[0, :, :2] = qb[1] = bad                                    # (six queries on four keys: the first two see none)
        dyb[0, :2] = dyb[1] = bad
        leaves = [t.clone().requires_grad_(True) for t in (qb, k, v)]
        o = attention(*leaves, m, True)
        got = [o.detach(), *torch.autograd.grad(o, leaves, dyb)]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not got[0][0, :2].any() and got[0][0, 2:].all() and got[2][0].any()


def test_training_ops_keep_inputs_whole_unless_8_bits_are_asked_for():
    from sdfx_nerf.sd15_arch import ResBlock, TransformerBlock, use_training_ops
    for block, x, more in ((ResBlock(32, 64, 16), _rn(2, 32, 4, 4, seed=1), (_rn(2, 16, seed=2),)),
                           (TransformerBlock(32, 24, heads=2), _rn(2, 32, 4, 4, seed=1), (_rn(2, 5, 24, seed=2),))):
        grads = {}
        for how in ((), ("full",), ("int8",)):
            y = use_training_ops(block, *how)(x, *more)
            grads[how] = torch.cat([g.flatten() for g in torch.autograd.grad(y, list(block.parameters()), torch.ones_like(y))])
        assert torch.equal(grads[()], grads[("full",)]) and not torch.equal(grads[()], grads[("int8",)])


def test_blocks_that_take_no_mask_still_stand_in():
    """A module put in the place of a cross-attention or of a transformer block with their older arguments is called with those."""
    from sdfx_nerf.sd15_arch import TransformerBlock, UNetSD15

    class Cross(torch.nn.Module):
        def forward(self, x, ctx, residual):
            return residual + ctx.mean()

    class Block(torch.nn.Module):
        def forward(self, x, ctx):
            return x + ctx.mean()
    torch.manual_seed(0)
    net = UNetSD15(in_ch=4, out_ch=4, base=32, mult=(1, 2), ctx_dim=24, heads=4, res_per_level=1)
    x, t, ctx = _rn(2, 4, 8, 8, seed=1), torch.tensor([3, 500]), _rn(2, 7, 24, seed=2)
    net.mid[1] = Block()
    for m in net.modules():
        if isinstance(m, TransformerBlock):
            m.attn2 = Cross()
    assert net(x, t, ctx).shape == x.shape
