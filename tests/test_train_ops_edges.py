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
