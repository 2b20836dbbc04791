"""Calls of the training operators (csrc/attention_train*.hip, groupnorm_train.hip, geglu_train.hip) at the edge of what their documentation
allows, against float64."""
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
