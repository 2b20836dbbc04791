"""GroupNorm (+ SiLU) of the frozen prior on channels-last fp16 activations: csrc/groupnorm.hip behind an `nn.GroupNorm`.

`GroupNormAct(32, C, act=True)(x)` == `F.silu(F.group_norm(x, 32, weight, bias, eps))`. On a CUDA fp16 tensor in channels-last
memory format, with frozen affine parameters, the forward and the input gradient are the two-pass NHWC kernels of
csrc/groupnorm.hip (the output stays channels-last, which is what MIOpen's NHWC convolutions take without a transpose);
everything else (CPU, float32, NCHW-contiguous inputs, trainable parameters, shapes the kernels do not take) goes through
PyTorch's own ops, so the module is a drop-in `nn.GroupNorm` (same parameters, same state_dict keys).
SDFX_GROUPNORM=0 forces the PyTorch ops everywhere (A/B switch).

For blocks that train: `group_norm_act(...)` is the same norm with every gradient (input, gamma, beta, `pre`) in fp16, bf16 and float32
(csrc/groupnorm_train.hip), `geglu(x, checkpoint=...)` GEGLU with its gradient (csrc/geglu_train.hip). `checkpoint` says how the input
is kept for the backward: "full" as it is, "int8" in 8 bits (csrc/act8.h: a shared power-of-two step per 32 channels, 33 bytes instead
of 64 in half precision). Set on a module (`GroupNormAct.checkpoint`, sd15_arch.use_training_ops) it selects these forms there."""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable
import _devswitch

_FUSED = _devswitch.get("SDFX_GROUPNORM", 1)
import _sdfx as _S

_SCRATCH = _S.StreamScratch()   # per (device, stream) float32 scratch, grown on demand (_sdfx.StreamScratch: what is kept, what is released)


def _scratch(device, nbytes):
    return _SCRATCH.get(device, nbytes)


class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pre, weight, bias, groups, eps, act):
        import _sdfx as S
        N, C, H, W = x.shape
        y = torch.empty_like(x)                                    # preserves the channels-last strides
        need_bwd = ctx.needs_input_grad[0]                         # (grad mode is off inside forward(): ask the context)
        mean_rstd = torch.empty(N, groups, 2, dtype=torch.float32, device=x.device) if need_bwd else None
        nbytes = int(S.lib().sdfx_group_norm_scratch_bytes(N, H * W, C, groups))
        S.call("sdfx_group_norm_forward", S.ptr(x), S.ptr(pre), S.ptr(weight), S.ptr(bias), N, H * W, C, groups, float(eps), int(act),
               S.ptr(y), S.ptr(mean_rstd), S.ptr(_scratch(x.device, nbytes)), S.stream())
        if need_bwd:
            ctx.save_for_backward(x, weight, bias, mean_rstd, *(() if pre is None else (pre,)))
            ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    def backward(ctx, dy):
        import _sdfx as S
        x, weight, bias, mean_rstd = ctx.saved_tensors[:4]
        pre = ctx.saved_tensors[4] if len(ctx.saved_tensors) > 4 else None
        N, C, H, W = x.shape
        dy = dy.to(torch.float16).contiguous(memory_format=torch.channels_last)
        dx = torch.empty_like(x)
        nbytes = int(S.lib().sdfx_group_norm_scratch_bytes(N, H * W, C, ctx.groups))
        S.call("sdfx_group_norm_backward", S.ptr(x), S.ptr(pre), S.ptr(dy), S.ptr(weight), S.ptr(bias), S.ptr(mean_rstd), N, H * W, C,
               ctx.groups, int(ctx.act), S.ptr(dx), S.ptr(_scratch(x.device, nbytes)), S.stream())
        return dx, None, None, None, None, None, None      # (`pre` is built from frozen parameters: no gradient)


class _AddBiasResidualFn(torch.autograd.Function):
    """a + b + bias[None, :, None, None] in one launch (channels-last fp16); the gradient passes to a and b unchanged."""

    @staticmethod
    def forward(ctx, a, b, bias):
        import _sdfx as S
        N, C, H, W = a.shape
        out = torch.empty_like(a)
        S.call("sdfx_add_bias_residual", S.ptr(a), S.ptr(b), S.ptr(bias), N, H * W, C, S.ptr(out), S.stream())
        return out

    @staticmethod
    def backward(ctx, g):
        return g, g, None


def add_bias_residual(a, b, bias):
    """`a + b + bias[None, :, None, None]` — fused when both maps are dense channels-last fp16 CUDA tensors and the bias is frozen."""
    if (_FUSED and a.is_cuda and a.dtype == torch.float16 and b.dtype == torch.float16 and a.dim() == 4 and a.shape == b.shape
            and bias is not None and bias.dtype == torch.float16 and not bias.requires_grad and a.shape[1] % 8 == 0
            and a.is_contiguous(memory_format=torch.channels_last) and b.is_contiguous(memory_format=torch.channels_last)
            and a.data_ptr() % 16 == 0 and b.data_ptr() % 16 == 0 and bias.data_ptr() % 16 == 0):
        return _AddBiasResidualFn.apply(a, b, bias)
    return a + (b if bias is None else b + bias[None, :, None, None])


# ---- training forms ---------------------------------------------------------------------------------------------------------------
_KERNEL_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_CHECKPOINTS = ("full", "int8")


def eight_bits(x):
    """What the 8-bit checkpoint form of `x` [..., C], C % 32 == 0, stands for, in x's own type (csrc/act8.h): blocks of 32 channels share
    the step 2^(floor(log2 max|x|) - 6), at least 2^-126; codes are round-half-even(x / step) in -127 .. 127; a block that holds an
    infinity or a NaN is NaN throughout."""
    w = x.double().unflatten(-1, (-1, 32))
    m = w.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(m)                                   # (its mantissa lies in [1/2, 1))
    # 2^(e - 7) from its bits: a power of two by `pow` is not exact on every device
    step = ((torch.where(torch.isfinite(m), e, 0).to(torch.int64) - 7).clamp(min=-126) + 1023 << 52).view(torch.float64)
    q = torch.round(w / step).clamp(-127, 127) * step
    return torch.where(torch.isfinite(m), q, torch.full_like(q, float("nan"))).flatten(-2).to(x.dtype)


def _check_checkpoint(checkpoint, channels, what):
    if checkpoint not in _CHECKPOINTS:
        raise ValueError(f"{what}: checkpoint must be one of {_CHECKPOINTS}, got {checkpoint!r}")
    if checkpoint == "int8" and channels % 32:
        raise ValueError(f"{what}: the 8-bit checkpoint needs a multiple of 32 channels (got {channels})")


class _GroupNormPlainFn(torch.autograd.Function):
    """The same formulas in tensor operations: CPU tensors, float64, and shapes the kernels do not take."""

    @staticmethod
    def forward(ctx, x, pre, weight, bias, groups, eps, act, eight, keep):
        wide = torch.float64 if x.dtype == torch.float64 else torch.float32
        u = x.to(wide) if pre is None else x.to(wide) + pre.to(wide)[:, :, None, None]
        r = u.reshape(x.shape[0], groups, -1)
        mean = r.mean(-1, keepdim=True)
        rstd = ((r - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
        z = ((r - mean) * rstd).view(x.shape) * weight.to(wide)[:, None, None] + bias.to(wide)[:, None, None]
        if keep:
            ctx.save_for_backward(eight_bits(x.permute(0, 2, 3, 1)).permute(0, 3, 1, 2) if eight else x, pre, weight, bias, mean, rstd)
            ctx.args = (groups, act)
        return (z * torch.sigmoid(z) if act else z).to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, pre, weight, bias, mean, rstd = ctx.saved_tensors
        groups, act = ctx.args
        wide, N = mean.dtype, x.shape[0]
        u = x.to(wide) if pre is None else x.to(wide) + pre.to(wide)[:, :, None, None]
        xr = (u.reshape(N, groups, -1) - mean) * rstd
        xh, w, dz = xr.view(x.shape), weight.to(wide)[:, None, None], dy.to(wide)
        if act:
            z = xh * w + bias.to(wide)[:, None, None]
            sg = torch.sigmoid(z)
            dz = dz * sg * (1 + z * (1 - sg))
        g = (dz * w).reshape(N, groups, -1)
        dx = (rstd * (g - g.mean(-1, keepdim=True) - xr * (g * xr).mean(-1, keepdim=True))).view(x.shape)
        return (dx.to(x.dtype), None if pre is None else dx.sum((2, 3)).to(pre.dtype), (dz * xh).sum((0, 2, 3)).to(weight.dtype),
                dz.sum((0, 2, 3)).to(bias.dtype), None, None, None, None, None)


def group_norm_act(x, groups, weight, bias, eps=1e-5, act=True, pre=None, checkpoint="full"):
    """`silu(group_norm(x + pre[:, :, None, None], groups, weight, bias, eps))` (the norm alone with `act` False) with gradients for x, `pre`,
    weight and bias. x [N, C, H, W] in fp16, bf16 or float32, channels-last (the kernels copy another layout into it and give a channels-last result);
    `pre` [N, C] (or None) in x's type; weight / bias [C] in x's type or float32. Statistics and sums are float32 or wider.

    `checkpoint`: "full" keeps x for the backward; "int8" keeps its 8-bit form (`eight_bits`; C % 32 == 0) and evaluates the
    derivative at it, with the statistics of x itself.

    C % 8 == 0, C <= 2560 and groups <= 64 run csrc/groupnorm_train.hip on CUDA tensors; everything else the same formulas in PyTorch
    ops. One derivative only (no double backward)."""
    if x.dim() != 4 or not x.is_floating_point():
        raise ValueError(f"group_norm_act: x must be a floating-point [N, C, H, W] tensor, got {x.dtype} {tuple(x.shape)}")
    N, C, H, W = x.shape
    if groups < 1 or C % groups:
        raise ValueError(f"group_norm_act: {C} channels do not divide into {groups} groups")
    if weight is None or bias is None or weight.shape != (C,) or bias.shape != (C,) or weight.dtype != bias.dtype:
        raise ValueError(f"group_norm_act: weight and bias must be [{C}] tensors of one type")
    if weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"group_norm_act: weight / bias must be {x.dtype} or float32, got {weight.dtype}")
    if pre is not None and (pre.shape != (N, C) or pre.dtype != x.dtype):
        raise ValueError(f"group_norm_act: pre must be a [{N}, {C}] tensor of type {x.dtype}, got {pre.dtype} {tuple(pre.shape)}")
    if any(t is not None and t.device != x.device for t in (pre, weight, bias)):
        raise ValueError("group_norm_act: x, pre, weight and bias must be on one device")
    if not eps >= 0:
        raise ValueError(f"group_norm_act: eps must not be negative, got {eps}")
    _check_checkpoint(checkpoint, C, "group_norm_act")
    if x.numel() == 0:
        return x + (weight.sum() + bias.sum()).to(x.dtype) * 0 + (0 if pre is None else pre[:, :, None, None] * 0)
    if x.is_cuda and x.dtype in _KERNEL_TYPES and C % 8 == 0 and C <= 2560 and groups <= 64 and H * W < 2 ** 31 and N < 2 ** 23:
        return _S.native().group_norm(x, pre, weight, bias, groups, eps, act, checkpoint == "int8")
    keep = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias.requires_grad or (pre is not None and pre.requires_grad))
    return _GroupNormPlainFn.apply(x, pre, weight, bias, groups, eps, act, checkpoint == "int8", keep)


class _GegluPlainFn(torch.autograd.Function):
    """The same formulas in tensor operations (see _GroupNormPlainFn)."""

    @staticmethod
    def forward(ctx, x, eight, keep):
        if keep:
            ctx.save_for_backward(eight_bits(x) if eight else x)
        a, g = (x if x.dtype == torch.float64 else x.float()).chunk(2, dim=-1)
        return (a * F.gelu(g)).to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        w = x if x.dtype == torch.float64 else x.float()
        a, g = w.chunk(2, dim=-1)
        cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        pdf = torch.exp(-0.5 * g * g) * 0.3989422804014327
        d = dy.to(w.dtype)
        return torch.cat([d * g * cdf, d * a * (cdf + g * pdf)], dim=-1).to(x.dtype), None, None


def geglu(x, checkpoint=None):
    """GEGLU of a feed-forward block: `a * gelu(gate)` for `a, gate = x.chunk(2, dim=-1)` (exact erf GELU).

    `checkpoint` None (the frozen UNet): one launch on a dense fp16 CUDA tensor that needs no gradient, PyTorch's two ops otherwise.
    "full" / "int8" (a block that trains): fp16, bf16 or float32 with its gradient, x kept for the backward as it is or in 8 bits
    (`eight_bits`: the last dimension a multiple of 64), at which the derivative is then evaluated. The last dimension a multiple of 16
    runs csrc/geglu_train.hip on CUDA tensors, everything else the same formulas in PyTorch ops. One derivative only."""
    n = x.shape[-1] // 2
    if checkpoint is not None:
        if x.dim() == 0 or x.shape[-1] % 2 or x.shape[-1] == 0 or not x.is_floating_point():
            raise ValueError(f"geglu: x must be a floating-point tensor with an even last dimension, got {x.dtype} {tuple(x.shape)}")
        _check_checkpoint(checkpoint, n, "geglu")
        if x.is_cuda and x.dtype in _KERNEL_TYPES and n % 8 == 0:
            return _S.native().geglu(x, checkpoint == "int8")
        return _GegluPlainFn.apply(x, checkpoint == "int8", torch.is_grad_enabled() and x.requires_grad)
    if (_FUSED and x.is_cuda and x.dtype == torch.float16 and not (x.requires_grad and torch.is_grad_enabled()) and x.is_contiguous()
            and x.shape[-1] % 16 == 0 and x.data_ptr() % 16 == 0):
        import _sdfx as S
        out = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
        S.call("sdfx_geglu", S.ptr(x), x.numel() // x.shape[-1], n, S.ptr(out), S.stream())
        return out
    a, gate = x.chunk(2, dim=-1)
    return a * F.gelu(gate)


def fused_ok(x, weight, bias, groups) -> bool:
    """The conditions under which csrc/groupnorm.hip takes the call (see the module docstring)."""
    if not (_FUSED and x.is_cuda and x.dtype == torch.float16 and x.dim() == 4 and weight is not None and bias is not None):
        return False
    if weight.requires_grad or bias.requires_grad or weight.dtype != torch.float16 or bias.dtype != torch.float16:
        return False
    N, C, H, W = x.shape
    if N == 0 or H * W == 0 or C % 8 or C % groups or C > 2560 or groups > 64:
        return False
    # dense NHWC memory (a [N, C, 1, 1] tensor is both contiguous and channels-last: either way its memory is [N, HW, C])
    return x.is_contiguous(memory_format=torch.channels_last)


class GroupNormAct(nn.GroupNorm):
    """`nn.GroupNorm` followed by SiLU when `act` (the pair the ResNet blocks of the SD-1.5 UNet / VAE apply), fused on the
    channels-last fp16 path."""

    def __init__(self, num_groups, num_channels, eps=1e-5, act=False):
        super().__init__(num_groups, num_channels, eps=eps, affine=True)
        self.act = bool(act)
        self.checkpoint = None      # "full" / "int8": the training form (`group_norm_act`), see sd15_arch.use_training_ops

    def forward(self, x, pre=None):
        """`pre` [N, C] (optional; no gradient unless `checkpoint` is set): the norm is taken of `x + pre[:, :, None, None]`."""
        if self.checkpoint is not None:
            w, b = (t if t.dtype == x.dtype else t.float() for t in (self.weight, self.bias))
            return group_norm_act(x, self.num_groups, w, b, self.eps, self.act, pre,
                                  self.checkpoint if x.shape[1] % 32 == 0 else "full")
        if fused_ok(x, self.weight, self.bias, self.num_groups) and (pre is None or (
                pre.dtype == torch.float16 and pre.shape == (x.shape[0], x.shape[1]) and pre.is_contiguous() and pre.data_ptr() % 16 == 0)):
            return _GroupNormActFn.apply(x, None if pre is None else pre.detach(), self.weight, self.bias, self.num_groups, self.eps, self.act)
        if pre is not None:
            x = x + pre[:, :, None, None].to(x.dtype)
        y = F.group_norm(x, self.num_groups, self.weight, self.bias, self.eps)
        return F.silu(y) if self.act else y
