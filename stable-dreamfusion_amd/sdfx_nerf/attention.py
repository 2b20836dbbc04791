"""Attention of the frozen prior's transformer blocks: csrc/attention.hip behind `attention_bnc(q, k, v)`.

`attention_bnc(q, k, v)` == `F.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, Nq, H * d)` for fp16 CUDA tensors
q [B, H, Nq, d], k / v [B, H, Nk, d] (any batch / head / token strides, unit channel stride — the `.view(B, N, H, d).transpose(1, 2)`
views of a projection's output are taken as they are) with d in (40, 80, 160) when no gradient is wanted (the UNet of the SDS
step runs under `no_grad`); every other call goes through PyTorch's op. SDFX_ATTENTION=0 forces PyTorch's op (A/B switch).

`attention(q, k, v, ...)` is attention for blocks that train (csrc/attention_train.hip): fp16 and bf16, any head width that is a multiple
of 8 up to 256, query heads that share key heads, key and causal masks, and a backward pass that recomputes the probabilities."""
from __future__ import annotations

import ctypes as C

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable
import _devswitch

_FUSED = _devswitch.get("SDFX_ATTENTION", 1)
_U3 = C.c_uint32 * 3


def attention_ok(q, k, v) -> bool:
    """The conditions under which csrc/attention.hip takes the call (see the module docstring)."""
    if not (_FUSED and q.is_cuda and q.dim() == 4 and k.dim() == 4 and v.dim() == 4):
        return False
    if not (q.dtype == k.dtype == v.dtype == torch.float16) or k.shape != v.shape:
        return False
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return False
    B, H, Nq, d = q.shape
    if k.shape[0] != B or k.shape[1] != H or k.shape[3] != d or d not in (40, 80, 160) or 0 in (B, H, Nq, k.shape[2]):
        return False
    for t in (q, k, v):
        sb, sh, sn, sd = t.stride()
        if sd != 1 or sb % 8 or sh % 8 or sn % 8 or t.data_ptr() % 16 or max(sb, sh, sn) >= 2 ** 32:
            return False
    return True


_AUTO_MAX_D = _devswitch.get("SDFX_ATTENTION_MAX_D", 80)   # wider heads: only when asked for (see attention_bnc)


def attention_bnc(q, k, v, waves=0, force=False):
    """See the module docstring. `waves`: 0 = chosen by shape; 1 / 2 / 4 waves per workgroup are for measurements. The 160-wide heads
    (256 and 64 tokens: 0.7 GFLOP, 32 workgroups) are left to PyTorch's op unless `force`: in the replayed UNet the kernel took 26 us
    per call there against ~12 us (profiles/r04_unet_kernel_stats_own_conv_attention.csv)."""
    B, H, Nq, d = q.shape
    if (force or waves or d <= _AUTO_MAX_D) and attention_ok(q, k, v):
        import _sdfx as S
        out = torch.empty(B, Nq, H * d, dtype=q.dtype, device=q.device)
        st = lambda t: _U3(t.stride(0), t.stride(2), t.stride(1))           # batch, token, head (elements)
        S.call("sdfx_attention_forward", S.ptr(q), S.ptr(k), S.ptr(v), B, H, Nq, k.shape[2], d, st(q), st(k), st(v), float(d) ** -0.5,
               int(waves), S.ptr(out), S.stream())
        return out
    return F.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, Nq, H * d)


_U64x3 = C.c_uint64 * 3


def _taken(t):
    """`t` [B, H, n, d] as the kernels read it (unit channel stride, 16-byte rows): itself, or a copy."""
    sb, sh, sn, sd = t.stride()
    return t if sd == 1 and not (sb % 8 or sh % 8 or sn % 8 or t.data_ptr() % 16) else t.contiguous()


def _strides(t):
    sb, sh, sn, _ = t.stride()
    return _U64x3(sb, sn, sh)


class _AttentionFn(torch.autograd.Function):
    """csrc/attention_train.hip. The scratch is allocated per call: calls on several streams, or graphs replayed at once, share none."""

    @staticmethod
    def forward(ctx, q, k, v, key_mask, causal, scale, keep):
        import _sdfx as S
        (B, H, Nq, d), (_, Hk, Nk, _) = q.shape, k.shape
        with S.on_device(q):
            o = torch.empty(B, Nq, H * d, dtype=q.dtype, device=q.device)
            o_lo = torch.empty_like(o) if keep else None
            lse = torch.empty(B, H, Nq, dtype=torch.float32, device=q.device) if keep else None
            nbytes = int(S.lib().sdfx_attention_train_scratch_bytes(B, H, Hk, Nq, Nk, d, 0))
            scratch = torch.empty(nbytes // 4, dtype=torch.float32, device=q.device) if nbytes else None
            S.call("sdfx_attention_train_forward", S.ptr(q), S.ptr(k), S.ptr(v), S.ptr(key_mask), B, H, Hk, Nq, Nk, d, _strides(q), _strides(k),
                   _strides(v), scale, causal, int(q.dtype == torch.bfloat16), S.ptr(o), S.ptr(o_lo), S.ptr(lse), S.ptr(scratch), S.stream())
        if keep:
            ctx.save_for_backward(q, k, v, key_mask, o, o_lo, lse)
            ctx.args = (causal, scale)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        import _sdfx as S
        q, k, v, key_mask, o, o_lo, lse = ctx.saved_tensors
        causal, scale = ctx.args
        (B, H, Nq, d), (_, Hk, Nk, _) = q.shape, k.shape
        with S.on_device(q):
            dy = dy.contiguous()
            dy = dy if dy.data_ptr() % 16 == 0 else dy.clone()
            new = lambda n, h: torch.empty(B, n, h, d, dtype=q.dtype, device=q.device)
            dq = new(Nq, H) if ctx.needs_input_grad[0] else None
            dk, dv = (new(Nk, Hk), new(Nk, Hk)) if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else (None, None)
            nbytes = int(S.lib().sdfx_attention_train_scratch_bytes(B, H, Hk, Nq, Nk, d, 1))
            scratch = torch.empty(nbytes // 4, dtype=torch.float32, device=q.device)
            S.call("sdfx_attention_train_backward", S.ptr(q), S.ptr(k), S.ptr(v), S.ptr(key_mask), S.ptr(o), S.ptr(o_lo), S.ptr(lse), S.ptr(dy), B, H,
                   Hk, Nq, Nk, d, _strides(q), _strides(k), _strides(v), scale, causal, int(q.dtype == torch.bfloat16), S.ptr(dq), S.ptr(dk),
                   S.ptr(dv), S.ptr(scratch), S.stream())
        view = lambda t: None if t is None else t.transpose(1, 2)
        return view(dq), view(dk), view(dv), None, None, None, None


def _attention_plain(q, k, v, key_mask, causal, scale):
    """The same function in PyTorch ops (differentiable): CPU tensors, float32 / float64, head widths the kernels do not take."""
    (B, H, Nq, d), (_, Hk, Nk, _) = q.shape, k.shape
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    qf, kf, vf = q.to(wide), k.to(wide), v.to(wide)
    see = torch.ones(1, 1, Nq, Nk, dtype=torch.bool, device=q.device)
    if key_mask is not None:
        see = see & key_mask[:, None, None, :]
        kf, vf = (t.masked_fill(~key_mask[:, None, :, None], 0.0) for t in (kf, vf))      # (whatever masked places hold)
    if causal:
        see = see & torch.ones(Nq, Nk, dtype=torch.bool, device=q.device).tril(Nk - Nq)
    some = see.any(-1, keepdim=True)
    kf, vf = (t.repeat_interleave(H // Hk, dim=1) for t in (kf, vf))
    s = torch.matmul(qf, kf.transpose(-1, -2).contiguous()) * scale
    s = s.masked_fill(~see, -float("inf")).masked_fill(~some, 0.0)                         # (a row that sees nothing: zero, below)
    o = torch.matmul(torch.softmax(s, dim=-1), vf).masked_fill(~some, 0.0)
    return o.transpose(1, 2).reshape(B, Nq, H * d).to(q.dtype)


def attention(q, k, v, key_mask=None, causal=False, scale=None):
    """softmax(scale q k^T over the visible keys) v with its gradient: q [B, H, Nq, d], k / v [B, Hk, Nk, d] -> [B, Nq, H * d].

    Hk divides H: query head h reads key head h // (H / Hk). `scale` (default d ** -0.5) is positive. `key_mask` [B, Nk] bool: False
    keys are seen by no query, whatever their k and v hold, and get zero gradients. `causal`: query i sees keys <= i + Nk - Nq. A row that
    sees no key gives zeros and has no gradient.

    fp16 / bf16 CUDA tensors with d a multiple of 8 up to 256 run csrc/attention_train.hip: any batch / head / token strides (0 of an
    expanded tensor included; other layouts are copied), float32 accumulation and statistics, probabilities and their gradients rounded to
    the inputs' type for the second products. Everything else runs the same formulas in PyTorch ops. One derivative only."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or not q.is_floating_point():
        raise ValueError("attention: q, k and v must be floating-point [B, H, N, d] tensors")
    (B, H, Nq, d), (Bk, Hk, Nk, dk) = q.shape, k.shape
    if k.shape != v.shape or Bk != B or dk != d or (H % Hk if Hk else H):
        raise ValueError(f"attention: q {tuple(q.shape)} does not go with k {tuple(k.shape)} and v {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype) or not (q.device == k.device == v.device):
        raise ValueError("attention: q, k and v must have one type and one device")
    if key_mask is not None and (key_mask.dtype != torch.bool or tuple(key_mask.shape) != (B, Nk) or key_mask.device != q.device):
        raise ValueError(f"attention: key_mask must be a [{B}, {Nk}] bool tensor on {q.device}")
    scale = float(scale) if scale is not None else d ** -0.5 if d else 1.0
    if not 0.0 < scale < 3e38:
        raise ValueError(f"attention: the scale must be positive and finite, got {scale}")
    if 0 in (B, H, Nq, d) or Nk == 0:
        return (q.sum() + k.sum() + v.sum()) * 0 + torch.zeros(B, Nq, H * d, dtype=q.dtype, device=q.device)
    if not (q.is_cuda and q.dtype in (torch.float16, torch.bfloat16) and d % 8 == 0 and d <= 256):
        return _attention_plain(q, k, v, key_mask, causal, scale)
    keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _AttentionFn.apply(_taken(q), _taken(k), _taken(v), None if key_mask is None else key_mask.contiguous(), int(bool(causal)), scale, keep)
