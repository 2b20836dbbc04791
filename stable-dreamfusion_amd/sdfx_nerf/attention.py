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
import _devswitch
import _sdfx

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
    qf = qf.masked_fill(~some, 0.0)                                                        # (nor what rows hold that see nothing)
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

    fp16 / bf16 CUDA tensors with d a multiple of 8 up to 256 and a scale in 1e-30 .. 1e30 run csrc/attention_train.hip: any batch / head / token strides (0 of an
    expanded tensor included; other layouts are copied), float32 accumulation and statistics, probabilities and their gradients rounded to
    the inputs' type for the second products. Scores are float32: a probability is off by 2^-24 of the largest scaled score beside those roundings
    (in the gradient, where it is found again from the log-sum-exp, as a factor of its row), so scaled scores should stay below some 10^4. Everything else runs the same formulas in PyTorch ops. One derivative only."""
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
        return torch.zeros(B, Nq, H * d, dtype=q.dtype, device=q.device) + sum(t[:0].sum() for t in (q, k, v))    # (in the graph; no value is read)
    if not (q.is_cuda and q.dtype in (torch.float16, torch.bfloat16) and d % 8 == 0 and d <= 256 and 1e-30 <= scale <= 1e30):
        return _attention_plain(q, k, v, key_mask, causal, scale)
    return _sdfx.native().attention(q, k, v, key_mask, causal, scale)
