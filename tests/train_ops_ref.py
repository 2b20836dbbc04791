"""float64 references of the training operators (sdfx_nerf.attention.attention, groupnorm.group_norm_act, groupnorm.geglu) with elementwise
error bounds, from the number of roundings each value goes through. u = eps / 2 is half a step of the inputs' type.

attention. Scores are float32 sums of d products: together with the exponential's argument and the row sum a probability is off by less than
S = 1e-4 of itself for the scores used here (|s| < 60). Probabilities and ds are rounded to the inputs' type (u each), results once (u).
  |o| error      <= (2 u + S) p |v|
  |dv| error     <= (2 u + S) p^T |do|
  dp - delta     <= 1e-4 E, E = |do| |v|^T + |do| |o|: float32 sums, and o known to u^2 <= 2^-16 of itself (it is kept with its rounding error)
  delta          also carries the forward's rounding of the probabilities in o: |sum_c do_c sum_j (rounding of p_j) v_jc| <= u F,
                 F = sum_c |do_c| sum_j p_j |v_jc|
  |dq| error     <= scale ((u + S) |ds| + p (1e-4 E + u F)) |k| + u |dq|, dk likewise with the transpose and |q|
fp16 also has a smallest step, 2^-25 after rounding: of the unnormalised probabilities in the forward (their largest is 1), of 2^15 p and of ds in
units of its bound in the backward (2^-37 max |do| max |v|), and of every result.

group norm / GEGLU. float32 arithmetic with a few dozen operations a value, hardware exponential and reciprocal: R = 2^-18 of the magnitudes that
enter (written out below), then one rounding u of the result."""
import math

import torch

S = 1e-4
R = 2.0 ** -18


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, dy, key_mask=None, causal=False, scale=None):
    """[o, dq, dk, dv] and their bounds, float64 on the CPU; q [B, H, Nq, d], k / v [B, Hk, Nk, d], dy [B, Nq, H * d]."""
    dt = q.dtype
    u = half_step(dt)
    q, k, v, dy = (t.detach().cpu().double() for t in (q, k, v, dy))
    B, H, Nq, d = q.shape
    Hk, Nk = k.shape[1:3]
    G = H // Hk
    scale = d ** -0.5 if scale is None else scale
    see = torch.ones(B, 1, Nq, Nk, dtype=torch.bool)
    if key_mask is not None:
        m = key_mask.cpu()
        see = see & m[:, None, None, :]
        k, v = (torch.where(m[:, None, :, None], t, torch.zeros_like(t)) for t in (k, v))
    if causal:
        see = see & (torch.arange(Nk)[None, :] <= torch.arange(Nq)[:, None] + (Nk - Nq))
    do = dy.view(B, Nq, H, d).transpose(1, 2)
    some = see.any(-1, keepdim=True)
    do = torch.where(some, do, torch.zeros_like(do))
    ke, ve = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.where(see, (q @ ke.transpose(-1, -2)) * scale, torch.full((), -1e300, dtype=torch.float64))
    p = torch.exp(s - s.amax(-1, keepdim=True)) * see
    p = p / torch.where(some, p.sum(-1, keepdim=True), torch.ones_like(some, dtype=torch.float64))
    o = p @ ve
    dp = do @ ve.transpose(-1, -2)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    shared = lambda t: t.view(B, Hk, G, Nk, d).sum(2)
    dq, dk, dv = scale * (ds @ ke), scale * shared(ds.transpose(-1, -2) @ q), shared(p.transpose(-1, -2) @ do)
    E = do.abs() @ ve.abs().transpose(-1, -2) + (do * o).abs().sum(-1, keepdim=True)
    F = (do.abs() * (p @ ve.abs())).sum(-1, keepdim=True)
    eds = (u + S) * ds.abs() + p * (1e-4 * E + u * F)
    least = 2.0 ** -25 if dt == torch.float16 else 0.0
    ds_least = 2.0 ** -37 * float(do.norm(dim=-1).max() * ve.norm(dim=-1).max()) if dt == torch.float16 else 0.0
    bo = (2 * u + S) * (p @ ve.abs()) + least * (1 + ve.abs().sum(-2, keepdim=True)) * some
    bdq = scale * (eds @ ke.abs() + ds_least * ke.abs().sum(-2, keepdim=True)) + u * dq.abs() + least
    bdk = shared(scale * (eds.transpose(-1, -2) @ q.abs() + ds_least * q.abs().sum(-2, keepdim=True))) + u * dk.abs() + least
    bdv = shared((2 * u + S) * (p.transpose(-1, -2) @ do.abs()) + least * 2.0 ** -15 * do.abs().sum(-2, keepdim=True)) + least
    flat = lambda t: t.transpose(1, 2).reshape(B, Nq, H * d)
    return [flat(o), dq, dk, dv], [flat(bo), bdq, bdk, bdv]


def eight_bits(x):
    """The 8-bit form, block by block in Python numbers' arithmetic (float64, exact): x [rows, C]."""
    b = x.detach().cpu().double().reshape(-1, 32)
    m = b.abs().amax(-1, keepdim=True)
    step = torch.pow(2.0, torch.floor(torch.log2(m.clamp(min=2.0 ** -140))) - 6).clamp(min=2.0 ** -126)
    out = torch.round(b / step).clamp(-127, 127) * step
    return torch.where(torch.isfinite(m), out, torch.full_like(out, math.nan)).reshape(x.shape)


def group_norm(x, groups, weight, bias, dy, eps=1e-5, act=True, pre=None, eight=False):
    """{name: (value, bound)} for y, dx, dweight, dbias and dpre."""
    u, up = half_step(x.dtype), half_step(weight.dtype)
    xd, w, b, dz = (t.detach().cpu().double() for t in (x, weight, bias, dy))
    N, C, H, W = xd.shape
    e = torch.zeros(N, C).double() if pre is None else pre.detach().cpu().double()
    per = lambda t: t.reshape(N, groups, -1)
    full = lambda t: t.expand(N, groups, C // groups * H * W).reshape(N, C, H, W)
    ch = lambda t: t[None, :, None, None]
    U = xd + e[:, :, None, None]
    mean, var = per(U).mean(-1, keepdim=True), per(U).var(-1, unbiased=False, keepdim=True)
    rstd = full((var + eps).rsqrt())
    mean = full(mean)
    sig = torch.sigmoid
    z = (U - mean) * rstd * ch(w) + ch(b)
    y = z * sig(z) if act else z
    far = (mean.abs() + e.abs()[:, :, None, None]) * rstd          # float32's view of a distant mean: its step against the deviation
    by = u * y.abs() + R * (1 + z.abs()) * (1 + z.abs() + (far + 1) * ch(w).abs())
    if eight:
        xd = eight_bits(xd.permute(0, 2, 3, 1).reshape(-1, C)).reshape(N, H, W, C).permute(0, 3, 1, 2)
    xh = (xd + e[:, :, None, None] - mean) * rstd
    z = xh * ch(w) + ch(b)
    if act:
        dz = dz * sig(z) * (1 + z * (1 - sig(z)))
    g = dz * ch(w)
    avg = lambda t: full(per(t).mean(-1, keepdim=True))
    dx = rstd * (g - avg(g) - xh * avg(g * xh))
    wide = (1 + z.abs()) * (1 + far * ch(w).abs())                 # how far z's error carries into dz
    a, ax = dy.detach().cpu().double().abs() * wide * (ch(w).abs() + 1e-30), (1 + xh.abs() + far)
    bdx = u * dx.abs() + R * rstd * (a + avg(a) + ax * avg(a * ax))
    da = dy.detach().cpu().double().abs() * wide
    out = {"y": (y, by), "dx": (dx, bdx)}
    red = lambda t: t.sum((0, 2, 3))
    out["dweight"] = (red(dz * xh), up * red(dz * xh).abs() + R * red(da * ax))
    out["dbias"] = (red(dz), up * red(dz).abs() + R * red(da))
    if pre is not None:
        d = dx.sum((2, 3))
        out["dpre"] = (d, u * d.abs() + R * (rstd * (a + avg(a) + ax * avg(a * ax))).sum((2, 3)))
    return out


def geglu(x, dy, eight=False):
    u = half_step(x.dtype)
    xd, d = x.detach().cpu().double(), dy.detach().cpu().double()
    n = xd.shape[-1] // 2
    cdf = lambda t: 0.5 * (1 + torch.erf(t * math.sqrt(0.5)))
    a, g = xd[..., :n], xd[..., n:]
    y = a * g * cdf(g)
    by = u * y.abs() + R * a.abs() * g.abs()
    if eight:
        xd = eight_bits(xd.reshape(-1, 2 * n)).reshape(xd.shape)
    a, g = xd[..., :n], xd[..., n:]
    pdf = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    dx = torch.cat([d * g * cdf(g), d * a * (cdf(g) + g * pdf)], -1)
    bdx = u * dx.abs() + R * torch.cat([d.abs() * g.abs(), d.abs() * a.abs() * (1 + g.abs())], -1)
    return {"y": (y, by), "dx": (dx, bdx)}


def check(name, got, want, bound, least=0.0):
    """Every element within its bound (`least`: the type's smallest step, where results may be subnormal)."""
    got = got.detach().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    least = max(least, {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}.get(got.dtype, 0.0))
    over = (got.double() - want).abs() - bound - least
    assert torch.isfinite(got.double()).all(), name
    worst = int(over.argmax())
    assert float(over.max()) <= 0, (name, float(got.double().flatten()[worst]), float(want.flatten()[worst]), float(bound.flatten()[worst]),
                                    f"{int((over > 0).sum())} of {over.numel()}")
