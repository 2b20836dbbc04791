"""Times the operators a gradient through the diffusion prior's blocks is made of: attention with its backward pass, group norm with
SiLU on channels-last maps, and GEGLU, the last two with their saved input held in 8 bits or as it is.

`run` with `own` false is the plain form of each (elementary tensor operations in float32, rounded once at the end); with `own` true
it makes the calls of sdfx_nerf. `exact` evaluates the definitions in float64 by other means (autograd on log-sum-exp, batch-norm-like
moments), for how far each of the two is off."""
import importlib
import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # self-attention of the UNet's top level (64 x 64 latents, classifier-free pair, 8 heads of 40), a training step's both directions
        {"name": "attn_self_4096_d40", "op": "attention", "B": 2, "H": 8, "Hk": 8, "Nq": 4096, "Nk": 4096, "d": 40, "dtype": "fp16",
         "causal": False, "mask": "none", "spread": 1.0, "grad": True},
        # cross-attention of the same level to 77 text tokens, prompts of unequal length: few keys, many queries
        {"name": "attn_cross_77_d40_mask", "op": "attention", "B": 2, "H": 8, "Hk": 8, "Nq": 4096, "Nk": 77, "d": 40, "dtype": "fp16",
         "causal": False, "mask": "prompt", "spread": 1.0, "grad": True},
        # the deepest attention level (16 x 16 latents, heads of 160): a small call, where latency counts
        {"name": "attn_self_256_d160_bf16", "op": "attention", "B": 2, "H": 8, "Hk": 8, "Nq": 256, "Nk": 256, "d": 160, "dtype": "bf16",
         "causal": False, "mask": "none", "spread": 1.0, "grad": True},
        # a causal text stack with shared key heads, odd length, peaked scores
        {"name": "attn_causal_1001_d64_gqa", "op": "attention", "B": 2, "H": 12, "Hk": 4, "Nq": 1001, "Nk": 1001, "d": 64, "dtype": "bf16",
         "causal": True, "mask": "none", "spread": 2.0, "grad": True},
        # one query against a long row of keys (no gradient): the single-token form
        {"name": "attn_one_query_16384_d128", "op": "attention", "B": 4, "H": 16, "Hk": 4, "Nq": 1, "Nk": 16384, "d": 128, "dtype": "fp16",
         "causal": False, "mask": "none", "spread": 1.0, "grad": False},
        # the norms of the UNet's top level, with the time embedding's vector, input kept in 8 bits
        {"name": "gn_64x64_c320_int8", "op": "group_norm", "N": 2, "H": 64, "W": 64, "C": 320, "G": 32, "dtype": "fp16", "params": "fp32",
         "act": True, "pre": True, "checkpoint": "int8"},
        # the largest map: the VAE encoder's first level at 512 x 512, input kept in 8 bits
        {"name": "gn_512x512_c128_int8", "op": "group_norm", "N": 1, "H": 512, "W": 512, "C": 128, "G": 32, "dtype": "fp16", "params": "fp16",
         "act": True, "pre": False, "checkpoint": "int8"},
        # the deepest level (8 x 8): latency
        {"name": "gn_8x8_c1280_bf16", "op": "group_norm", "N": 2, "H": 8, "W": 8, "C": 1280, "G": 32, "dtype": "bf16", "params": "bf16",
         "act": True, "pre": True, "checkpoint": "full"},
        # an odd map in float32 (a prior that runs without half precision), no activation
        {"name": "gn_37x53_c96_fp32", "op": "group_norm", "N": 3, "H": 37, "W": 53, "C": 96, "G": 8, "dtype": "fp32", "params": "fp32",
         "act": False, "pre": False, "checkpoint": "full"},
        # the feed-forward of the UNet's top level: 2 x 4096 tokens, 2 x 1280 channels, input kept in 8 bits
        {"name": "geglu_8192_n1280_int8", "op": "geglu", "rows": 8192, "n": 1280, "dtype": "fp16", "checkpoint": "int8"},
        # the deepest level: 2 x 64 tokens, 2 x 5120 channels
        {"name": "geglu_128_n5120", "op": "geglu", "rows": 128, "n": 5120, "dtype": "bf16", "checkpoint": "full"},
        # a ragged number of tokens
        {"name": "geglu_1001_n640_int8_bf16", "op": "geglu", "rows": 1001, "n": 640, "dtype": "bf16", "checkpoint": "int8"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "group_norm", "geglu"])
    half = rng.choice(["fp16", "bf16"])
    if op == "attention":
        hk = rng.choice([1, 2, 3, 4, 8])
        c = {"op": op, "B": rng.randint(1, 4), "H": hk * rng.choice([1, 1, 2, 3]), "Hk": hk, "Nq": _log(rng, 1, 4096), "Nk": _log(rng, 1, 8192),
             "d": 8 * rng.randint(1, 32), "dtype": half, "causal": rng.random() < 0.3, "mask": rng.choice(["none", "prompt", "holes"]),
             "spread": rng.choice([0.5, 1.0, 2.0]), "grad": rng.random() < 0.8}
        if c["causal"]:
            c["Nk"] = c["Nq"]
        while c["B"] * c["H"] * c["Nq"] * c["Nk"] * max(c["d"], 40) > 2 * 8 * 4096 * 4096 * 40:
            c["Nq"] = (c["Nq"] + 1) // 2
            c["Nk"] = c["Nq"] if c["causal"] else (c["Nk"] + 1) // 2
        return c
    if op == "group_norm":
        G = rng.choice([8, 16, 32])
        check = rng.choice(["full", "int8"])
        dtype = rng.choice([half, half, "fp32"])
        C = 32 * rng.randint(1, 40) if check == "int8" else G * rng.choice([1, 2, 4, 5, 8, 10, 20, 40])
        C = C if C % G == 0 and C % 8 == 0 else 32 * ((C + 31) // 32)
        N = rng.randint(1, 4)
        most = 512 * 512 * 128 // (N * C * (2 if dtype == "fp32" else 1))
        px = _log(rng, 16, max(16, min(512 * 512, most)))     # (a group of a few elements has no gradient but rounding)
        H = _log(rng, 1, max(1, int(px ** 0.5)))
        return {"op": op, "N": N, "H": H, "W": max(1, px // H), "C": C, "G": G, "dtype": dtype, "params": rng.choice([dtype, "fp32"]),
                "act": rng.random() < 0.7, "pre": rng.random() < 0.5, "checkpoint": check}
    check = rng.choice(["full", "int8"])
    dtype = rng.choice([half, half, "fp32"])
    n = 32 * rng.randint(1, 160) if check == "int8" else 8 * rng.randint(1, 640)
    return {"op": op, "rows": _log(rng, 1, max(1, min(65536, 8192 * 1280 // n))), "n": n, "dtype": dtype, "checkpoint": check}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    rn = lambda *shape, s=1.0, dtype=dt: (torch.randn(*shape, generator=g, device=dev) * s).to(dtype)
    st = dict(case)
    if case["op"] == "attention":
        B, H, Hk, Nq, Nk, d = (case[k] for k in ("B", "H", "Hk", "Nq", "Nk", "d"))
        heads = lambda n, h, s: rn(B, n, h * d, s=s).view(B, n, h, d).transpose(1, 2)     # the views of a projection's output
        st["q"], st["k"], st["v"] = heads(Nq, H, case["spread"]), heads(Nk, Hk, case["spread"]), heads(Nk, Hk, 1.0)
        st["key_mask"] = None
        if case["mask"] == "prompt":          # prompts of unequal length, the first of them empty where there are three or more
            n = torch.randint(1, Nk + 1, (B,), generator=g, device=dev)
            if B > 2:
                n[0] = 0
            st["key_mask"] = torch.arange(Nk, device=dev)[None] < n[:, None]
        elif case["mask"] == "holes":
            st["key_mask"] = torch.rand(B, Nk, generator=g, device=dev) < 0.7
        if case["grad"]:
            st["q"], st["k"], st["v"] = (t.requires_grad_(True) for t in (st["q"], st["k"], st["v"]))
            st["dy"] = rn(B, Nq, H * d)
    elif case["op"] == "group_norm":
        N, H, W, C = (case[k] for k in ("N", "H", "W", "C"))
        cl = lambda t: t.permute(0, 3, 1, 2)                                              # [N, H, W, C] memory
        pt = _DTYPES[case["params"]]
        shift = torch.randn(C, generator=g, device=dev)
        st["x"] = cl((torch.randn(N, H, W, C, generator=g, device=dev) * 1.5 + shift).to(dt)).requires_grad_(True)
        st["pre"] = rn(N, C).requires_grad_(True) if case["pre"] else None
        st["weight"] = (1 + 0.2 * torch.randn(C, generator=g, device=dev)).to(pt).requires_grad_(True)
        st["bias"] = rn(C, s=0.2, dtype=pt).requires_grad_(True)
        st["dy"] = cl(rn(N, H, W, C))
    else:
        st["x"] = rn(case["rows"], 2 * case["n"]).requires_grad_(True)
        st["dy"] = rn(case["rows"], case["n"])
    if own:
        importlib.import_module("stable-dreamfusion_amd")
        st["attention"] = importlib.import_module("sdfx_nerf.attention")
        st["groupnorm"] = importlib.import_module("sdfx_nerf.groupnorm")
    return st


def run(st):
    if own:
        return _own(st)
    with torch.no_grad():
        return {"attention": _plain_attention, "group_norm": _plain_group_norm, "geglu": _plain_geglu}[st["op"]](st)


def _own(st):
    if st["op"] == "attention":
        if not st["grad"]:
            with torch.no_grad():
                return {"o": st["attention"].attention(st["q"], st["k"], st["v"], key_mask=st["key_mask"], causal=st["causal"])}
        o = st["attention"].attention(st["q"], st["k"], st["v"], key_mask=st["key_mask"], causal=st["causal"])
        dq, dk, dv = torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["dy"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    if st["op"] == "group_norm":
        y = st["groupnorm"].group_norm_act(st["x"], st["G"], st["weight"], st["bias"], eps=1e-5, act=st["act"], pre=st["pre"],
                                           checkpoint=st["checkpoint"])
        names = ["x", "weight", "bias"] + (["pre"] if st["pre"] is not None else [])
        grads = torch.autograd.grad(y, [st[n] for n in names], st["dy"])
        return {"y": y.detach(), **{"d" + n: t for n, t in zip(names, grads)}}
    y = st["groupnorm"].geglu(st["x"], checkpoint=st["checkpoint"])
    (dx,) = torch.autograd.grad(y, (st["x"],), st["dy"])
    return {"y": y.detach(), "dx": dx}


# ---- plain forms ----------------------------------------------------------------------------------------------------------------

def _visible(st, Nq, Nk, device):
    """[B or 1, 1, Nq or 1, Nk] truth values, or None: which keys a query sees (the last query sees every key of a causal row)."""
    see = None if st["key_mask"] is None else st["key_mask"][:, None, None, :]
    if st["causal"]:
        tri = torch.arange(Nk, device=device)[None, :] <= torch.arange(Nq, device=device)[:, None] + (Nk - Nq)
        see = tri[None, None] if see is None else see & tri[None, None]
    return see


def _plain_attention(st):
    dt = st["q"].dtype
    q, k, v = st["q"].float().contiguous(), st["k"].float().contiguous(), st["v"].float().contiguous()
    B, H, Nq, d = q.shape
    Hk, Nk = k.shape[1], k.shape[2]
    scale = d ** -0.5
    if Hk != H:
        k, v = k.repeat_interleave(H // Hk, dim=1), v.repeat_interleave(H // Hk, dim=1)
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    see = _visible(st, Nq, Nk, q.device)
    if see is not None:
        s = s.masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    del s
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, torch.ones_like(l), l)
    o = torch.matmul(p, v)
    out = {"o": o.transpose(1, 2).reshape(B, Nq, H * d).to(dt)}
    if not st["grad"]:
        return out
    do = st["dy"].float().view(B, Nq, H, d).transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q)
    if Hk != H:
        dk, dv = (t.view(B, Hk, H // Hk, Nk, d).sum(2) for t in (dk, dv))
    return {**out, "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt)}


def _eight_bits(x):
    """What the 8-bit form of x [..., C] stands for: blocks of 32 channels share a step 2^(floor(log2 max|x|) - 6)."""
    b = x.unflatten(-1, (-1, 32))
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (e - 7).clamp(min=-126)                                       # frexp's mantissa lies in [1/2, 1): floor(log2) = e - 1
    return torch.ldexp(torch.round(torch.ldexp(b, -e)).clamp(-127, 127), e).flatten(-2)


def _plain_group_norm(st):
    N, C, H, W = st["x"].shape
    G, act = st["G"], st["act"]
    x = st["x"].float().permute(0, 2, 3, 1)
    pre = 0.0 if st["pre"] is None else st["pre"].float()[:, None, None, :]
    w, b = st["weight"].float(), st["bias"].float()
    grouped = lambda t: t.reshape(N, H * W, G, C // G)
    u = grouped((x + pre).contiguous())
    mean = u.double().mean((1, 3), keepdim=True)                      # (moments of long rows: in float64)
    rstd = 1.0 / torch.sqrt((u.double() - mean).square().mean((1, 3), keepdim=True) + 1e-5)
    mean, rstd = mean.float(), rstd.float()
    z = ((u - mean) * rstd).view(N, H, W, C) * w + b
    y = z / (1 + torch.exp(-z)) if act else z
    xs = _eight_bits(x) if st["checkpoint"] == "int8" else x
    xh = (grouped((xs + pre).contiguous()) - mean) * rstd
    dz = st["dy"].float().permute(0, 2, 3, 1)
    if act:
        z = xh.view(N, H, W, C) * w + b
        sg = 1 / (1 + torch.exp(-z))
        dz = dz * sg * (1 + z * (1 - sg))
    g = grouped((dz * w).contiguous())
    dx = (rstd * (g - g.double().mean((1, 3), keepdim=True).float() - xh * (g * xh).double().mean((1, 3), keepdim=True).float())).view(N, H, W, C)
    dt, pt = st["x"].dtype, st["weight"].dtype
    flat = lambda t: t.reshape(N * H * W, C).double().sum(0)
    out = {"y": y.to(dt).permute(0, 3, 1, 2), "dx": dx.to(dt).permute(0, 3, 1, 2), "dweight": flat(dz * xh.view(N, H, W, C)).to(pt),
           "dbias": flat(dz).to(pt)}
    if st["pre"] is not None:
        out["dpre"] = dx.reshape(N, H * W, C).double().sum(1).to(dt)
    return out


def _plain_geglu(st):
    n, dt = st["n"], st["x"].dtype
    x, dy = st["x"].float(), st["dy"].float()
    cdf = lambda g: 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    y = x[:, :n] * x[:, n:] * cdf(x[:, n:])
    if st["checkpoint"] == "int8":
        x = _eight_bits(x)
    a, g = x[:, :n], x[:, n:]
    phi = torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    dx = torch.cat([dy * g * cdf(g), dy * a * (cdf(g) + g * phi)], dim=1)
    return {"y": y.to(dt), "dx": dx.to(dt)}


# ---- definitions in 64 bits -----------------------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    with torch.enable_grad():
        return {"attention": _exact_attention, "group_norm": _exact_group_norm, "geglu": _exact_geglu}[case["op"]](st)


def _exact_attention(st):
    B, H, Nq, d = st["q"].shape
    Hk, Nk = st["k"].shape[1:3]
    see = _visible(st, Nq, Nk, st["q"].device)
    names = ("o", "dq", "dk", "dv") if st["grad"] else ("o",)
    out = {"o": torch.zeros(B, Nq, H, d, dtype=torch.float64, device=st["q"].device)}
    if st["grad"]:
        out.update({"d" + n: torch.zeros(st[n].shape, dtype=torch.float64, device=st[n].device) for n in ("q", "k", "v")})
        dy = st["dy"].view(B, Nq, H, d)
    for b in range(B):                                                # a head at a time: 4096 x 4096 scores in float64 are 128 MB
        vis = None if see is None else see[b if see.shape[0] > 1 else 0, 0]
        for h in range(H):
            hk = h // (H // Hk)
            q, k, v = (t.detach().double().requires_grad_(st["grad"]) for t in (st["q"][b, h], st["k"][b, hk], st["v"][b, hk]))
            s = (q / math.sqrt(d)) @ k.t()
            if vis is not None:
                s = torch.where(vis, s, torch.full((), -1e300, dtype=s.dtype, device=s.device))
            p = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
            if vis is not None:
                p = p * vis.double()                                  # (a row that sees nothing: zero, not the mean)
            o = p @ v
            out["o"][b, :, h] = o.detach()
            if st["grad"]:
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), dy[b, :, h].double())
                out["dq"][b, h] += gq
                out["dk"][b, hk] += gk
                out["dv"][b, hk] += gv
    out["o"] = out["o"].view(B, Nq, H * d)
    return {n: out[n] for n in names}


def _exact_group_norm(st):
    N, C, H, W = st["x"].shape
    leaf = lambda t: t.detach().double().requires_grad_(True)
    x, w, b = leaf(st["x"]), leaf(st["weight"]), leaf(st["bias"])
    pre = None if st["pre"] is None else leaf(st["pre"])

    def normed(u):
        r = u.reshape(N, st["G"], -1)
        mean = r.mean(-1, keepdim=True)
        rstd = (r.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
        return r, mean, rstd

    def output(r, mean, rstd):
        z = ((r - mean) * rstd).view(N, C, H, W) * w[None, :, None, None] + b[None, :, None, None]
        return z * torch.sigmoid(z) if st["act"] else z

    shifted = lambda t: t if pre is None else t + pre[:, :, None, None]
    r, mean, rstd = normed(shifted(x))
    y = output(r, mean, rstd)
    leaves = [x, w, b] + ([] if pre is None else [pre])
    if st["checkpoint"] == "int8":
        # the backward evaluates the derivative's formula at the 8-bit input with the statistics of the forward
        xs = _eight_bits(st["x"].detach().double().permute(0, 2, 3, 1)).permute(0, 3, 1, 2)
        with torch.no_grad():
            xh = ((shifted(xs).reshape(N, st["G"], -1) - mean) * rstd).view(N, C, H, W)
        z = (xh * w[None, :, None, None] + b[None, :, None, None]).detach().requires_grad_(True)
        ya = z * torch.sigmoid(z) if st["act"] else z * 1.0
        (dz,) = torch.autograd.grad(ya, z, st["dy"].double())
        with torch.no_grad():
            gr, xr = (dz * w[None, :, None, None]).reshape(N, st["G"], -1), xh.reshape(N, st["G"], -1)
            dx = (rstd * (gr - gr.mean(-1, keepdim=True) - xr * (gr * xr).mean(-1, keepdim=True))).view(N, C, H, W)
            grads = [dx, (dz * xh).sum((0, 2, 3)), dz.sum((0, 2, 3))] + ([] if pre is None else [dx.sum((2, 3))])
    else:
        grads = torch.autograd.grad(y, leaves, st["dy"].double())
    out = {"y": y.detach(), "dx": grads[0], "dweight": grads[1], "dbias": grads[2]}
    if pre is not None:
        out["dpre"] = grads[3]
    return out


def _exact_geglu(st):
    x = st["x"].detach().double().requires_grad_(True)
    a, g = x.chunk(2, dim=1)
    y = a * torch.nn.functional.gelu(g)
    at = x if st["checkpoint"] == "full" else _eight_bits(x.detach()).requires_grad_(True)
    a, g = at.chunk(2, dim=1)
    (dx,) = torch.autograd.grad(a * torch.nn.functional.gelu(g), at, st["dy"].double())
    return {"y": y.detach(), "dx": dx}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "attention":
        B, H, Hk, Nq, Nk, d = (case[k] for k in ("B", "H", "Hk", "Nq", "Nk", "d"))
        pairs = B * H * (Nq * (Nq + 1) // 2 if case["causal"] else Nq * Nk)
        qs, ks = B * H * Nq * d, B * Hk * Nk * d
        if not case["grad"]:
            return {"bytes": size * (2 * qs + 2 * ks), "flops": 4 * pairs * d}
        return {"bytes": size * (4 * qs + 4 * ks), "flops": 14 * pairs * d}          # q, dy, o, dq; k, v, dk, dv; 2 + 5 products
    if case["op"] == "group_norm":
        e = case["N"] * case["H"] * case["W"] * case["C"]
        return {"bytes": 4 * size * e, "flops": 30 * e}
    e = case["rows"] * case["n"]
    return {"bytes": 6 * size * e, "flops": 40 * e}
