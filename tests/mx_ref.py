"""Plain 64-bit implementations of MXFP4 and of the mixture-of-experts layer,
with the error bounds the kernels' arithmetic allows.

Bounds. A bf16 rounding is off by at most 2^-8 |value| (half a step), an fp32
sum of n exact products by at most n 2^-24 times the sum of their magnitudes
(in any order; 8 more steps allowed for how the matrix cores align terms).
"""
import numpy as np
import torch

U32, UBF = 2.0 ** -24, 2.0 ** -8
TINY = 2.0 ** -133                         # half of bf16's smallest subnormal is 2^-134


def bits(x):
    """uint16 codes of a bf16 tensor as int64."""
    return x.view(torch.int16).to(torch.int64) & 0xffff


def quantize(x):
    """(codes, scales) of a bf16 tensor [..., K], from its bits: integers
    throughout, each element the nearest of the eight magnitudes, ties to the
    even code."""
    c = bits(x).unflatten(-1, (-1, 32))
    e = (c & 0x7fff).amax(-1) >> 7
    s = torch.where(e == 255, e, (e - 2).clamp(min=0))
    v = x.double().abs().unflatten(-1, (-1, 32)) * torch.exp2(127.0 - s.double()).unsqueeze(-1)
    mags = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    d = (v.clamp(max=6.0).unsqueeze(-1) - mags).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best
    odd = torch.arange(8, device=x.device) % 2
    code = torch.where(near, odd + 1.0, 9.0).argmin(-1)          # of two as near, the even
    code = code | ((c >> 15) << 3)
    code = torch.where((s == 255).unsqueeze(-1), torch.zeros_like(code), code).flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8), s.to(torch.uint8)


def values(codes, scales):
    """The float64 values of (codes, scales)."""
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6],
                       dtype=torch.float64, device=codes.device)
    v = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).flatten(-2)
    s = torch.exp2(scales.double() - 127.0)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return v * s.repeat_interleave(32, -1)


def gemm(wv, xv):
    """y = x w^T in 64 bits, and the bound of its bf16 result."""
    y = xv @ wv.t()
    esc = xv.abs() @ wv.abs().t()
    return y, UBF * y.abs() * 1.01 + (wv.shape[1] + 8) * U32 * esc * 1.01 + TINY


def silu(g):
    return g * torch.sigmoid(g)


def _ffn(x, gu, dn):
    """One expert on rows x: values and error bounds of down(silu(g) u)."""
    H, I = x.shape[1], dn.shape[1]
    n = gu.shape[0] // 2
    g, u = x @ gu[:n].t(), x @ gu[n:].t()
    eg = (H + 8) * U32 * (x.abs() @ gu[:n].abs().t())
    eu = (H + 8) * U32 * (x.abs() @ gu[n:].abs().t())
    h = silu(g) * u
    # |silu'| <= 1.1; silu in fp32 (exp, add, divide, two products) <= 16
    # roundings and exp's argument error |g| 2^-24; h in 16 bits: 2^-16
    eh = 1.1 * u.abs() * eg + silu(g).abs() * eu + 1.1 * eg * eu + h.abs() * (
        2.0 ** -16 + (16 + 2 * g.abs()) * U32)
    o = h @ dn.t()
    eo = eh @ dn.abs().t() + (2 * I + 8) * U32 * ((h.abs() + eh) @ dn.abs().t())
    return o, eo


def moe(x, w, topk, norm, mx):
    """The layer in 64 bits: y, its bound, and per token the gap between the
    last chosen and the first left-out logit less what fp32 can move them
    (positive: the choice is safe)."""
    x = x.double()
    wt = lambda n, at=...: values(w["w_" + n][at], w["s_" + n][at]) if mx else w["w_" + n][at].double()
    wr = w["w_router"].double()
    T, H = x.shape
    E = wr.shape[0]
    l = x @ wr.t()
    el = ((H + 8) * U32 * (x.abs() @ wr.abs().t()))
    order = torch.argsort(l, dim=-1, descending=True, stable=True)
    top = order[:, :topk]
    gap = torch.full((T,), float("inf"), dtype=torch.float64, device=x.device)
    if topk < E:
        s = l.gather(1, order)
        gap = s[:, topk - 1] - s[:, topk] - 2 * el.amax(1)
    p = torch.zeros_like(l)
    q = torch.softmax(l.gather(1, top), -1) if norm else torch.softmax(l, -1).gather(1, top)
    p.scatter_(1, top, q)
    # each exponential moves by its argument's error (two logits') and 4 ulp
    # and its argument's rounding; the sum of them likewise; one division
    span = (l.amax(1, keepdim=True) - l.amin(1, keepdim=True))
    rp = 4 * el.amax(1, keepdim=True) + (2 * span + 2 * E + 32) * U32
    y, ey = torch.zeros_like(x), torch.zeros_like(x)
    ymag = torch.zeros_like(x)
    for e in range(E):
        rows = (p[:, e] > 0).nonzero().flatten()
        if rows.numel() == 0:
            continue
        o, eo = _ffn(x[rows], wt("gate_up", e), wt("down", e))
        pe = p[rows, e:e + 1]
        y[rows] += pe * o
        ymag[rows] += pe * o.abs()
        ey[rows] += pe * (eo + rp[rows] * (o.abs() + eo))
    if "w_shared_gate_up" in w:
        o, eo = _ffn(x, wt("shared_gate_up"), wt("shared_down"))
        if w.get("w_shared_gate") is not None:
            sg = w["w_shared_gate"].double()
            g = (x @ sg).unsqueeze(1)
            eg = ((H + 8) * U32 * (x.abs() @ sg.abs())).unsqueeze(1) + (8 + g.abs()) * U32
            s = torch.sigmoid(g)
        else:
            s, eg = torch.ones_like(x[:, :1]), torch.zeros_like(x[:, :1])
        y += s * o
        ymag += s * o.abs()
        ey += s * (eo + eg * (o.abs() + eo))
    bound = 1.01 * (UBF * y.abs() + (1 + UBF) * (ey + (2 * topk + 4) * U32 * ymag)) + TINY
    return y, bound, gap


def check(got, ref, bound, what=""):
    """Every element of a bf16 tensor within its bound, and the tensor within
    what the one rounding allows: 2^-8 of its norm, and 2^-12 for the sums,
    whose errors do not all point one way as the elements' bounds have it."""
    d = (got.double() - ref).abs()
    r = float((d / bound).max()) if d.numel() else 0.0
    n = float(d.norm() / ref.norm().clamp_min(1e-300)) if d.numel() else 0.0
    print(f"[mx] {what}: worst error {r:.3f} of its bound, normwise {n:.2e}", flush=True)
    assert bool((d <= bound).all()), f"{what}: {r} of the bound"
    assert n <= UBF + 2.0 ** -12, f"{what}: normwise {n}"


def normal(gen, *shape, scale=1.0, device="cuda"):
    return (torch.randn(*shape, generator=gen, device=device) * scale).to(torch.bfloat16)


def moe_weights(gen, H, I, E, Is, gate=True, mx=False, device="cuda"):
    w = dict(w_router=normal(gen, E, H, scale=H ** -0.5, device=device),
             w_gate_up=normal(gen, E, 2 * I, H, scale=H ** -0.5, device=device),
             w_down=normal(gen, E, H, I, scale=I ** -0.5, device=device))
    if Is:
        w.update(w_shared_gate_up=normal(gen, 2 * Is, H, scale=H ** -0.5, device=device),
                 w_shared_down=normal(gen, H, Is, scale=Is ** -0.5, device=device))
        if gate:
            w["w_shared_gate"] = normal(gen, H, scale=H ** -0.5, device=device)
    if mx:
        for n in [n for n in w if n.endswith(("gate_up", "down"))]:
            w[n], w["s" + n[1:]] = quantize(w[n])
    return w


def safe_tokens(gen, w, T, topk, H, skew=0.5):
    """T tokens whose choice of experts no fp32 sum's error can change."""
    dev = w["w_router"].device
    x = (torch.randn(3 * T + 64, H, generator=gen, device=dev)
         + skew * torch.randn(H, generator=gen, device=dev)).to(torch.bfloat16)
    E = w["w_router"].shape[0]
    if topk < E:
        wr = w["w_router"].double()
        l = (x.double() @ wr.t()).sort(dim=-1, descending=True).values
        el = (H + 8) * U32 * (x.double().abs() @ wr.abs().t()).amax(1)
        x = x[(l[:, topk - 1] - l[:, topk]) > 2 * el + 1e-4]
    assert x.shape[0] >= T
    return x[:T].contiguous()
