"""A decode step as a program makes it of the library's calls: an attention
layer on a paged cache, then the mixture-of-experts layer, whose weights were
brought to MXFP4 by mxfp4_quantize, then an MXFP4 output product. Residuals and
norms between them are torch's. What each call returns is held against the
64-bit implementation on that call's own inputs, and the same steps on a stream
of their own give the same bits."""
import numpy as np
import pytest

import mx_ref
import synth

pytestmark = pytest.mark.gpu

H, I, E, K, IS, OUT = 2048, 256, 24, 4, 128, 1000


def _norm(torch, x):
    v = x.float()
    return (v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)


def _mx(hip, torch, w):
    """(codes, scales) of weights [..., K] by the library, checked bit for bit."""
    rows = w.reshape(-1, w.shape[-1])
    c = torch.empty(rows.shape[0], rows.shape[1] // 2, dtype=torch.uint8, device="cuda")
    s = torch.empty(rows.shape[0], rows.shape[1] // 32, dtype=torch.uint8, device="cuda")
    hip.mxfp4_quantize(rows, c, s)
    rc, rs = mx_ref.quantize(rows)
    assert torch.equal(c, rc) and torch.equal(s, rs)
    return c.view(*w.shape[:-1], -1), s.view(*w.shape[:-1], -1)


def _attn(hip, torch, rng):
    nh, nkv, d, _, _ = synth.ATTN_DIMS
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int16)
                                     if a.dtype == np.uint16 else np.ascontiguousarray(a)).to("cuda")
    s = H ** -0.5
    layer = hip.attn_layer(synth.ATTN_DIMS, {n: dev(v) for n, v in synth.attn_weights(rng).items()})
    proj = hip.attn_proj(H, dict(wq=dev(synth.normal_bf16(rng, (nh * 2 * d, H), s)),
                                 wk=dev(synth.normal_bf16(rng, (nkv * d, H), s)),
                                 wv=dev(synth.normal_bf16(rng, (nkv * d, H), s)),
                                 wo=dev(synth.normal_bf16(rng, (H, nh * d), (nh * d) ** -0.5))))
    return layer, proj


@pytest.mark.parametrize("B", [1, 2, 7, 20])
def test_decode_steps(hip, B):
    import torch
    print(f"[step] B={B}", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(B)
    layer, proj = _attn(hip, torch, np.random.default_rng(B))
    nh, nkv, d, _, _ = synth.ATTN_DIMS
    w = mx_ref.moe_weights(g, H, I, E, IS)
    for n in [n for n in w if n.endswith(("gate_up", "down"))]:
        w[n], w["s" + n[1:]] = _mx(hip, torch, w[n])
    moe = hip.moe_layer((H, I, E, K, IS), w)
    work = hip.MoeWork(moe, B)
    head, hs = _mx(hip, torch, mx_ref.normal(g, OUT, H, scale=H ** -0.5))
    x0 = mx_ref.normal(g, B, H)
    cu = np.arange(B + 1, dtype=np.int32)
    bf = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")

    def steps(n, keep):
        pool = hip.KvPool(1, nkv, d, B + 1, B, 1)
        rows = [pool.open() for _ in range(B)]
        for r in rows:
            pool.reserve(r, 32)
        x = x0
        for t in range(n):
            ao = torch.empty(B, H, dtype=torch.int16, device="cuda")
            hip.attn_layer_decode_paged(layer, proj, rows, cu, np.full(B, t, np.int32), _norm(torch, x).view(torch.int16),
                                        pool.cache(0), ao)
            x = x + ao.view(torch.bfloat16)
            ln2, y = _norm(torch, x), bf(B, H)
            hip.moe_layer_decode(moe, work, ln2, y)
            x = x + y
            last, z, zq = _norm(torch, x), bf(B, OUT), bf(B, OUT)
            hip.mxfp4_gemm(head, hs, last, z)
            c, s = (torch.empty(B, H // q, dtype=torch.uint8, device="cuda") for q in (2, 32))
            hip.mxfp4_quantize(last, c, s)
            hip.mxfp4_gemm_mx(head, hs, c, s, zq)
            keep.append((ln2, y, last, z, c, s, zq))
        torch.cuda.current_stream().synchronize()
        pool.destroy()

    eager, other = [], []
    steps(4, eager)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        hip.set_stream(st.cuda_stream)
        try:
            steps(4, other)
        finally:
            hip.set_stream(0)
    torch.cuda.synchronize()
    for a, b in zip(eager, other):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    safe = 0
    hv = mx_ref.values(head, hs)
    for ln2, y, last, z, c, s, zq in eager:
        r, b, gap = mx_ref.moe(ln2, w, K, True, True)
        ok = gap > 1e-4                                    # (the choice no fp32 sum's error can change)
        safe += int(ok.sum())
        mx_ref.check(y[ok], r[ok], b[ok], "moe")
        mx_ref.check(z, *mx_ref.gemm(hv, last.double()), "head")
        rc, rs = mx_ref.quantize(last)
        assert torch.equal(c, rc) and torch.equal(s, rs)
        mx_ref.check(zq, *mx_ref.gemm(hv, mx_ref.values(c, s)), "head of MXFP4")
    assert safe >= 2 * B                                   # (most of the 4 B choices)
    work.destroy()
