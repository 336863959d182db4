"""The norms around a block on the GPU, against 64-bit arithmetic."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()


def rows(rng, t, n, pad, f32, scale=1.0):
    x = rng.normal(size=(t, n + pad)) * scale
    return dev(x.astype(np.float32) if f32 else R.bf16(x))[:, pad:]


def val(t):
    a = t.cpu().numpy()
    return a.astype(np.float64) if a.dtype == np.float32 else R.f64(a.view(np.uint16))


def rms(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + w)


def expect(y, h, post, pre, gate, scale, eps):
    """(h', its terms' magnitudes, x, its error where h' is off by a step of fp32)."""
    if y is None:
        t = np.zeros_like(h)
    else:
        t = y if post is None else rms(y, post, eps)
        t = scale * (t if gate is None else t * gate)
    h2 = h + t
    mag = np.abs(h) + np.abs(t)
    return h2, mag, None if pre is None else rms(h2, pre, eps)


# fp32: a sum of n squares in some order, its root and at most 8 operations on a
# value: n 2^-24 / 2 for the root of the sum, 8 2^-24 for the rest
def rel32(n):
    return (n / 2 + 8) * 2.0 ** -24


def check(norm, y, h, h_out, x, post, pre, gate, scale, eps):
    h0, y0 = val(h), None if y is None else val(y)
    n = h.shape[1]
    g = None if gate is None else val(gate) if gate.dim() == 2 else val(gate[None])
    wp, wq = (None if w is None else val(w[None])[0] for w in (post, pre))
    yield_ = expect(y0, h0, wp, wq, g, float(np.float32(scale)), float(np.float32(eps)))
    h2, mag, x2 = yield_
    f = rel32(n) * mag                     # h' before its rounding
    if h_out is not None:
        u = 2.0 ** -24 if h_out.dtype == torch.float32 else R.U
        assert (np.abs(val(h_out) - h2) <= f * (1 + u) + u * np.abs(h2) + 2.0 ** -133).all()
    if x is not None:
        # x = h' r: its own h' and the root of the mean of the squares
        ss = np.sqrt((h2 * h2).mean(-1, keepdims=True) + eps)
        dr = (f * np.abs(h2)).sum(-1, keepdims=True) / n / ss ** 2 + rel32(n)
        e = (f + np.abs(h2) * dr) / ss * np.abs(1 + wq)
        assert (np.abs(val(x) - x2) <= e * (1 + R.U) + R.U * np.abs(x2) + 2.0 ** -133).all()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("gate", ["none", "one", "rows"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("t,n,pad", [(1, 2048, 0), (5, 8, 0), (3, 1, 0), (7, 333, 3), (2, 512, 8), (9, 1000, 72),
                                     (4, 2056, 0), (3, 4097, 1), (2, 8200, 0), (1, 16384, 8), (130, 64, 1), (3, 16001, 3), (2, 9001, 0)])
def test_block_norm(hip, t, n, pad, post, gate, f32):
    rng = np.random.default_rng(n + t)
    y, h = rows(rng, t, n, pad, False, 0.5), rows(rng, t, n, pad, f32, 4.0)
    w_pre = dev(R.bf16(rng.normal(size=n) * 0.2))
    w_post = dev(R.bf16(rng.normal(size=n) * 0.2)) if post else None
    g = {"none": None, "one": dev(R.bf16(rng.normal(size=n))), "rows": rows(rng, t, n, pad, False)}[gate]
    norm = hip.block_norm_weights(n, w_pre, w_post, g, scale=-0.7, eps=1e-5)
    out = rows(rng, t + 1, n, pad, f32)
    x = rows(rng, t + 1, n, pad, False)
    last = (val(out[t:]), val(x[t:]))
    h_in, y_in = h.clone(), y.clone()
    hip.block_norm(norm, y, h, out[:t], x[:t])
    check(norm, y, h, out[:t], x[:t], w_post, w_pre, g, -0.7, 1e-5)
    assert np.array_equal(val(out[t:]), last[0]) and np.array_equal(val(x[t:]), last[1])
    assert torch.equal(h, h_in) and torch.equal(y, y_in)
    # in place: h' over h, x over y
    want = out[:t].clone(), x[:t].clone()
    hip.block_norm(norm, y, h, h, y)
    torch.cuda.synchronize()
    assert torch.equal(h, want[0]) and torch.equal(y, want[1])


def test_parts(hip):
    """Without y (a model's first norm), without x (its last residual)."""
    rng = np.random.default_rng(2)
    y, h = rows(rng, 6, 640, 0, False), rows(rng, 6, 640, 0, False)
    w = dev(R.bf16(rng.normal(size=640) * 0.2))
    norm = hip.block_norm_weights(640, w_pre=w)
    x, out = torch.empty_like(y), torch.empty_like(h)
    hip.block_norm(norm, None, h, None, x)
    check(norm, None, h, None, x, None, w, None, 1.0, 1e-6)
    hip.block_norm(norm, None, h, out, x)
    assert torch.equal(out, h)
    norm = hip.block_norm_weights(640, scale=2.0)
    hip.block_norm(norm, y, h, out, None)
    check(norm, y, h, out, None, None, None, None, 2.0, 1e-6)
    hip.block_norm(norm, y[:0], h[:0], out[:0], None)


def test_rows_do_not_mix(hip):
    """A row of NaN or infinities, or of zeros, leaves the others as they are."""
    rng = np.random.default_rng(3)
    y, h = rows(rng, 9, 2048, 0, False), rows(rng, 9, 2048, 0, False)
    w = dev(R.bf16(rng.normal(size=2048) * 0.2))
    norm = hip.block_norm_weights(2048, w, w)
    a, b = torch.empty_like(h), torch.empty_like(y)
    hip.block_norm(norm, y, h, a, b)
    y2, h2 = y.clone(), h.clone()
    y2[4, 7], h2[6, 9] = 0x7fc0, 0x7f80
    y2[2], h2[2] = 0, 0
    c, d = torch.empty_like(h), torch.empty_like(y)
    hip.block_norm(norm, y2, h2, c, d)
    torch.cuda.synchronize()
    keep = [0, 1, 3, 5, 7, 8]
    assert torch.equal(a[keep], c[keep]) and torch.equal(b[keep], d[keep])
    assert np.isnan(val(d[4:5])).all()
    assert (val(c[2:3]) == 0).all() and (val(d[2:3]) == 0).all()
    assert np.isinf(val(c[6:7])[0, 9]) and np.isnan(val(d[6:7])[0, 9])


def test_matches_attn_rmsnorm(hip):
    """x without a block is the tier-1 op's norm, to its one rounding."""
    rng = np.random.default_rng(4)
    n = 2048
    h, w = R.bf16(rng.normal(size=n)), R.bf16(rng.normal(size=n) * 0.2)
    norm = hip.block_norm_weights(n, w_pre=dev(w))
    x = torch.empty(1, n, dtype=torch.int16, device="cuda")
    hip.block_norm(norm, None, dev(h)[None], None, x)
    a, b = R.f64(x.cpu().numpy().view(np.uint16)[0]), R.f64(hip.attn_rmsnorm(h, w))
    assert (np.abs(a - b) <= 2.0 ** -7 * np.abs(b)).all() and np.mean(a != b) < 0.01


def test_graph_and_strides(hip):
    """A captured call, replayed between eager work on a stream of its own; rows
    that lie on top of each other are refused."""
    rng = np.random.default_rng(3)
    T, n = 5, 2048
    y, h, gate = rows(rng, T, n, 0, False), rows(rng, T, n, 0, True), rows(rng, T, n, 0, False)
    w = [dev(R.bf16(rng.normal(size=n) * 0.1)) for _ in range(2)]
    norm = hip.block_norm_weights(n, w_pre=w[0], w_post=w[1], gate=gate, scale=0.7)
    ho, x = torch.empty_like(h), torch.empty_like(y)
    hip.block_norm(norm, y, h, ho, x)
    torch.cuda.synchronize()
    want = ho.clone(), x.clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    hip.set_stream(st.cuda_stream)
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            hip.block_norm(norm, y, h, ho, x)
        for i in range(3):
            ho.zero_()
            x.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(ho, want[0]) and torch.equal(x, want[1]), i
            torch.randn(1000, device="cuda").sum().item()
    finally:
        hip.set_stream(0)
    for a in (dict(h=h[:1].expand(T, n)), dict(y=y[:1].expand(T, n)), dict(h_out=ho[:1].expand(T, n)),
              dict(x=x[:1].expand(T, n))):
        with pytest.raises(hip.ApusHipError, match="pitch"):
            hip.block_norm(norm, **dict(dict(y=y, h=h, h_out=ho, x=x), **a))
    with pytest.raises(ValueError, match="gate"):
        hip.block_norm_weights(n, w_pre=w[0], gate=gate[:1].expand(T, n))
    for a in (dict(h=h[:4]), dict(y=y.float()), dict(h_out=ho.to(torch.bfloat16)), dict(x=x.cpu()), dict(x=x[:, :-8])):
        with pytest.raises(ValueError):
            hip.block_norm(norm, **dict(dict(y=y, h=h, h_out=ho, x=x), **a))
    torch.cuda.synchronize()
    assert torch.equal(ho, want[0]) and torch.equal(x, want[1])
