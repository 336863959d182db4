"""Prompts and decode steps as a program makes them of the library's calls: an
attention layer on an 8-bit cache in a pool, the norms around each block fused
with the fp32 residual, the mixture-of-experts layer. What each call returns is
held against 64-bit arithmetic on that call's own inputs; a captured step,
replayed, and the same steps on a stream of their own give the same bits."""
import numpy as np
import pytest
import torch

import kv8_ref as R
import mx_ref
import synth

pytestmark = pytest.mark.gpu

H, I, E, K, IS = 2048, 256, 24, 4, 128
NH, NKV, D, ROT, THETA = synth.ATTN_DIMS
PROMPTS, MAX = [45, 1, 96, 31], 5


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16) if a.dtype == np.uint16 else np.ascontiguousarray(a)).cuda()


def host(t):
    return t.view(torch.int16).cpu().numpy().view(np.uint16)


def empty(*s):
    return torch.empty(s, dtype=torch.int16, device="cuda")


class Model:
    def __init__(self, hip, seed):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        s = H ** -0.5
        self.hip, self.rng = hip, rng
        self.aw = synth.attn_weights(rng)
        self.pw = dict(wq=synth.normal_bf16(rng, (NH * 2 * D, H), s), wk=synth.normal_bf16(rng, (NKV * D, H), s),
                       wv=synth.normal_bf16(rng, (NKV * D, H), s),
                       wo=synth.normal_bf16(rng, (H, NH * D), (NH * D) ** -0.5))
        self.layer = hip.attn_layer(synth.ATTN_DIMS, {n: dev(v) for n, v in self.aw.items()})
        self.proj = hip.attn_proj(H, {n: dev(v) for n, v in self.pw.items()})
        self.mw = mx_ref.moe_weights(g, H, I, E, IS)
        for n in [n for n in self.mw if n.endswith(("gate_up", "down"))]:
            w = self.mw[n].reshape(-1, self.mw[n].shape[-1])
            c = torch.empty(w.shape[0], w.shape[1] // 2, dtype=torch.uint8, device="cuda")
            sc = torch.empty(w.shape[0], w.shape[1] // 32, dtype=torch.uint8, device="cuda")
            hip.mxfp4_quantize(w, c, sc)
            lead = self.mw[n].shape[:-1]
            self.mw[n], self.mw["s" + n[1:]] = c.view(*lead, -1), sc.view(*lead, -1)
        self.moe = hip.moe_layer((H, I, E, K, IS), self.mw)
        self.norms = [R.bf16(rng.normal(size=H) * 0.1) for _ in range(4)]
        w = [dev(a) for a in self.norms]
        self.first = hip.block_norm_weights(H, w_pre=w[0])
        self.mid = hip.block_norm_weights(H, w_pre=w[1], w_post=w[2], scale=0.5)
        self.last = hip.block_norm_weights(H, w_pre=w[0], w_post=w[3])
        B = len(PROMPTS)
        self.pool = hip.KvPool(1, NKV, D, B * MAX + 2, B, MAX, kv8=True)
        self.rows = [self.pool.open() for _ in range(B)]
        for r in self.rows:
            self.pool.reserve(r, MAX * 32)
        self.kv = self.pool.cache(0)
        self.work = hip.AttnKv8Work(self.layer, B, MAX * 32)
        self.mwork = hip.MoeWork(self.moe, 4 * B)

    def prompt(self, x):
        """h (fp32) and the next block's input after the attention of a prompt."""
        hip, T = self.hip, len(x)
        cu = np.concatenate(([0], np.cumsum(PROMPTS))).astype(np.int32)
        ln, ln2, ao, y = (empty(T, n) for n in (H, H, H, NH * D))
        qg, k, v = empty(T, NH * 2 * D), empty(T, NKV * D), empty(T, NKV * D)
        h = torch.empty_like(x)
        hip.block_norm(self.first, None, x, None, ln)
        for n, o in (("wq", qg), ("wk", k), ("wv", v)):
            hip.bf16_gemm_dev(self.proj._tensors[n], ln, o, exact=False)
        hip.attn_prefill_kv8(self.layer, self.work, self.rows, cu, [0] * len(PROMPTS), qg, k, v, self.kv, y)
        hip.bf16_gemm_dev(self.proj._tensors["wo"], y, ao, exact=False)
        hip.block_norm(self.mid, ao, x, h, ln2)
        return ln, qg, k, v, y, ao, h, ln2

    def step(self, cu, pos, x, out):
        """A decode step; out: its buffers."""
        hip = self.hip
        hip.block_norm(self.first, None, x, None, out["ln"])
        hip.attn_layer_decode_kv8(self.layer, self.proj, self.work, self.rows, cu, pos, out["ln"], self.kv, out["ao"])
        hip.block_norm(self.mid, out["ao"], x, out["h"], out["ln2"])
        hip.moe_layer_decode(self.moe, self.mwork, out["ln2"], out["y"])
        hip.block_norm(self.last, out["y"], out["h"], out["h2"], out["x"])

    def buffers(self, T):
        o = {n: empty(T, H) for n in ("ln", "ao", "ln2", "y", "x")}
        o["h"], o["h2"] = (torch.empty(T, H, device="cuda") for _ in range(2))
        return o


def rel(got, want, bound):
    """Largest error of bf16 codes or fp32 values in parts of a bound a row."""
    g = got.cpu().double().numpy() if got.dtype == torch.float32 else R.f64(host(got))
    return (np.abs(g - want) / bound).max()


def norm_close(model, norm, post, pre, scale, y, x, h, out):
    """block_norm on its own inputs: n / 2 + 8 roundings of fp32 and that of the result."""
    f = (H / 2 + 8) * 2.0 ** -24
    rms = lambda v, w: v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * (1.0 + R.f64(w))       # noqa: E731
    x64 = x.cpu().double().numpy()
    t = 0.0 if y is None else scale * rms(R.f64(host(y)), model.norms[post])
    h2, mag = x64 + t, np.abs(x64) + np.abs(t)
    if h is not None:
        assert rel(h, h2, f * mag + 2.0 ** -24 * np.abs(h2) + 1e-30) <= 1
    want = rms(h2, model.norms[pre])
    spread = f * mag.max(-1, keepdims=True) / np.sqrt((h2 * h2).mean(-1, keepdims=True)) * 2 * (1.0 + np.abs(R.f64(model.norms[pre])))
    assert rel(out, want, R.U * np.abs(want) + spread + f * np.abs(want)) <= 1


def test_steps(hip):
    m = Model(hip, 5)
    B, T0 = len(PROMPTS), sum(PROMPTS)
    x0 = torch.randn(T0, H, device="cuda")
    ln, qg, k, v, y, ao, h, ln2 = m.prompt(x0)
    torch.cuda.synchronize()
    norm_close(m, m.first, None, 0, 1.0, None, x0, None, ln)
    norm_close(m, m.mid, 2, 1, 0.5, ao, x0, h, ln2)
    # the cache: what the bf16 mixer would append, quantised
    cu = np.concatenate(([0], np.cumsum(PROMPTS))).astype(np.int32)
    ref = R.Cache(NKV, B, MAX)

    def mixer_rows(cu, pos, n, qg, k, v):
        """The rows k (normed, roped) and v of new tokens, from the bf16 mixer."""
        ms = MAX * 32
        kc, vc = (torch.zeros(B * ms * NKV * D, dtype=torch.int16, device="cuda") for _ in range(2))
        hip.attn_prefill(m.layer, cu, pos, qg, k, v, kc, vc, ms, empty(int(cu[-1]), NH * D))
        for s in range(B):
            a, b = empty(pos[s] + n[s], NKV * D), empty(pos[s] + n[s], NKV * D)
            if n[s]:
                hip.attn_cache_unpack(kc[s * ms * NKV * D:], vc[s * ms * NKV * D:], pos[s] + n[s], NKV, D, ms, a, b)
                ref.append(m.rows[s], pos[s], host(a)[pos[s]:], host(b)[pos[s]:])

    def attention_close(cu, pos, n, qg, y):
        for s in range(B):
            if not n[s]:
                continue
            kk, vv = ref.values(m.rows[s], 0, pos[s] + n[s])
            sl = slice(cu[s], cu[s + 1])
            r, tol = R.attention(host(qg)[sl].reshape(-1, NH, 2 * D), m.aw["qn_w"], pos[s], kk, vv, THETA)
            assert (np.abs(R.f64(host(y)[sl]).reshape(r.shape) - r) <= tol).all(), (s, pos[s], n[s])

    mixer_rows(cu, [0] * B, PROMPTS, qg, k, v)
    attention_close(cu, [0] * B, PROMPTS, qg, y)
    # steps of several tokens, one, and none
    pos = np.array(PROMPTS, np.int32)
    for n in ([1, 1, 1, 1], [1, 4, 0, 2], [2, 0, 1, 1], [1, 1, 1, 1]):
        cu = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        T = int(cu[-1])
        x, out = torch.randn(T, H, device="cuda"), m.buffers(T)
        m.step(cu, pos, x, out)
        torch.cuda.synchronize()
        # the layer's products and mixer, call by call, give the same bits
        P = m.proj._tensors
        qg, k, v, y, ao = empty(T, NH * 2 * D), empty(T, NKV * D), empty(T, NKV * D), empty(T, NH * D), empty(T, H)
        for w, o in (("wq", qg), ("wk", k), ("wv", v)):
            hip.bf16_gemm_dev(P[w], out["ln"], o, exact=False)
        hip.attn_decode_kv8(m.layer, m.work, m.rows, cu, pos, qg, None, None, m.kv, y)
        hip.bf16_gemm_dev(P["wo"], y, ao, exact=False)
        assert torch.equal(ao, out["ao"])
        hip.attn_decode_kv8(m.layer, m.work, m.rows, cu, pos, qg, k, v, m.kv, y)
        hip.bf16_gemm_dev(P["wo"], y, ao, exact=False)
        assert torch.equal(ao, out["ao"])
        mixer_rows(cu, pos, n, qg, k, v)
        attention_close(cu, pos, n, qg, y)
        norm_close(m, m.first, None, 0, 1.0, None, x, None, out["ln"])
        norm_close(m, m.mid, 2, 1, 0.5, out["ao"], x, out["h"], out["ln2"])
        norm_close(m, m.last, 3, 0, 1.0, out["y"], out["h"], out["h2"], out["x"])
        r, b, gap = mx_ref.moe(out["ln2"].view(torch.bfloat16), m.mw, K, True, True)
        ok = gap > 1e-4
        mx_ref.check(out["y"].view(torch.bfloat16)[ok], r[ok], b[ok], "moe")
        # captured and replayed on a stream of its own: the same bits each time
        want = {q: t.clone() for q, t in out.items()}
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        hip.set_stream(st.cuda_stream)
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                m.step(cu, pos, x, out)
            for i in range(3):
                for t in out.values():
                    t.zero_()
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                for q, t in out.items():
                    assert torch.equal(t, want[q]), (i, q)
                torch.randn(1000, device="cuda").sum().item()
            with torch.cuda.stream(st):
                for t in out.values():
                    t.zero_()
                m.step(cu, pos, x, out)
            torch.cuda.synchronize()
            for q, t in out.items():
                assert torch.equal(t, want[q]), q
        finally:
            hip.set_stream(0)
        pos = pos + np.array(n, np.int32)
    m.work.destroy()
    m.mwork.destroy()
    m.pool.destroy()


def test_layer_refusals(hip):
    m = Model(hip, 6)
    cu, pos = np.arange(5, dtype=np.int32), np.zeros(4, np.int32)
    ln, ao = empty(4, H).zero_(), empty(4, H)
    call = lambda rows=m.rows, cu=cu, pos=pos, work=m.work: hip.attn_layer_decode_kv8(                # noqa: E731
        m.layer, m.proj, work, rows, cu, pos, ln, m.kv, ao)
    before = [t.clone() for t in (ln, ao)]
    with pytest.raises(hip.ApusHipError, match="one row"):
        call(rows=[0, 1, 1, 2])
    with pytest.raises(hip.ApusHipError, match="overflows|reserved|position"):
        call(pos=np.array([0, 0, 0, MAX * 32], np.int32))
    with pytest.raises(hip.ApusHipError, match="rows"):
        call(rows=[0, 1, 2, 9])
    small = hip.AttnKv8Work(m.layer, 3, 64)
    with pytest.raises(hip.ApusHipError, match="holds 3"):
        call(work=small)
    small.destroy()
    with pytest.raises(hip.ApusHipError, match="workspace"):
        call(work=small)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((ln, ao), before))
    for w in (m.work, m.mwork, m.pool):
        w.destroy()
