"""The 8-bit KV cache, attention over it, and the norms around a block: the calls
a program makes of them, as cases that can be timed and compared.

  store    new tokens' k and v rows written into the 8-bit cache (e4m3 codes,
           one power-of-two scale for each 32 positions and kv head), and the
           blocks they touch read back
  decode   gated GQA attention of 1 to 4 new tokens a sequence over the cache:
           q norm, RoPE, causal softmax, output gate
  prefill  the same for any number of new tokens
  norm     h' = h + scale gate post(y), x = pre(h'): the residual and the two
           RMSNorms around a block

With `own` false, `run` computes them from elementary torch operations in 32
bits; with `own` true, through the library's Python binding.
"""
import math
import os
import random
import sys

import torch

own = False

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
BLK = 32                                   # positions of a cache block
D, ROT, GRP, THETA = 256, 64, 8, 1e7       # head size, rotary dims, q heads per kv head
EPS = 1e-6
HID = 2048                                 # the model's hidden size
EMIN = -117                                # smallest exponent of a block's scale


# ------------------------------------------------------------------ cases
# batch sequences with up to `new` new tokens after up to `ctx` cached ones;
# ragged: 0, or the seed of lengths that differ
def listed():
    return [
        # one user's chat step: one token's rows, in the middle of a block
        dict(name="store_1", kind="store", batch=1, new=1, ctx=1500, ragged=0, nkv=2, paged=False, pad=0),
        # a serving batch's verify step, rows as slices of the projections' output
        dict(name="store_128_verify", kind="store", batch=128, new=4, ctx=4000, ragged=3, nkv=2,
             paged=True, pad=64),
        # a long prompt filling its cache
        dict(name="store_8192", kind="store", batch=1, new=8192, ctx=0, ragged=0, nkv=2, paged=False, pad=0),
        # one user's chat step
        dict(name="decode_1", kind="decode", batch=1, new=1, ctx=1500, ragged=0, nkv=2, paged=False),
        # one user far into a long document, verifying three tokens
        dict(name="decode_1_long", kind="decode", batch=1, new=3, ctx=60001, ragged=0, nkv=2, paged=True),
        # a serving batch at long contexts
        dict(name="decode_64_long", kind="decode", batch=64, new=1, ctx=32767, ragged=0, nkv=2, paged=False),
        # 128 sequences of very different contexts verifying 1 to 4 tokens
        dict(name="decode_128_verify", kind="decode", batch=128, new=4, ctx=24000, ragged=5, nkv=2, paged=True),
        # a long prompt
        dict(name="prefill_8192", kind="prefill", batch=1, new=8192, ctx=0, ragged=0, nkv=2, paged=False),
        # a few users' turns after different histories in one batch
        dict(name="prefill_ragged", kind="prefill", batch=6, new=900, ctx=2500, ragged=9, nkv=2, paged=True),
        # one token between attention and experts: latency
        dict(name="norm_1", kind="norm", rows=1, hidden=HID, post=False, gate="none", f32=False, pad=0),
        # a verify step of 128 sequences, post-norm and a learned scale per channel
        dict(name="norm_325", kind="norm", rows=325, hidden=HID, post=True, gate="one", f32=False, pad=0),
        # a long prompt, residual stream in fp32, a gate per token and channel
        dict(name="norm_8192", kind="norm", rows=8192, hidden=HID, post=True, gate="rows", f32=True, pad=64),
    ]


def _logu(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("store", "decode", "decode", "prefill", "norm"))
    if kind == "norm":
        hidden = 8 * _logu(rng, 8, 512) + rng.choice((0, 0, 0, rng.randint(1, 7)))
        return dict(kind=kind, rows=_logu(rng, 1, 4000), hidden=hidden, post=rng.random() < 0.5,
                    gate=rng.choice(("none", "one", "rows")), f32=rng.random() < 0.4, pad=rng.choice((0, 8, 72)))
    c = dict(kind=kind, ragged=rng.randint(1, 999), nkv=rng.choice((1, 2, 2, 4)), paged=rng.random() < 0.5)
    if kind == "store":
        c["batch"] = _logu(rng, 1, 128)
        c.update(new=_logu(rng, 1, 8192 // c["batch"]), ctx=rng.randint(0, 3000), pad=rng.choice((0, 8, 72)))
    elif kind == "decode":
        c["batch"] = _logu(rng, 1, 128)
        c.update(new=rng.randint(1, 4), ctx=_logu(rng, 1, min(60000, 1000000 // c["batch"])))
    else:
        c["batch"] = _logu(rng, 1, 8)
        c.update(new=_logu(rng, 1, 4000 // c["batch"]), ctx=rng.randint(0, 4000))
    return c


def _lens(case):
    """(new tokens, cached tokens) of each sequence."""
    b, new, ctx = case["batch"], case["new"], case["ctx"]
    if not case["ragged"]:
        return [new] * b, [ctx] * b
    r = random.Random(case["ragged"])
    n = [r.randint(1, new) for _ in range(b)]
    # contexts spread over their logarithm, as chats' are
    p = [min(ctx, int(ctx * math.exp(-abs(r.gauss(0.0, 1.3))))) for _ in range(b)]
    return n, p


def work(case):
    if case["kind"] == "norm":
        n, hb = case["rows"] * case["hidden"], 4 if case["f32"] else 2
        return {"bytes": n * (2 + 2 * hb + 2 + (2 if case["gate"] == "rows" else 0)), "flops": 10 * n}
    new, pos = _lens(case)
    t, nkv = sum(new), case["nkv"]
    if case["kind"] == "store":            # rows in, codes out; the touched blocks' codes in, rows out
        back = sum(n + p % BLK for n, p in zip(new, pos))
        return {"bytes": 2 * nkv * D * (3 * t + 3 * back), "flops": 4 * nkv * D * t}
    keys = sum(n + p for n, p in zip(new, pos))
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, pos))
    return {"bytes": 2 * nkv * D * keys + t * nkv * GRP * D * 6, "flops": 4 * nkv * GRP * D * pairs}


# ------------------------------------------------------------------ inputs
def _binding():
    pkg = os.path.join(os.getcwd(), "apus-qwen3.6-35b-a3b_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import apus_hip
    apus_hip.init(0)
    return apus_hip


def _cum(n):
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=BF):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    d = {}
    if case["kind"] == "norm":
        t, h, pad = case["rows"], case["hidden"], case["pad"]

        def rows(scale=1.0, dtype=BF):
            w = normal(t, h + pad, scale=scale, dtype=dtype)
            return w[:, pad:] if pad else w
        d["y"], d["h"] = rows(0.7), rows(3.0, torch.float32 if case["f32"] else BF)
        d["w_pre"] = normal(h, scale=0.1)
        d["w_post"] = normal(h, scale=0.1) if case["post"] else None
        d["gate"] = {"none": None, "one": normal(h), "rows": rows()}[case["gate"]]
        return d
    new, pos = _lens(case)
    nkv, store = case["nkv"], case["kind"] == "store"

    def kv(n, pad):                        # tokens and channels of different magnitudes
        w = torch.randn(n, nkv * D + pad, generator=g, device="cuda")
        w *= torch.exp2(torch.randint(-1, 2, (n, 1), generator=g, device="cuda").float())
        w[:, pad:pad + 7] *= 3.0
        w = w.to(BF)
        return w[:, pad:] if pad else w
    # what the cache holds before the call, one sequence's tokens after the other's
    old = pos if store else [p + n for p, n in zip(pos, new)]
    d["old"] = old
    d["k_old"], d["v_old"] = kv(sum(old), 0), kv(sum(old), 0)
    if store:
        d["k"], d["v"] = kv(sum(new), case["pad"]), kv(sum(new), case["pad"])
    else:
        d["qg"] = normal(sum(new), nkv * GRP, 2 * D)
        d["qn_w"], d["kn_w"] = normal(D, scale=0.1), normal(D, scale=0.1)
    # the block table: the blocks of a sequence one after the other, or scattered
    nb = [(p + n + BLK - 1) // BLK for p, n in zip(pos, new)]
    most = max(nb)
    if case["paged"]:
        ids = torch.randperm(sum(nb) + 3, generator=g, device="cuda").to(torch.int32)
        at = torch.tensor(_cum(nb), device="cuda")[:-1, None] + torch.arange(most, device="cuda")
        d["table"] = torch.where(torch.arange(most, device="cuda") < torch.tensor(nb, device="cuda")[:, None],
                                 ids[at.clamp_max(sum(nb) - 1)], 0).to(torch.int32)
        d["blocks"] = sum(nb) + 3
    else:
        d["table"] = torch.arange(case["batch"] * most, device="cuda", dtype=torch.int32).view(-1, most)
        d["blocks"] = case["batch"] * most
    return d


def _tokens(lens, first):
    """(sequence, position) of each token of sequences with lens tokens from position first."""
    n = torch.tensor(lens, device="cuda")
    s = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), n)
    at = torch.arange(sum(lens), device="cuda") - torch.tensor(_cum(lens), device="cuda")[s]
    return s, at + torch.tensor(first, device="cuda")[s]


def prepare(case, seed):
    d = _inputs(case, seed)
    st = dict(case=case, d=d)
    if case["kind"] == "norm":
        st["h2"], st["x"] = torch.empty_like(d["h"]), torch.empty_like(d["y"])
        if own:
            hip = st["hip"] = _binding()
            st["norm"] = hip.block_norm_weights(case["hidden"], w_pre=d["w_pre"], w_post=d["w_post"],
                                                gate=d["gate"], scale=0.5, eps=EPS)
        return st
    new, pos = _lens(case)
    nkv, store = case["nkv"], case["kind"] == "store"
    zero = [0] * case["batch"]
    back = [p // BLK * BLK for p in pos]                   # from the first touched block on
    nback = [n + p - b for n, p, b in zip(new, pos, back)]
    if store:
        st["k"] = torch.empty(sum(nback), nkv * D, dtype=BF, device="cuda")
        st["v"] = torch.empty_like(st["k"])
    else:
        st["y"] = torch.empty(sum(new), nkv * GRP * D, dtype=BF, device="cuda")
    if own:
        hip = st["hip"] = _binding()
        kv = st["kv"] = hip.kv8_cache(nkv, d["blocks"], d["table"].shape[1],
                                      block_table=d["table"] if case["paged"] else None)
        rows = list(range(case["batch"])) if case["paged"] else None
        hip.kv8_append(kv, rows, _cum(d["old"]), zero, d["k_old"], d["v_old"])
        if store:
            st["calls"] = (hip.kv8_append_bound(kv, rows, _cum(new), pos, d["k"], d["v"]),
                           hip.kv8_read_bound(kv, rows, _cum(nback), back, st["k"], st["v"]))
        else:
            layer = hip.attn_layer((nkv * GRP, nkv, D, ROT, THETA), dict(qn_w=d["qn_w"], kn_w=d["kn_w"]))
            work = st["work"] = hip.AttnKv8Work(layer, case["batch"], max(p + n for p, n in zip(pos, new)))
            call = hip.attn_decode_kv8_bound if case["kind"] == "decode" else hip.attn_prefill_kv8_bound
            st["calls"] = (call(layer, work, rows, _cum(new), pos, d["qg"], None, None, kv, st["y"]),)
    else:
        st["cache"] = [_empty(d, nkv), _empty(d, nkv)]
        st["new"], st["pos"] = _tokens(new, pos), torch.tensor(pos, device="cuda")
        st["back"], st["cum"] = _tokens(nback, back), torch.tensor(_cum(new), device="cuda")
        st["most"] = max(new)
        st["inv"] = torch.tensor([THETA ** (-2.0 * i / ROT) for i in range(ROT // 2)], device="cuda")
        # the blocks that hold tokens already
        st["kept"] = torch.tensor([s for s, p in enumerate(pos) if p % BLK], dtype=torch.long, device="cuda")
        st["kept"] = d["table"][st["kept"], st["pos"][st["kept"]] // BLK].long()
        for c, x in zip(st["cache"], (d["k_old"], d["v_old"])):
            _write(c, d["table"], _tokens(d["old"], zero), None, x)
    for n in ("k_old", "v_old"):           # the cache holds them now
        del d[n]
    return st


# ------------------------------------------------------------------- run
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    if st["case"]["kind"] == "norm":
        d = st["d"]
        st["hip"].block_norm(st["norm"], d["y"], d["h"], st["h2"], st["x"])
        return st["h2"], st["x"]
    for call in st["calls"]:
        call()
    return (st["k"], st["v"]) if "k" in st else st["y"]


def _run_plain(st):
    kind, d = st["case"]["kind"], st["d"]
    if kind == "norm":
        return _norm_plain(d)
    if kind == "store":
        out = []
        for c, x in zip(st["cache"], (d["k"], d["v"])):
            _write(c, d["table"], st["new"], st["kept"], x)
            out.append(_read(c, d["table"], st["back"]))
        return tuple(out)
    return _attention(st)


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + w.float())


def _norm_plain(d):
    y = d["y"].float()
    if d["w_post"] is not None:
        y = _rms(y, d["w_post"])
    if d["gate"] is not None:
        y = y * d["gate"].float()
    h = d["h"].float() + 0.5 * y
    return h.to(d["h"].dtype), _rms(h, d["w_pre"]).to(BF)


# The cache in the plain form: e4m3 codes [blocks][nkv][32][256] as bytes and
# the exponents of the scales [blocks][nkv].
def _empty(d, nkv):
    return (torch.zeros(d["blocks"], nkv, BLK, D, dtype=torch.uint8, device="cuda"),
            torch.zeros(d["blocks"], nkv, dtype=torch.int32, device="cuda"))


def _codes(x, e):
    return torch.ldexp(x, -e).to(F8).view(torch.uint8)


def _values(codes, e):
    return torch.ldexp(codes.view(F8).float(), e)


def _exponent(amax):
    """The smallest e with amax <= 448 2^e, at least EMIN."""
    m, e = torch.frexp(amax)               # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(amax > 0, e.clamp_min(EMIN), torch.full_like(e, EMIN)).to(torch.int32)


def _write(cache, table, at, kept, x):
    codes, exps = cache
    s, p = at
    nkv = codes.shape[1]
    if not s.numel():
        return
    x = x.unflatten(-1, (nkv, D)).float()
    blk = table[s, p // BLK].long()
    amax = torch.zeros(exps.shape, device=x.device)
    amax.scatter_reduce_(0, blk[:, None].expand(-1, nkv), x.abs().amax(-1), "amax", include_self=True)
    e = _exponent(amax)
    if kept is not None:                   # blocks that hold tokens keep them: their scale only grows
        e[kept] = torch.maximum(e[kept], exps[kept])
        codes[kept] = _codes(_values(codes[kept], exps[kept][..., None, None]), e[kept][..., None, None])
    exps[blk] = e[blk]
    codes[blk, :, p % BLK] = _codes(x, e[blk][..., None])


def _read(cache, table, at):
    codes, exps = cache
    s, p = at
    blk = table[s, p // BLK].long()
    return _values(codes[blk, :, p % BLK], exps[blk][..., None]).flatten(1).to(BF)


def _rope(x, pos, inv):
    """Rotary embedding of the first ROT of x [..., D]; cos and sin are bf16 as the model keeps them."""
    a = (pos.float()[:, None] * inv).double()
    c, s = torch.cos(a).float().to(BF).float()[:, None], torch.sin(a).float().to(BF).float()[:, None]
    u, v = x[..., :ROT // 2], x[..., ROT // 2:ROT]
    return torch.cat((u * c - v * s, v * c + u * s, x[..., ROT:]), -1)


def _attention(st):
    d, nkv = st["d"], st["case"]["nkv"]
    s, p = st["new"]
    q, gate = d["qg"].float().split(D, -1)
    q = _rope(_rms(q, d["qn_w"]), p, st["inv"]) / math.sqrt(D)
    # sequences side by side, padded to the longest
    b, n = st["pos"].numel(), st["most"]
    t = torch.arange(s.numel(), device=s.device) - st["cum"][s]
    wide = torch.zeros(b, n, nkv, GRP, D, device=q.device)
    wide[s, t] = q.unflatten(1, (nkv, GRP))
    wide = wide.permute(0, 2, 3, 1, 4).reshape(b * nkv, GRP * n, D)

    def values(cache, perm):
        at = d["table"].long()
        x = _values(cache[0][at], cache[1][at][..., None, None])
        return x.permute(0, 2, *perm)      # [b][nkv] and keys x D, or D x keys
    k = values(st["cache"][0], (4, 1, 3)).reshape(b * nkv, D, -1)
    a = (wide @ k).view(b, nkv, GRP, n, -1)
    key = torch.arange(a.shape[-1], device=a.device)
    own_at = st["pos"][:, None] + torch.arange(n, device=a.device)
    seen = key <= own_at[..., None]
    a = a.masked_fill_(~seen[:, None, None], -math.inf)
    a = torch.exp_(a - a.amax(-1, keepdim=True))
    a = a / a.sum(-1, keepdim=True)
    v = values(st["cache"][1], (1, 3, 4)).reshape(b * nkv, -1, D)
    v = v.masked_fill((key > (st["pos"].repeat_interleave(nkv)[:, None] + n))[..., None], 0.0)
    o = (a.view(b * nkv, GRP * n, -1) @ v).view(b, nkv, GRP, n, D)
    o = o.permute(0, 3, 1, 2, 4)[s, t].flatten(1, 2)
    return (o / (1.0 + torch.exp(-gate))).flatten(1).to(BF)


# ----------------------------------------------------------------- exact
def _exact_codes(x, e=None):
    """x [tokens][nkv][D] of one block in 64 bits to e4m3 values and the
    exponent: the definition, from the list of e4m3's magnitudes."""
    mags = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8.0) * 2.0 ** (n - 7) for n in range(1, 16) for m in range(8)][:-1]
    grid = torch.tensor(mags, dtype=torch.float64, device=x.device)
    if e is None:
        amax = x.abs().amax((0, 2))
        e = torch.ceil(torch.log2((amax / 448.0).clamp_min(2.0 ** EMIN)))
        e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
    v = x / torch.exp2(e)[:, None]
    mid = (grid[1:] + grid[:-1]) / 2
    lo = torch.bucketize(v.abs(), mid)                     # mid[lo - 1] < |v| <= mid[lo]
    tie = (lo < mid.numel()) & (v.abs() == mid[lo.clamp_max(mid.numel() - 1)])
    lo = torch.where(tie & (lo % 2 == 1), lo + 1, lo)      # a tie goes to the even code
    return torch.sign(v) * grid[lo], e


def _exact_cache(x, nkv):
    """The values that one sequence's cache stands for, all tokens written at once."""
    n = x.shape[0]
    x = torch.nn.functional.pad(x.double(), (0, 0, 0, -n % BLK)).view(-1, BLK, nkv, D)
    # blocks as heads of their own: a scale for each
    x = x.permute(1, 0, 2, 3).reshape(BLK, -1, D)
    v, e = _exact_codes(x)
    v = v * torch.exp2(e)[:, None]
    return v.view(BLK, -1, nkv, D).permute(1, 0, 2, 3).reshape(-1, nkv, D)[:n]


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "norm":
        y, h = d["y"].double(), d["h"].double()

        def rms(v, w):
            return v / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + EPS) * (w.double() + 1.0)
        if d["w_post"] is not None:
            y = rms(y, d["w_post"])
        h = h + (y * d["gate"].double() if d["gate"] is not None else y) / 2
        return h, rms(h, d["w_pre"])
    new, pos = _lens(case)
    nkv, cu, cold = case["nkv"], _cum(new), _cum(d["old"])
    outs = []
    if case["kind"] == "store":
        for old, x in ((d["k_old"], d["k"]), (d["v_old"], d["v"])):
            parts = []
            for s, (n, p) in enumerate(zip(new, pos)):
                b = p // BLK * BLK
                kept = old[cold[s] + b:cold[s + 1]].double().view(-1, nkv, D)
                rows = x[cu[s]:cu[s + 1]].double().reshape(-1, nkv, D)
                first = rows[:BLK - (p - b)]               # those that go into the kept tokens' block
                if p > b:
                    kv, ke = _exact_codes(kept)
                    e = torch.maximum(ke, _exact_codes(first)[1])
                    kv = _exact_codes(kv * torch.exp2(ke)[:, None], e)[0]
                    parts.append((torch.cat((kv, _exact_codes(first, e)[0])) * torch.exp2(e)[:, None]).flatten(1))
                    rows = rows[first.shape[0]:]
                if rows.shape[0]:
                    parts.append(_exact_cache(rows.reshape(-1, nkv * D), nkv).flatten(1))
            outs.append(torch.cat(parts))
        return tuple(outs)
    inv = torch.tensor([THETA ** (-2.0 * i / ROT) for i in range(ROT // 2)], device="cuda")
    for s, (n, p) in enumerate(zip(new, pos)):
        k = _exact_cache(d["k_old"][cold[s]:cold[s + 1]], nkv)
        v = _exact_cache(d["v_old"][cold[s]:cold[s + 1]], nkv)
        qg = d["qg"][cu[s]:cu[s + 1]].double()
        q = qg[..., :D]
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) / D + EPS) * (d["qn_w"].double() + 1.0)
        at = torch.arange(p, p + n, device="cuda")
        # the model's cos and sin: of the 32-bit angle, kept in bf16
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (at.float()[:, None] * inv).double())
        c, r = z.real.to(BF).double()[:, None], z.imag.to(BF).double()[:, None]
        q1, q2 = q[..., :ROT // 2].clone(), q[..., ROT // 2:ROT].clone()
        q[..., :ROT // 2], q[..., ROT // 2:ROT] = q1 * c - q2 * r, q2 * c + q1 * r
        o = torch.empty_like(q)
        for h in range(nkv):
            a = torch.matmul(q[:, h * GRP:(h + 1) * GRP], k[:, h].t()) / 16.0
            a = a.masked_fill(torch.arange(p + n, device="cuda") > at[:, None, None], -math.inf)
            o[:, h * GRP:(h + 1) * GRP] = torch.matmul(torch.softmax(a, -1), v[:, h])
        outs.append((o * torch.sigmoid(qg[..., D:])).flatten(1))
    return torch.cat(outs)
