"""The 8-bit KV cache on the GPU: codes and scales against the definition, bit
for bit, and attention over it against 64-bit arithmetic on the cache's values."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu
THETA = 1e7


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16) if a.dtype == np.uint16 else np.ascontiguousarray(a)).cuda()


def host(t):
    return t.cpu().numpy().view(np.uint16)


def cum(n):
    return np.concatenate(([0], np.cumsum(n))).astype(np.int32)


def table(rng, rows, max_blocks, spare=3):
    """Scattered blocks, and entries past every use that name no block."""
    ids = rng.permutation(rows * max_blocks + spare)[:rows * max_blocks]
    return torch.from_numpy(ids.reshape(rows, max_blocks).astype(np.int32)).cuda(), rows * max_blocks + spare


def make(hip, rng, nkv, rows, max_blocks, paged):
    if paged:
        t, blocks = table(rng, rows, max_blocks)
        kv = hip.kv8_cache(nkv, blocks, max_blocks, block_table=t)
    else:
        kv = hip.kv8_cache(nkv, rows * max_blocks, max_blocks)
    for x in kv._tensors[:2]:
        x.fill_(0x7f)                      # whatever lies in the cache before: NaN codes, NaN scales
    kv._tensors[2].fill_(float("nan"))
    return kv


def kv_rows(rng, n, nkv, spread=6.0):
    """k or v rows of very different magnitudes."""
    x = rng.normal(size=(n, nkv, R.D)) * 2.0 ** rng.uniform(-spread, spread, (n, 1, 1)) * 2.0 ** rng.uniform(-3, 3, (1, nkv, R.D))
    return R.bf16(x).reshape(n, nkv * R.D)


def read(hip, kv, row, p0, n, nkv):
    k = torch.empty(n, nkv * R.D, dtype=torch.int16, device="cuda")
    v = torch.empty_like(k)
    hip.kv8_read(kv, [row], [0, n], [p0], k, v)
    return host(k), host(v)


def same(a, b):
    """bf16 codes equal, any NaN equal to any NaN, -0 told from 0."""
    nan = lambda x: (x & 0x7fff) > 0x7f80                  # noqa: E731
    return np.array_equal(np.where(nan(a), 0x7fc0, a), np.where(nan(b), 0x7fc0, b))


def check_row(hip, kv, ref, row, p0, p1):
    k, v = read(hip, kv, row, p0, p1 - p0, ref.nkv)
    rk, rv = ref.values(row, p0, p1)
    assert same(k, R.bf16(rk).reshape(k.shape))
    assert same(v, R.bf16(rv).reshape(v.shape))


@pytest.mark.parametrize("top", [448.0, 1.0, 2.0 ** -100, 3e38, 2.0 ** -130])
def test_every_bf16_value(hip, top):
    """All finite bf16 values up to top, with top itself in every block, then
    infinities and NaN."""
    c = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    c = c[np.abs(np.nan_to_num(R.f64(c), nan=0.0, posinf=0.0, neginf=0.0)) <= top]
    t = R.bf16(np.array([top]))[0]
    per = 31 * R.D
    n = -(-len(c) // per)
    x = np.zeros(n * per, np.uint16)
    x[:len(c)] = c
    x = np.concatenate((x.reshape(n, 31, R.D), np.full((n, 1, R.D), t)), 1).reshape(n * 32, R.D)
    kv, ref = make(hip, None, 1, 1, n, False), R.Cache(1, 1, n)
    hip.kv8_append(kv, None, [0, n * 32], [0], dev(x), dev(x[::-1].copy()))
    ref.append(0, 0, x, x[::-1])
    check_row(hip, kv, ref, 0, 0, n * 32)


@pytest.mark.parametrize("nkv,paged", [(2, False), (1, True), (3, True)])
def test_append_in_pieces(hip, nkv, paged):
    """Blocks that fill over several calls, their scales growing; positions taken
    back; a batch with sequences without tokens; rows of a pitch."""
    rng = np.random.default_rng(11 + nkv)
    rows, max_blocks = 4, 5
    kv, ref = make(hip, rng, nkv, rows, max_blocks, paged), R.Cache(nkv, rows, max_blocks)
    pos = np.zeros(rows, np.int64)
    for step in range(24):
        order = rng.permutation(rows)[:rng.integers(1, rows + 1)] if paged else np.arange(rows)
        new = np.array([min(int(rng.choice([0, 1, 1, 2, 3, 31, 32, 33, 70])), max_blocks * 32 - pos[r]) for r in order])
        T, pad = int(new.sum()), int(rng.choice([0, 8, 40]))
        k, v = (np.concatenate((np.full((T, pad), 0x7fc0, np.uint16), kv_rows(rng, T, nkv)), 1) for _ in range(2))
        cu = cum(new)
        hip.kv8_append(kv, order if paged else None, cu, pos[order], dev(k)[:, pad:], dev(v)[:, pad:])
        for i, r in enumerate(order):
            ref.append(r, int(pos[r]), k[cu[i]:cu[i + 1], pad:], v[cu[i]:cu[i + 1], pad:])
            pos[r] += new[i]
            if pos[r]:
                check_row(hip, kv, ref, int(r), 0, int(pos[r]))
            back = int(rng.choice([0, 0, 1, 3]))
            pos[r] = max(0, pos[r] - back)
            if pos[r] == max_blocks * 32:
                pos[r] = 5


def test_append_leaves_the_rest(hip):
    """Bytes of other blocks, other positions and other rows stay as they were."""
    rng = np.random.default_rng(3)
    nkv = 2
    kv = make(hip, rng, nkv, 3, 4, False)
    k, v, scale, _ = kv._tensors
    for t in (k, v):
        t.copy_(torch.from_numpy(rng.integers(0, 0x7e, t.shape, dtype=np.uint8)).cuda())
    scale.fill_(2.0 ** 20)                 # (large: the new tokens do not move it)
    k0, v0, s0 = k.clone(), v.clone(), scale.clone()
    x = kv_rows(rng, 3, nkv, spread=1.0)
    hip.kv8_append(kv, None, [0, 0, 3, 3], [0, 40, 0], dev(x), dev(x))
    torch.cuda.synchronize()
    # row 1, block 1 (id 5), positions 40..42
    for a, b, which in ((k, k0, "k"), (v, v0, "v")):
        diff = (a != b).cpu().numpy()
        assert not diff[[i for i in range(12) if i != 5]].any()
        at = np.zeros(8192, bool)
        for key in range(8, 11):
            for d in range(R.D):
                if which == "k":
                    at[((key // 16) * 16 + d // 16) * 256 + key % 16 * 16 + d % 16] = True
                else:
                    at[d // 32 * 1024 + (key % 16 // 4 * 16 + d % 16) * 16 + d // 16 % 2 * 8 + key // 16 * 4 + key % 4] = True
        assert not diff[5][:, ~at].any()
    s = scale.cpu().numpy()
    assert (s == s0.cpu().numpy()).all()


def test_bad_table_entries(hip):
    """Entries that are no block: nothing is written through them, and reading
    them reads some block."""
    rng = np.random.default_rng(5)
    t = torch.tensor([[0, 1], [-1, 1 << 30]], dtype=torch.int32).cuda()
    kv = hip.kv8_cache(1, 3, 2, block_table=t)
    for x in kv._tensors[:2]:
        x.zero_()
    kv._tensors[2].fill_(1.0)
    before = [x.clone() for x in kv._tensors[:3]]
    x = dev(kv_rows(rng, 40, 1))
    hip.kv8_append(kv, [1], [0, 40], [0], x, x)
    for a, b in zip(kv._tensors, before):
        assert torch.equal(a, b)
    out = torch.empty_like(x)
    hip.kv8_read(kv, [1], [0, 40], [0], out, torch.empty_like(out))
    torch.cuda.synchronize()


class Setup:
    """A batch of sequences whose caches are filled, and the reference's."""

    def __init__(self, hip, seed, nkv, ctx, new, paged, spread=1.0, fill=True):
        self.rng = rng = np.random.default_rng(seed)
        self.hip, self.nkv, self.nh = hip, nkv, nkv * R.GRP
        self.ctx, self.new = np.asarray(ctx), np.asarray(new)
        B = len(ctx)
        self.max_blocks = int(max(1, -(-(self.ctx + self.new).max() // 32)))
        self.kv = make(hip, rng, nkv, B, self.max_blocks, paged)
        self.ref = R.Cache(nkv, B, self.max_blocks)
        self.rows = rng.permutation(B).astype(np.int32) if paged else None
        self.cu = cum(self.new)
        self.w = dict(qn_w=R.bf16(rng.normal(size=R.D) * 0.1), kn_w=R.bf16(rng.normal(size=R.D) * 0.1))
        self.dw = {k: dev(v) for k, v in self.w.items()}
        self.layer = hip.attn_layer((self.nh, nkv, R.D, R.ROT, THETA), self.dw)
        self.work = hip.AttnKv8Work(self.layer, B, self.max_blocks * 32)
        n = self.ctx + (self.new if fill else 0)
        T = int(n.sum())
        self.k, self.v = kv_rows(rng, T, nkv, spread), kv_rows(rng, T, nkv, spread)
        c = cum(n)
        if T:
            hip.kv8_append(self.kv, self.rows, c, np.zeros(B, np.int32), dev(self.k), dev(self.v))
        for s in range(B):
            self.ref.append(self.row(s), 0, self.k[c[s]:c[s + 1]], self.v[c[s]:c[s + 1]])
        self.qg = R.bf16(rng.normal(size=(int(self.new.sum()), self.nh, 2 * R.D)))
        self.y = torch.full((len(self.qg) + 2, self.nh * R.D), 0x1234, dtype=torch.int16, device="cuda")

    def row(self, s):
        return int(self.rows[s]) if self.rows is not None else s

    def call(self, f, k=None, v=None):
        T = len(self.qg)
        f(self.layer, self.work, self.rows, self.cu, self.ctx, dev(self.qg), k, v, self.kv, self.y[:T])
        torch.cuda.synchronize()
        assert (self.y[T:] == 0x1234).all()                # rows behind the last sequence
        return host(self.y[:T]).reshape(T, self.nh, R.D)

    def check(self, y, seqs=None):
        for s in range(len(self.ctx)) if seqs is None else seqs:
            n, p = int(self.new[s]), int(self.ctx[s])
            if not n:
                continue
            k, v = self.ref.values(self.row(s), 0, p + n)
            r, tol = R.attention(self.qg[self.cu[s]:self.cu[s + 1]], self.w["qn_w"], p, k, v, THETA)
            d = np.abs(R.f64(y[self.cu[s]:self.cu[s + 1]]) - r)
            assert (d <= tol).all(), f"sequence {s} ({p} + {n}): {np.max(d / tol)} of the bound"


CTX = [0, 1, 30, 31, 32, 33, 62, 63, 64, 255, 257, 1000]


@pytest.mark.parametrize("tq", [1, 2, 3, 4])
@pytest.mark.parametrize("nkv,paged", [(2, False), (1, True), (3, True)])
def test_decode(hip, tq, nkv, paged):
    rng = np.random.default_rng(tq)
    new = [tq] + list(rng.integers(0, tq + 1, len(CTX) - 1))
    s = Setup(hip, 100 + tq + nkv, nkv, CTX, new, paged)
    s.check(s.call(hip.attn_decode_kv8))


@pytest.mark.parametrize("tq,ctx", [(1, 0), (1, 1499), (3, 29), (4, 7000), (2, 20000)])
def test_decode_one_sequence(hip, tq, ctx):
    s = Setup(hip, ctx, 2, [ctx], [tq], ctx % 2 == 0)
    s.check(s.call(hip.attn_decode_kv8))


@pytest.mark.parametrize("new", [[1, 1, 0, 1, 1, 1], [4, 1, 0, 2, 3, 4]])
def test_decode_long_runs(hip, new):
    """Enough keys for runs of unequal length, two a CU (shared blocks: a row's
    table repeats a few): every part of each context counts, at its position."""
    rng = np.random.default_rng(17)
    nkv, few, max_blocks = 2, 40, 4096
    ctx = np.array([131000, 64000, 90000, 33, 100, 120001])
    t = rng.integers(0, few, (len(ctx), max_blocks)).astype(np.int32)
    kv = hip.kv8_cache(nkv, few, max_blocks, block_table=torch.from_numpy(t).cuda())
    ident = hip.kv8_cache(nkv, few, few, block_table=torch.arange(few, dtype=torch.int32, device="cuda")[None].contiguous())
    ident.k, ident.v, ident.scale = kv.k, kv.v, kv.scale
    x = [kv_rows(rng, few * 32, nkv, 1.0) for _ in range(2)]
    hip.kv8_append(ident, None, [0, few * 32], [0], dev(x[0]), dev(x[1]))
    ref = R.Cache(nkv, 1, few)
    ref.append(0, 0, x[0], x[1])
    kk, vv = (a.reshape(few, 32, nkv, R.D) for a in ref.values(0, 0, few * 32))
    w = dict(qn_w=R.bf16(rng.normal(size=R.D) * 0.1), kn_w=R.bf16(rng.normal(size=R.D) * 0.1))
    layer = hip.attn_layer((nkv * R.GRP, nkv, R.D, R.ROT, THETA), {k: dev(v) for k, v in w.items()})
    work = hip.AttnKv8Work(layer, len(ctx), max_blocks * 32)
    cu = cum(new)
    qg = R.bf16(rng.normal(size=(int(cu[-1]), nkv * R.GRP, 2 * R.D)))
    y = torch.empty(len(qg), nkv * R.GRP * R.D, dtype=torch.int16, device="cuda")
    hip.attn_decode_kv8(layer, work, None, cu, ctx, dev(qg), None, None, kv, y)
    got = R.f64(host(y)).reshape(len(qg), -1, R.D)
    for s in range(len(ctx)):
        if not new[s]:
            continue
        n = int(ctx[s] + new[s])
        b = t[s, :-(-n // 32)]
        k, v = (a[b].reshape(-1, nkv, R.D)[:n] for a in (kk, vv))
        r, tol = R.attention(qg[cu[s]:cu[s + 1]], w["qn_w"], int(ctx[s]), k, v, THETA)
        assert (np.abs(got[cu[s]:cu[s + 1]] - r) <= tol).all(), s
    z = torch.empty_like(y)
    hip.attn_decode_kv8(layer, work, None, cu, ctx, dev(qg), None, None, kv, z)
    torch.cuda.synchronize()
    assert torch.equal(y, z)


@pytest.mark.parametrize("tq", [1, 4])
def test_decode_many_sequences(hip, tq):
    """More sequences than one launch takes."""
    rng = np.random.default_rng(tq)
    ctx = rng.integers(0, 150, 461)
    s = Setup(hip, 7 + tq, 2, ctx, rng.integers(0, tq + 1, 461), True)
    s.check(s.call(hip.attn_decode_kv8), list(range(0, 461, 9)) + [206, 207, 208, 209, 222, 223, 224, 225, 415, 416, 447, 448, 449, 460])


def test_decode_growing_scores(hip):
    """Scores that rise along the context, far past the first keys'."""
    s = Setup(hip, 21, 2, [900], [4], False, spread=0.1)
    k = R.f64(s.k).reshape(-1, 2, R.D) * np.linspace(0.1, 40.0, len(s.k))[:, None, None]
    s.k = R.bf16(k).reshape(len(k), -1)
    hip.kv8_append(s.kv, None, [0, 904], [0], dev(s.k), dev(s.v))
    s.ref.append(0, 0, s.k, s.v)
    s.check(s.call(hip.attn_decode_kv8))
    s.check(s.call(hip.attn_prefill_kv8))


@pytest.mark.parametrize("f", ["attn_decode_kv8", "attn_prefill_kv8"])
@pytest.mark.parametrize("q,k", [(0.0, 0.0), (2.0 ** -126, 0.0), (2.0 ** -126, 2.0 ** -133), (1.0, 0.0), (2.0 ** -126, 1.0),
                                 (0.0, 1.0), (1.0, 2.0 ** 100)])
def test_tiny_and_large_rows(hip, f, q, k):
    """Rows of zeros and of the smallest values: every key counts the same; and k
    so large that one key has it all."""
    s = Setup(hip, 23, 2, [37, 0], [4, 3], False)
    s.qg.reshape(-1, 2 * R.D)[:, :R.D] = R.bf16(R.f64(s.qg).reshape(-1, 2 * R.D)[:, :R.D] * q)
    s.k = R.bf16(R.f64(s.k) * k)
    n = s.ctx + s.new
    c = cum(n)
    hip.kv8_append(s.kv, None, c, [0, 0], dev(s.k), dev(s.v))
    for i in range(2):
        s.ref.append(i, 0, s.k[c[i]:c[i + 1]], s.v[c[i]:c[i + 1]])
    s.check(s.call(getattr(hip, f)))


@pytest.mark.parametrize("f", ["attn_decode_kv8", "attn_prefill_kv8"])
@pytest.mark.parametrize("what", ["k", "v"])
def test_nan_reaches_only_those_that_see_it(hip, f, what):
    """A token whose k or v holds NaN or infinity: rows before it are as without
    it; rows that see a NaN k are NaN, those that see NaN v are NaN in that dim."""
    s = Setup(hip, 31, 2, [61], [4], False)
    x = {"k": s.k.copy(), "v": s.v.copy()}
    x[what][62, 300] = 0x7fc0              # position 62: the second new token; head 1, dim 44
    x[what][62, 301] = 0xff80
    hip.kv8_append(s.kv, None, [0, 65], [0], dev(x["k"]), dev(x["v"]))
    y = s.call(getattr(hip, f))
    clean = R.Cache(2, 1, s.max_blocks)
    x[what][62, 300:302] = 0
    clean.append(0, 0, x["k"], x["v"])
    k, v = clean.values(0, 0, 65)
    r, tol = R.attention(s.qg, s.w["qn_w"], 61, k, v, THETA)
    bad = np.zeros(y.shape, bool)
    if what == "k":
        bad[1:, 8:] = True
    else:
        bad[1:, 8:, 44:46] = True
    got = R.f64(y)
    assert np.array_equal(np.isnan(got), bad)
    ok = ~bad
    if what == "k":
        ok[1:] = False                     # (head 0's rows have another key set: checked below)
        ok[1:, :8] = True
    assert (np.abs(got - r)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("ctx,new", [([127], [1]), ([255, 100], [2, 1]), ([1000], [2]), ([90, 3, 60], [1, 1, 2])])
def test_decode_nan_in_the_last_block(hip, ctx, new):
    """One row block (at most two tokens), a NaN v among the keys of the last block,
    while the other wavefronts are done with theirs: its dims alone are NaN."""
    s = Setup(hip, 33, 2, ctx, new, False)
    n = np.asarray(ctx) + new
    c = cum(n)
    bad = np.zeros((int(sum(new)), s.nh, R.D), bool)
    for i, p in enumerate(ctx):
        at = c[i] + (n[i] - 1) // 32 * 32                  # the last block's first position
        s.v[at, 3::7] = 0x7fc0                             # head 0's and 1's dims
        head = (np.arange(512) % 7 == 3).reshape(2, R.D)
        for t in range(new[i]):
            if p + t >= at - c[i]:
                bad[s.cu[i] + t] = head.repeat(R.GRP, 0)
    hip.kv8_append(s.kv, None, c, np.zeros(len(ctx), np.int32), dev(s.k), dev(s.v))
    for i in range(len(ctx)):
        v = s.v[c[i]:c[i + 1]].copy()
        v[(v & 0x7fff) > 0x7f80] = 0
        s.ref.append(i, 0, s.k[c[i]:c[i + 1]], v)
    y = s.call(hip.attn_decode_kv8)
    assert np.array_equal(np.isnan(R.f64(y)), bad)
    for i in range(len(ctx)):
        k, v = s.ref.values(i, 0, int(n[i]))
        sl = slice(s.cu[i], s.cu[i + 1])
        r, tol = R.attention(s.qg[sl], s.w["qn_w"], ctx[i], k, v, THETA)
        assert (np.abs(R.f64(y[sl]) - r) <= tol)[~bad[sl]].all()


def test_shared_rows(hip):
    """Without k and v, sequences may read one row: a shared prompt."""
    s = Setup(hip, 41, 2, [500, 500], [2, 2], True)
    y0 = s.call(hip.attn_decode_kv8)
    T = len(s.qg)
    y = torch.empty(T, s.nh * R.D, dtype=torch.int16, device="cuda")
    hip.attn_decode_kv8(s.layer, s.work, [s.row(0), s.row(0)], s.cu, [500, 500],
                        dev(np.concatenate((s.qg[:2], s.qg[:2]))), None, None, s.kv, y)
    y = host(y).reshape(T, s.nh, R.D)
    s.check(np.concatenate((y[:2], y0[2:])))
    s.check(np.concatenate((y[2:], y0[2:])))


@pytest.mark.parametrize("f,new", [("attn_decode_kv8", [1, 3, 0, 4, 2]), ("attn_prefill_kv8", [1, 40, 0, 33, 97])])
def test_mixer_appends(hip, f, new):
    """With k and v: the rows that the bf16 mixer appends (bitwise the
    reference's), quantised; then the same attention as without."""
    ctx = [0, 33, 9, 250, 64]
    s = Setup(hip, 51, 2, ctx, new, True, fill=False)
    T = int(sum(new))
    k, v = kv_rows(s.rng, T, 2, 1.0), kv_rows(s.rng, T, 2, 1.0)
    y = s.call(getattr(hip, f), dev(k), dev(v))
    # the bf16 mixer's appended rows
    ms = s.max_blocks * 32
    kc, vc = (torch.zeros(len(ctx) * ms * 512, dtype=torch.int16, device="cuda") for _ in range(2))
    live = [i for i in range(len(ctx)) if new[i]]
    yb = torch.empty(T, s.nh * R.D, dtype=torch.int16, device="cuda")
    hip.attn_prefill(s.layer, s.cu, ctx, dev(s.qg), dev(k), dev(v), kc, vc, ms, yb)
    for i in live:
        a, b = (torch.empty(ctx[i] + new[i], 512, dtype=torch.int16, device="cuda") for _ in range(2))
        hip.attn_cache_unpack(kc[i * ms * 512:], vc[i * ms * 512:], ctx[i] + new[i], 2, 256, ms, a, b)
        s.ref.append(s.row(i), ctx[i], host(a)[ctx[i]:], host(b)[ctx[i]:])
        check_row(hip, s.kv, s.ref, s.row(i), 0, ctx[i] + new[i])
    s.check(y)
    assert np.array_equal(y, s.call(getattr(hip, f)))


@pytest.mark.parametrize("ctx,new,nkv,paged", [
    ([0], [1], 2, False), ([0], [31], 2, False), ([0], [65], 1, False), ([0], [300], 2, True),
    ([31, 0, 100, 64, 5], [33, 0, 1, 130, 64], 2, True), ([777, 3], [50, 129], 3, True), ([2050], [9], 2, False)])
def test_prefill(hip, ctx, new, nkv, paged):
    s = Setup(hip, 60 + len(ctx) + new[0], nkv, ctx, new, paged)
    s.check(s.call(hip.attn_prefill_kv8))


@pytest.mark.parametrize("ctx,new,nkv,paged", [
    ([5000], [3], 2, True), ([9000], [40], 1, False), ([30000], [1], 2, True), ([5000, 40, 1200, 700], [3, 20, 17, 0], 2, True),
    ([0, 3000], [700, 5], 1, False), ([0], [1000], 1, True), ([6000] * 9, [1, 2, 15, 16, 17, 1, 0, 33, 8], 3, True)])
def test_prefill_split(hip, ctx, new, nkv, paged):
    """Few new tokens after long contexts: a tile's keys in several parts, of which
    a prompt's first tiles have fewer than the last; rows see NaN by position."""
    s = Setup(hip, 80 + len(ctx) + new[0], nkv, ctx, new, paged)
    y = s.call(hip.attn_prefill_kv8)
    s.check(y)
    q = int(np.argmax(s.ctx))
    n = int(s.ctx[q] + s.new[q])
    c = cum(s.ctx + s.new)
    v = s.v[c[q]:c[q + 1]].copy()
    at = [n // 2, n - 1]                                   # dims 5 and 250 of the last head
    v[at[0], -R.D + 5], v[at[1], -R.D + 250] = 0x7fc0, 0xff80
    hip.kv8_append(s.kv, [s.row(q)], [0, n], [0], dev(s.k[c[q]:c[q + 1]]), dev(v))
    bad = np.zeros(y.shape, bool)
    for t in range(int(s.new[q])):
        for d, a in ((5, at[0]), (250, at[1])):
            bad[s.cu[q] + t, -R.GRP:, d] = s.ctx[q] + t >= a
    z = s.call(hip.attn_prefill_kv8)
    assert np.array_equal(np.isnan(R.f64(z)), bad)
    v[at, [-R.D + 5, -R.D + 250]] = 0
    s.ref.append(s.row(q), 0, s.k[c[q]:c[q + 1]], v)
    kk, vv = s.ref.values(s.row(q), 0, n)
    sl = slice(s.cu[q], s.cu[q + 1])
    r, tol = R.attention(s.qg[sl], s.w["qn_w"], int(s.ctx[q]), kk, vv, THETA)
    assert (np.abs(R.f64(z[sl]) - r) <= tol)[~bad[sl]].all()


@pytest.mark.parametrize("nkv,nan", [(2, None), (3, "k"), (2, "v")])
def test_prefill_many_tokens(hip, nkv, nan):
    """Work for every CU many times over (tiles of 32 tokens): ragged sequences;
    with a NaN in a new token of one, which reaches the rows from it on."""
    rng = np.random.default_rng(13)
    B = 160
    ctx, new = rng.integers(0, 200, B), rng.integers(1, 75, B)
    ctx[:4], new[:4] = [0, 31, 64, 33], [70, 33, 32, 66]
    s = Setup(hip, 73, nkv, ctx, new, True)
    picks = [0, 1, 2, 3] + list(range(7, B, 23))
    if nan is None:
        s.check(s.call(hip.attn_prefill_kv8), picks)
        return
    want = s.call(hip.attn_prefill_kv8)
    n = ctx + new
    c, q = cum(n), 3
    x = {"k": s.k.copy(), "v": s.v.copy()}
    x[nan][c[q] + 33 + 40, 256 + 17] = 0xffc0              # the 41st new token; head 1, dim 17
    sl = slice(c[q], c[q + 1])
    hip.kv8_append(s.kv, [s.row(q)], [0, int(n[q])], [0], dev(x["k"][sl]), dev(x["v"][sl]))
    y = s.call(hip.attn_prefill_kv8)
    bad = np.zeros(y.shape, bool)
    at, end = s.cu[q] + 40, s.cu[q + 1]
    bad[at:end, 8:16, slice(17, 18) if nan == "v" else slice(None)] = True
    got = R.f64(y)
    assert np.array_equal(np.isnan(got), bad)
    # (the sequence's block has another scale where the NaN stood for its largest value)
    s.check(want, picks)
    others = np.ones(len(y), bool)
    others[s.cu[q]:end] = False
    assert np.array_equal(y[others], want[others])
    x[nan][c[q] + 73, 273] = 0
    s.ref.append(s.row(q), 0, x["k"][sl], x["v"][sl])
    kk, vv = s.ref.values(s.row(q), 0, int(n[q]))
    rs = slice(s.cu[q], end)
    r, tol = R.attention(s.qg[rs], s.w["qn_w"], int(ctx[q]), kk, vv, THETA)
    ok = ~bad[rs]
    if nan == "k":
        ok[40:, 8:16] = False
    assert (np.abs(got[rs] - r) <= tol)[ok].all()


def test_prefill_many_sequences(hip):
    rng = np.random.default_rng(9)
    s = Setup(hip, 71, 1, rng.integers(0, 60, 230), rng.integers(0, 6, 230), True)
    s.check(s.call(hip.attn_prefill_kv8), list(range(0, 230, 11)) + [206, 207, 208, 209, 223, 224, 229])


def test_pool(hip):
    """An 8-bit pool: rows grow, close and are taken again; positions past a
    row's blocks are refused; the bf16 descriptor is refused."""
    rng = np.random.default_rng(81)
    p = hip.KvPool(2, 2, 256, 6, 3, 4, kv8=True)
    with pytest.raises(hip.ApusHipError):
        c = hip.KvCache()
        hip._chk(hip.load().apus_hip_kv_pool_cache(p.h, 0, hip.C.byref(c)))
    kv = p.cache(1)
    a, b = p.open(), p.open()
    p.reserve(a, 40)
    x = kv_rows(rng, 40, 2)
    hip.kv8_append(kv, [a], [0, 40], [0], dev(x), dev(x))
    with pytest.raises(hip.ApusHipError):
        hip.kv8_append(kv, [a], [0, 40], [25], dev(x), dev(x))
    with pytest.raises(hip.ApusHipError):
        hip.kv8_append(kv, [b], [0, 1], [0], dev(x)[:1], dev(x)[:1])
    ref = R.Cache(2, 3, 4)
    ref.append(a, 0, x, x)
    check_row(hip, kv, ref, a, 0, 40)
    p.close(a)
    with pytest.raises(hip.ApusHipError):
        hip.kv8_read(kv, [a], [0, 1], [0], dev(x)[:1], dev(x)[:1])
    assert p.free_blocks() == 6
    p.reserve(b, 128)
    y = kv_rows(rng, 128, 2)
    hip.kv8_append(kv, [b], [0, 128], [0], dev(y), dev(y))
    ref.append(b, 0, y, y)
    check_row(hip, kv, ref, b, 0, 128)
    p.destroy()


def test_other_stream_and_graph(hip):
    """A whole step (append, attention) captured and replayed, between eager
    work: every replay as the eager call; host arrays are the call's."""
    s = Setup(hip, 91, 2, [100, 700], [1, 3], True, fill=False)
    T = 4
    k, v = dev(kv_rows(s.rng, T, 2, 1.0)), dev(kv_rows(s.rng, T, 2, 1.0))
    qg, y = dev(s.qg), torch.empty(T, s.nh * R.D, dtype=torch.int16, device="cuda")
    pos = np.array(s.ctx, np.int32)
    call = hip.attn_decode_kv8_bound(s.layer, s.work, s.rows, s.cu, pos, qg, k, v, s.kv, y)
    call()
    torch.cuda.synchronize()
    want = y.clone()
    st = torch.cuda.Stream()
    hip.set_stream(st.cuda_stream)
    try:
        st.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            call()
        pos[:] = 0                                         # (the graph keeps what the call was given)
        for i in range(4):
            y.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), i
            torch.randn(1000, device="cuda").sum().item()
    finally:
        hip.set_stream(0)


def test_overlapping_replays(hip):
    """Two captured calls with a workspace each, replayed at once on two streams;
    two with one, one after the other."""
    a, b = (Setup(hip, 95 + i, 2, [3000, 2500 + i], [2, 1], False) for i in range(2))
    want, graphs = [], []
    for s in (a, b):
        want.append(s.call(hip.attn_decode_kv8))
        st, y = torch.cuda.Stream(), torch.zeros(3, s.nh * R.D, dtype=torch.int16, device="cuda")
        call = hip.attn_decode_kv8_bound(s.layer, s.work, s.rows, s.cu, s.ctx, dev(s.qg), None, None, s.kv, y)
        st.wait_stream(torch.cuda.current_stream())
        hip.set_stream(st.cuda_stream)
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                for _ in range(20):
                    call()
        finally:
            hip.set_stream(0)
        graphs.append((g, st, y, call))
    for i in range(4):
        for _, _, y, _ in graphs:
            y.zero_()
        torch.cuda.synchronize()
        for g, st, _, _ in graphs:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (_, _, y, _), w in zip(graphs, want):
            assert np.array_equal(host(y).reshape(w.shape), w), i
        torch.randn(1000, device="cuda").sum().item()
    # one workspace: b's call with a's
    y = torch.zeros(3, b.nh * R.D, dtype=torch.int16, device="cuda")
    graphs[0][0].replay()
    torch.cuda.synchronize()
    hip.attn_decode_kv8(b.layer, a.work, b.rows, b.cu, b.ctx, dev(b.qg), None, None, b.kv, y)
    torch.cuda.synchronize()
    assert np.array_equal(host(y).reshape(want[1].shape), want[1])


def test_call_refusals(hip):
    """What only a workspace's call can refuse, and the binding's own checks;
    nothing is written."""
    s = Setup(hip, 97, 2, [100, 64], [1, 4], False)
    k = torch.zeros(5, 512, dtype=torch.int16, device="cuda")
    qg, y = dev(s.qg), torch.full((5, s.nh * R.D), 0x77, dtype=torch.int16, device="cuda")
    base = dict(layer=s.layer, work=s.work, rows=None, cu=s.cu, pos0=s.ctx, qg=qg, k=k, v=k, kv=s.kv, y=y)
    state = [t.clone().view(torch.uint8) for t in s.kv._tensors[:3]]   # (bytes: untouched scales are NaN)

    def refused(match, f=hip.attn_decode_kv8, exc=hip.ApusHipError, **kw):
        with pytest.raises(exc, match=match):
            f(**dict(base, **kw))

    refused("0..4 new", cu=[0, 0, 5])
    refused("both", k=None)
    refused("both", v=None, f=hip.attn_prefill_kv8)
    refused("overlap", y=qg.view(-1)[:5 * s.nh * R.D].view(5, -1))
    refused("overlap", y=s.kv._tensors[0].view(torch.int16).view(-1)[:5 * s.nh * R.D].view(5, -1))
    refused("overlap", k=s.kv._tensors[1].view(torch.int16).view(-1)[:5 * 512].view(5, -1))
    refused("one row", rows=[1, 1])
    refused("outside", rows=[1, 2])
    refused("offsets", cu=[1, 1, 5])
    refused("ascend", cu=[0, 6, 5])
    refused("overflows", pos0=[-1, 0])
    refused("overflows", pos0=[0, s.max_blocks * 32 - 3])
    short, other = hip.AttnKv8Work(s.layer, 1, 100), hip.AttnKv8Work(hip.attn_layer((24, 3, R.D, R.ROT, THETA), s.dw), 2, 200)
    refused("position", work=short)
    refused("position", work=short, f=hip.attn_prefill_kv8)
    refused("holds 1", work=short, pos0=[0, 0])
    refused("other dims", work=other)
    for w in (short, other):
        w.destroy()
        refused("workspace", work=w)
    bound = hip.attn_decode_kv8_bound(**dict(base, work=hip.AttnKv8Work(s.layer, 2, 200)))
    bound._keep[1].destroy()
    with pytest.raises(hip.ApusHipError, match="workspace"):
        bound()
    refused("qg", exc=ValueError, qg=qg[:4])
    refused("y", exc=ValueError, y=y.float())
    refused("k", exc=ValueError, k=k.cpu())
    refused("heads", exc=ValueError, kv=hip.kv8_cache(1, 8, 4))
    refused("offset", exc=ValueError, cu=[0, 1, 2, 5])
    rows = lambda **kw: dict(dict(kv=s.kv, rows=None, cu=s.cu, pos0=s.ctx, k=k, v=k), **kw)      # noqa: E731
    for kw, exc, match in ((dict(k=k[:1].expand(5, 512)), hip.ApusHipError, "pitch"), (dict(k=k[:, ::2]), ValueError, "k"),
                           (dict(v=k[:, :256]), ValueError, "v"), (dict(k=k.view(5, 2, 256).transpose(1, 2)), ValueError, "k"),
                           (dict(k=torch.zeros(5, 2, 512, dtype=torch.int16, device="cuda")[:, :, :256]), ValueError, "k"),
                           (dict(k=k[:4]), ValueError, "k"), (dict(rows=[0, 0]), hip.ApusHipError, "one row")):
        with pytest.raises(exc, match=match):
            hip.kv8_append(**rows(**kw))
    with pytest.raises(ValueError):
        hip.kv8_cache(2, 8, 4, d=128)
    with pytest.raises(ValueError, match="block_table"):
        hip.kv8_cache(2, 8, 4, block_table=torch.zeros(2, 4, dtype=torch.int64, device="cuda"))
    torch.cuda.synchronize()
    assert (y == 0x77).all()
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(state, s.kv._tensors))
    # nothing to do: no tokens at all, no sequences
    none = torch.empty(0, s.nh * R.D, dtype=torch.int16, device="cuda")
    for f in (hip.attn_decode_kv8, hip.attn_prefill_kv8):
        f(s.layer, s.work, None, [0, 0, 0], [5, 0], qg[:0], k[:0], k[:0], s.kv, none)
        f(s.layer, s.work, None, [0], [], qg[:0], None, None, s.kv, none)
    hip.kv8_append(s.kv, None, [0, 0, 0], [5, 0], k[:0], k[:0])
    hip.kv8_read(s.kv, None, [0], [], k[:0], k[:0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(state, s.kv._tensors))


def test_nan_stays_through_a_rescale(hip):
    """A stored NaN and a -0 keep what they are when later tokens of their block
    bring a larger scale."""
    rng = np.random.default_rng(99)
    kv, ref = make(hip, rng, 1, 1, 1, False), R.Cache(1, 1, 1)
    pos = 0
    for n, size in ((5, 1.0), (3, 100.0), (1, 3e5), (4, 1e-3), (2, 1e30)):
        k, v = (R.bf16(rng.normal(size=(n, R.D)) * size) for _ in range(2))
        k[0, 7], v[0, 9], k[-1, 11], v[-1, 12] = 0x7fc0, 0xff80, 0x8000, 0x8000
        hip.kv8_append(kv, None, [0, n], [pos], dev(k), dev(v))
        ref.append(0, pos, k, v)
        pos += n
        check_row(hip, kv, ref, 0, 0, pos)


def test_blocks_past_4_gib(hip):
    """A cache of 4.9 GB each for K and V: blocks on both sides of 4 GiB."""
    rng = np.random.default_rng(101)
    nkv, blocks = 2, 300000
    t = torch.tensor([[299999, 7, 262144, 131072], [262143, 299998, 0, 262145]], dtype=torch.int32).cuda()
    kv, ref = hip.kv8_cache(nkv, blocks, 4, block_table=t), R.Cache(nkv, 2, 4)
    ctx, new = np.array([100, 90]), np.array([3, 4])
    n = ctx + new
    c = cum(n)
    k, v = kv_rows(rng, int(c[-1]), nkv, 1.0), kv_rows(rng, int(c[-1]), nkv, 1.0)
    hip.kv8_append(kv, None, c, [0, 0], dev(k), dev(v))
    for s in range(2):
        ref.append(s, 0, k[c[s]:c[s + 1]], v[c[s]:c[s + 1]])
        check_row(hip, kv, ref, s, 0, int(n[s]))
    w = dict(qn_w=R.bf16(rng.normal(size=R.D) * 0.1), kn_w=R.bf16(rng.normal(size=R.D) * 0.1))
    layer = hip.attn_layer((nkv * R.GRP, nkv, R.D, R.ROT, THETA), {a: dev(b) for a, b in w.items()})
    work = hip.AttnKv8Work(layer, 2, 128)
    for f, take in ((hip.attn_decode_kv8, new), (hip.attn_prefill_kv8, n)):
        cu, pos = cum(take), n - take
        qg = R.bf16(rng.normal(size=(int(cu[-1]), nkv * R.GRP, 2 * R.D)))
        y = torch.empty(len(qg), nkv * R.GRP * R.D, dtype=torch.int16, device="cuda")
        f(layer, work, None, cu, pos, dev(qg), None, None, kv, y)
        got = R.f64(host(y)).reshape(len(qg), -1, R.D)
        for s in range(2):
            a, b = ref.values(s, 0, int(n[s]))
            r, tol = R.attention(qg[cu[s]:cu[s + 1]], w["qn_w"], int(pos[s]), a, b, THETA)
            assert (np.abs(got[cu[s]:cu[s + 1]] - r) <= tol).all(), s


@pytest.mark.parametrize("pad", [0, 8, 24])
def test_read_leaves_the_rest(hip, pad):
    """Rows of a pitch, sequences without tokens: nothing beside the rows."""
    rng = np.random.default_rng(103)
    kv, ref = make(hip, rng, 2, 3, 3, True), R.Cache(2, 3, 3)
    x, z = kv_rows(rng, 200, 2), kv_rows(rng, 200, 2)
    cu, n = [0, 70, 70, 165], [70, 0, 95]
    hip.kv8_append(kv, None, cu, [0, 0, 0], dev(x[:165]), dev(z[:165]))
    for s in (0, 2):
        ref.append(s, 0, x[cu[s]:cu[s + 1]], z[cu[s]:cu[s + 1]])
    out = [torch.full((60, 512 + pad), 0x55, dtype=torch.int16, device="cuda") for _ in range(2)]
    hip.kv8_read(kv, [2, 1, 0], [0, 40, 40, 57], [31, 0, 33], out[0][:57, pad:], out[1][:57, pad:])
    torch.cuda.synchronize()
    for i, o in enumerate(out):
        g = host(o)
        assert (g[57:] == 0x55).all() and (g[:, :pad] == 0x55).all()
        a = R.bf16(ref.values(2, 31, 71)[i]).reshape(40, 512)
        b = R.bf16(ref.values(0, 33, 50)[i]).reshape(17, 512)
        assert same(g[:57, pad:], np.concatenate((a, b)))
