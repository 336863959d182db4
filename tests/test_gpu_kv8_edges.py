"""The 8-bit KV cache on the GPU where its calls are at their limits."""
import numpy as np
import pytest
import torch

import kv8_ref as R
from test_gpu_kv8 import Setup, check_row, cum, dev, make, table
from test_gpu_kv8_step import H, MAX, Model, empty

pytestmark = pytest.mark.gpu
TOP = 240.0 * 2.0 ** 120                   # the largest finite value: 256 2^120 is no bf16


class Cache(R.Cache):
    """The reference's cache up to bf16's largest value: codes at 2^120 end at 240."""

    def append(self, row, pos0, k, v):
        super().append(row, pos0, k, v)
        c, mag = self.codes[row], self.codes[row] & 0x7f
        at = (self.exps[row].repeat(R.BLK, 0) == 120)[..., None] & (mag > 0x77) & (mag < 0x7f)
        self.codes[row] = np.where(at, c & 0x80 | 0x77, c)


def refill(s):
    """The caches of a Setup from its k and v again."""
    n = s.ctx + s.new
    c = cum(n)
    s.hip.kv8_append(s.kv, s.rows, c, np.zeros(len(n), np.int32), dev(s.k), dev(s.v))
    s.ref = Cache(s.nkv, len(n), s.max_blocks)
    for i in range(len(n)):
        s.ref.append(s.row(i), 0, s.k[c[i]:c[i + 1]], s.v[c[i]:c[i + 1]])


@pytest.mark.parametrize("ctx,new", [
    ([0, 4080], [0, 16]), ([0, 700], [0, 500]), ([0, 5000, 40], [0, 20, 20]), ([5000, 0, 40, 30000], [20, 0, 20, 0]),
    ([0, 0, 9000], [0, 0, 7])])
def test_prefill_split_beside_idle_rows(hip, ctx, new):
    """Keys in parts, beside sequences without tokens or cached positions."""
    s = Setup(hip, 110 + len(ctx) + new[-1], 2, ctx, new, True)
    s.check(s.call(hip.attn_prefill_kv8))


def test_largest_values_stay_finite(hip):
    """Every bf16 value from 2^127 on, in blocks of their own and with smaller ones
    before and after them in the block; infinities and NaN beside them are NaN."""
    kv, ref = make(hip, None, 1, 3, 2, False), Cache(1, 3, 2)
    big = np.arange(0x7f00, 0x7f80).astype(np.uint16)
    x = np.concatenate((big, big | 0x8000))[None].repeat(64, 0)                    # [64][256]
    small = R.bf16(np.random.default_rng(7).normal(size=(64, R.D)) * 2.0 ** np.arange(60, 124).repeat(R.D).reshape(64, R.D))
    wild = x[:3].copy()
    wild[:, ::5], wild[:, 1::7] = 0x7f80, 0xffc0
    for row, pieces in enumerate(([x], [small[:9], x[:1], small[9:30], x[:12], small[:10]], [x[:5], wild, small[:40]])):
        pos = 0
        for p in pieces:
            hip.kv8_append(kv, None, cum([0] * row + [len(p)] + [0] * (2 - row)), [pos if r == row else 0 for r in range(3)],
                           dev(p), dev(p[::-1].copy()))
            ref.append(row, pos, p, p[::-1])
            pos += len(p)
        check_row(hip, kv, ref, row, 0, pos)
    assert np.abs(ref.values(0, 0, 64)[0]).max() == TOP


def huge(rng, shape, small=0.0):
    """Values of both signs from 2^120 to bf16's largest; a share of them near 1."""
    x = rng.choice([-1.0, 1.0], shape) * 2.0 ** rng.uniform(120.0, 127.99, shape)
    return R.bf16(np.where(rng.random(shape) < small, rng.normal(size=shape), x))


BATCHES = {
    "decode": [([100, 900], [1, 2]), ([0, 1, 40], [4, 3, 1]), ([7000], [3]), ([30000], [1])],
    "prefill": [([0], [40]), ([64, 3], [33, 70]), ([5000], [20])],
}


@pytest.mark.parametrize("f,ctx,new", [(f, *b) for f in BATCHES for b in BATCHES[f]])
@pytest.mark.parametrize("kind", ["same sign", "both", "some blocks", "rising scores", "tiny"])
def test_sums_of_large_and_tiny_v(hip, f, ctx, new, kind):
    """y is a mean of v whatever v's size: no sum on the way leaves fp32."""
    s = Setup(hip, 130 + len(ctx) + new[-1], 2, ctx, new, True)
    rng = np.random.default_rng(3)
    s.v = huge(rng, s.v.shape)
    if kind == "same sign":
        s.v &= 0x7fff
    elif kind == "some blocks":
        calm = np.arange(len(s.v)) // 64 % 3 > 0           # (most blocks have values near 1 alone)
        s.v[calm] = R.bf16(rng.normal(size=(int(calm.sum()), s.v.shape[1])))
    elif kind == "rising scores":
        s.v &= 0x7fff
        up = np.linspace(0.1, 6.0, len(s.k))[:, None]
        s.k = R.bf16(R.f64(s.k) * up)
    elif kind == "tiny":
        s.v = R.bf16(rng.normal(size=s.v.shape) * 2.0 ** -110)
    refill(s)
    s.check(s.call(getattr(hip, f"attn_{f}_kv8")))


def test_sums_of_large_v_many_tokens(hip):
    """The same with tiles of 32 tokens."""
    rng = np.random.default_rng(19)
    B = 160
    s = Setup(hip, 131, 2, rng.integers(0, 200, B), rng.integers(5, 75, B), True)
    s.v = huge(rng, s.v.shape, 0.3)
    refill(s)
    s.check(s.call(hip.attn_prefill_kv8), range(3, B, 31))


@pytest.mark.parametrize("f", ["attn_decode_kv8", "attn_prefill_kv8"])
@pytest.mark.parametrize("value", [0x7f7f, 0xff78, 0x7f77])
def test_large_v_of_a_later_token(hip, f, value):
    """A value at the end of bf16's range in a position that earlier tokens do not
    attend to: their rows are means of what they see."""
    s = Setup(hip, 137, 2, [61, 40], [4, 4] if f == "attn_decode_kv8" else [12, 9], False)
    n = s.ctx + s.new
    c = cum(n)
    for i in range(2):
        s.v[c[i + 1] - 1, 5::9] = value
    refill(s)
    y = s.call(getattr(hip, f))
    s.check(y)
    assert np.isfinite(R.f64(y)).all()


def test_layer_refused_before_its_scratch(hip):
    """The layer call on an 8-bit cache refuses a bad batch before it takes scratch
    for so many tokens, and a bad workspace or cache where there are no tokens."""
    m = Model(hip, 7)
    T = 40000                              # (0.65 GB of q rows, were it to go on)
    ln, ao = empty(T, H).zero_(), empty(T, H).zero_()
    call = lambda cu, pos, rows=None, work=m.work, kv=m.kv: hip.attn_layer_decode_kv8(               # noqa: E731
        m.layer, m.proj, work, rows, cu, pos, ln[:cu[-1]], kv, ao[:cu[-1]])
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for cu, pos, rows, match in (([0, T], [0], [m.rows[0]], "overflows"), ([0, T // 2, T], [0, 0], m.rows[:2], "overflows"),
                                 ([0] + [MAX * 32 * i for i in range(1, 5)], [0] * 4, m.rows, "0..4 new"),
                                 ([0, 1], [MAX * 32], [m.rows[0]], "overflows")):
        with pytest.raises(hip.ApusHipError, match=match):
            call(cu, pos, rows)
    assert torch.cuda.mem_get_info()[0] == free
    gone = hip.AttnKv8Work(m.layer, 4, 64)
    gone.destroy()
    bad = m.pool.cache(0)
    bad.scale = None
    for cu, pos in (([0], []), ([0, 0], [0])):
        call(cu, pos, m.rows[:len(pos)])
        with pytest.raises(hip.ApusHipError, match="workspace"):
            call(cu, pos, m.rows[:len(pos)], work=gone)
        with pytest.raises(hip.ApusHipError, match="descriptor"):
            call(cu, pos, m.rows[:len(pos)], kv=bad)
    torch.cuda.synchronize()
    assert not ao.any()
    for w in (m.work, m.mwork, m.pool):
        w.destroy()


def test_layer_operands_apart_from_the_cache(hip):
    """ln1 and ao may not lie in the cache's arrays, nor ao in its block table."""
    m = Model(hip, 8)
    t, blocks = table(np.random.default_rng(1), 4, 512)    # (8 KiB: two rows of ao)
    kv = hip.kv8_cache(m.kv.nkv, blocks, 512, block_table=t)
    cu, pos = [0, 1, 2], [0, 0]
    ln, ao = empty(2, H).zero_(), empty(2, H).zero_()
    k, v, scale = (x.view(torch.int16).flatten()[:2 * H].view(2, H) for x in kv._tensors[:3])
    over = t.view(torch.int16).flatten()[-2 * H:].view(2, H)
    before = [x.clone().view(torch.uint8) for x in kv._tensors]
    for args in ((k, ao), (v, ao), (scale, ao), (ln, k), (ln, v), (ln, scale), (ln, over)):
        with pytest.raises(hip.ApusHipError, match="overlap"):
            hip.attn_layer_decode_kv8(m.layer, m.proj, m.work, [0, 1], cu, pos, args[0], kv, args[1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, kv._tensors))
    hip.attn_layer_decode_kv8(m.layer, m.proj, m.work, [0, 1], cu, pos, ln, kv, ao)
    for w in (m.work, m.mwork, m.pool):
        w.destroy()


# Prefill's own kernels (calls of up to 4 tokens a sequence are decode's): tiles of 16
# tokens, the same with the keys in parts, tiles of 32 (work for every CU many times
# over; a few sequences are checked)
def prefill_batch(hip, kind, seed, **kw):
    if kind == "tiles of 32":
        rng = np.random.default_rng(29)
        ctx, new = rng.integers(0, 200, 160), rng.integers(5, 75, 160)
        ctx[:3], new[:3] = [0, 31, 200], [70, 33, 5]
        return Setup(hip, seed, 2, ctx, new, True, **kw), [0, 1, 2, 80, 159]
    ctx, new = ([37, 0], [5, 40]) if kind == "tiles of 16" else ([9000, 0], [6, 5])
    return Setup(hip, seed, 2, ctx, new, True, **kw), None


def prefill_call(s, kind):
    """The call, having run the kernels that the batch is for."""
    s.hip.timing_enable(True)
    try:
        y = s.call(s.hip.attn_prefill_kv8)
        ran = [s.hip.timing_get(n)[1] for n in ("k_kv8_fa", "k_kv8_fa_combine", "k_kv8_attn")]
    finally:
        s.hip.timing_enable(False)
    assert ran == [1, int(kind == "parts"), 0]
    return y


KERNELS = ["tiles of 16", "parts", "tiles of 32"]


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("q,k", [(0.0, 0.0), (2.0 ** -126, 0.0), (2.0 ** -126, 2.0 ** -133), (1.0, 0.0), (2.0 ** -126, 1.0),
                                 (0.0, 1.0), (1.0, 2.0 ** 100)])
def test_prefill_tiny_and_large_rows(hip, kind, q, k):
    """Rows of zeros and of the smallest values: every key counts the same, masked
    ones not at all; and k so large that one key has it all."""
    s, picks = prefill_batch(hip, kind, 151)
    rows = s.qg.reshape(-1, 2 * R.D)
    rows[:, :R.D] = R.bf16(R.f64(rows[:, :R.D]) * q)
    s.k = R.bf16(R.f64(s.k) * k)
    refill(s)
    s.check(prefill_call(s, kind), picks)


@pytest.mark.parametrize("kind", KERNELS)
def test_prefill_growing_scores(hip, kind):
    """Scores that rise along the context, far past the first keys': the reference
    point moves, and what was summed with it."""
    s, picks = prefill_batch(hip, kind, 157, spread=0.1)
    c = cum(s.ctx + s.new)
    up = np.concatenate([np.linspace(0.1, 40.0, int(n)) for n in np.diff(c)])[:, None]
    s.k = R.bf16(R.f64(s.k) * up)
    refill(s)
    s.check(prefill_call(s, kind), picks)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("what", ["k", "v"])
def test_prefill_nan_reaches_only_those_that_see_it(hip, kind, what):
    """A NaN and an infinity in a new token's k or v: rows before it are as without
    it; rows that see a NaN k are NaN, those that see NaN v are NaN in that dim."""
    s, picks = prefill_batch(hip, kind, 163)
    q = 0                                  # of the sequence: its third new token; head 1, dims 44 and 45
    c = cum(s.ctx + s.new)
    at, first, end = c[q] + s.ctx[q] + 2, s.cu[q] + 2, s.cu[q + 1]
    x = s.k if what == "k" else s.v
    x[at, 300], x[at, 301] = 0x7fc0, 0xff80
    refill(s)
    y = prefill_call(s, kind)
    bad = np.zeros(y.shape, bool)
    bad[first:end, 8:16, slice(44, 46) if what == "v" else slice(None)] = True
    got = R.f64(y)
    assert np.array_equal(np.isnan(got), bad)
    x[at, 300:302] = 0                     # (does not count in the block's scale, as these do not)
    refilled = Cache(2, len(s.ctx), s.max_blocks)
    for i in picks or range(len(s.ctx)):
        refilled.append(s.row(i), 0, s.k[c[i]:c[i + 1]], s.v[c[i]:c[i + 1]])
    s.ref = refilled
    s.check(y, [i for i in picks or range(len(s.ctx)) if i != q])
    k, v = refilled.values(s.row(q), 0, int(s.ctx[q] + s.new[q]))
    r, tol = R.attention(s.qg[s.cu[q]:end], s.w["qn_w"], int(s.ctx[q]), k, v, 1e7)
    ok = ~bad[s.cu[q]:end]
    assert (np.abs(got[s.cu[q]:end] - r) <= tol)[ok].all()
