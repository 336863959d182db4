"""The 8-bit KV cache and attention over it, plainly and in 64 bits: what the
GPU tests compare with. numpy only."""
import numpy as np

D, BLK, ROT, GRP = 256, 32, 64, 8
EMIN = -117
U = 2.0 ** -8                              # half a step of bf16, relative
# e4m3 magnitudes by code (0x7f is NaN)
MAGS = np.array([m * 2.0 ** -9 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7) for e in range(16) for m in range(8)])
MAGS[127] = np.nan


def f64(codes):
    """bf16 codes (uint16) as float64."""
    with np.errstate(invalid="ignore"):
        return (np.asarray(codes, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def bf16(x):
    """float64 to bf16 codes, one rounding to nearest even."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        e = np.floor(np.log2(np.where((x == 0) | ~np.isfinite(x), 1.0, np.abs(x))))
        e = np.where(np.abs(x) < 2.0 ** e, e - 1, e)       # (log2 rounded up)
        step = 2.0 ** (np.maximum(e, -126) - 7)
        r = np.where(np.isfinite(x), np.rint(x / step) * step, x)
        f = r.astype(np.float32)
    return (f.view(np.uint32) >> 16).astype(np.uint16)


def e4m3(x):
    """float64 (magnitudes up to 448) to e4m3 codes: nearest, ties to the even code."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    mid = (MAGS[1:127] + MAGS[:126]) / 2
    c = np.searchsorted(mid, a, side="left")               # mid[c-1] < a <= mid[c]
    tie = (c < 126) & (a == mid[np.minimum(c, 125)]) & (c % 2 == 1)
    c = np.where(tie, c + 1, c)
    c = np.where(np.isfinite(x), c, 127)
    return (c | (np.signbit(x).astype(np.int64) << 7)).astype(np.uint8)


def value(c):
    return np.where(c & 0x80, -1.0, 1.0) * MAGS[c & 0x7f]


def exponent(x, axes):
    """Smallest e >= EMIN with amax <= 448 2^e over the finite values."""
    a = np.where(np.isfinite(x), np.abs(x), 0.0).max(axes)
    e = np.full(a.shape, EMIN)
    while (a > 448.0 * 2.0 ** e).any():
        e = np.where(a > 448.0 * 2.0 ** e, e + 1, e)
    return e


class Cache:
    """rows: {row: (codes [positions][nkv][2][D], exponents [blocks][nkv][2])}."""

    def __init__(self, nkv, rows, max_blocks):
        self.nkv = nkv
        self.codes = np.zeros((rows, max_blocks * BLK, nkv, 2, D), np.uint8)
        self.exps = np.full((rows, max_blocks, nkv, 2), EMIN)

    def append(self, row, pos0, k, v):
        """k, v [n][nkv * D] bf16 codes."""
        x = np.stack((f64(k).reshape(-1, self.nkv, D), f64(v).reshape(-1, self.nkv, D)), 2)
        for b in range(pos0 // BLK, -(-(pos0 + len(x)) // BLK) if len(x) else 0):
            lo, hi = max(pos0, b * BLK), min(pos0 + len(x), (b + 1) * BLK)
            new = x[lo - pos0:hi - pos0]
            e = exponent(new, (0, 3))
            if lo > b * BLK:
                old = self.codes[row, b * BLK:lo]
                e = np.maximum(e, self.exps[row, b])
                up = self.exps[row, b] - e
                self.codes[row, b * BLK:lo] = e4m3(value(old) * (2.0 ** up)[..., None])
            self.exps[row, b] = e
            self.codes[row, lo:hi] = e4m3(new * (2.0 ** -e.astype(float))[..., None])

    def values(self, row, p0, p1):
        """(k, v) [p1 - p0][nkv][D] in float64."""
        e = self.exps[row].repeat(BLK, 0)[p0:p1].astype(float)
        x = value(self.codes[row, p0:p1]) * (2.0 ** e)[..., None]
        return x[:, :, 0], x[:, :, 1]


def rope_tab(pos, theta):
    """cos, sin [n][ROT/2] as the model keeps them: of the fp32 angle, in bf16."""
    inv = (1.0 / theta ** (2.0 * np.arange(ROT // 2) / ROT)).astype(np.float32)
    a = (np.asarray(pos, np.float32)[:, None] * inv).astype(np.float64)
    r = lambda t: f64(bf16(t.astype(np.float32).astype(np.float64)))     # noqa: E731
    return r(np.cos(a)), r(np.sin(a))


def rope(x, pos, theta):
    """x [n][heads][D] float64."""
    c, s = (t[:, None] for t in rope_tab(pos, theta))
    a, b = x[..., :ROT // 2], x[..., ROT // 2:ROT]
    return np.concatenate((a * c - b * s, b * c + a * s, x[..., ROT:]), -1)


def q_rows(q, w, pos, theta, eps=1e-6):
    """q codes [n][nh][D] after norm and RoPE, not rounded."""
    x = f64(q)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + f64(w))
    return rope(x, pos, theta)


def attention(qg, w, pos0, k, v, theta):
    """One sequence: qg [n][nh][2D] codes at positions pos0 ..., k, v [>= pos0 + n]
    [nkv][D] float64. Returns y [n][nh][D] and its bound.

    q's rounding to fp16: half a step, 2^-11 of an element, or of 2^-20 of the row's
    largest m (which lies at 2^6 or above, an element below 2^-14 at steps of
    2^-24), so a score is off by 2^-11 a_j, a_j = sum_d max(|q_d|, 2^-20 m) |K_jd| /
    16, and a probability by the factors of its own and of the sum of all.
    The probabilities' rounding: p_j (1 + d_j), |d_j| <= U, for the product with V
    and for their sum, y' = sum p_j (1 + d_j) v_j / sum p_j (1 + d_j) = y + sum p_j
    d_j (v_j - y) / sum p_j (1 + d_j): U / (1 - U) sum_j p_j |v_j - y|.
    fp32 arithmetic: 2^-10 of the terms is far more than it makes (scores of some
    20 with 256 terms of 2^-24; exponents of 1 ulp). And the rounding of y."""
    n, nh = qg.shape[:2]
    nkv = k.shape[1]
    q = q_rows(qg[..., :D], w, pos0 + np.arange(n), theta)
    y, tol = np.zeros((n, nh, D)), np.zeros((n, nh, D))
    sig = 1.0 / (1.0 + np.exp(-f64(qg[..., D:])))
    for t in range(n):
        m = pos0 + t + 1
        for h in range(nkv):
            hs = slice(h * GRP, (h + 1) * GRP)
            s = q[t, hs] @ k[:m, h].T / 16.0
            qa = np.abs(q[t, hs])
            a = np.maximum(qa, 2.0 ** -20 * qa.max(-1, keepdims=True)) @ np.abs(k[:m, h]).T / 16.0
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            e = 2.0 ** -11 * (a + (p * a).sum(-1, keepdims=True))
            y[t, hs] = p @ v[:m, h]
            with np.errstate(over="ignore", invalid="ignore"):
                move = np.fmin(p * np.expm1(e), 1.0)       # (between 0 and 1 it cannot move further; 0 inf: 1)
            tol[t, hs] = (p * 2.0 ** -10 + move) @ np.abs(v[:m, h])
            for i in range(GRP):
                tol[t, h * GRP + i] += U / (1 - U) * (p[i] @ np.abs(v[:m, h] - y[t, h * GRP + i]))
    y *= sig
    tol = tol * sig + U * np.abs(y)
    return y, tol * (1 + U) + 2.0 ** -133
