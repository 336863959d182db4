"""GPU parity at the edges of the MXFP4 products, within the bound of fp32
accumulation and one bf16 rounding: K taken in two halves side by side (tiles of
128 x 128, at most one a CU), and tiles of the few-row form with nothing in them."""
import pytest

import mx_ref

pytestmark = pytest.mark.gpu


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _bytes_at_end(torch, t):
    """t as the last bytes of a buffer of its own."""
    b = torch.empty(t.numel() + 240, dtype=torch.uint8, device="cuda")
    v = b[240:].view(t.shape)
    assert v.data_ptr() % 16 == 0
    return v.copy_(t)


def _product(hip, torch, w, ws, x, mx):
    """y of the call, and the values of the activations it stands for."""
    y = torch.empty(x.shape[0], w.shape[0], dtype=torch.bfloat16, device="cuda")
    if not mx:
        hip.mxfp4_gemm(w, ws, x, y)
        return y, x.double()
    c = torch.empty(x.shape[0], x.shape[1] // 2, dtype=torch.uint8, device="cuda")
    s = torch.empty(x.shape[0], x.shape[1] // 32, dtype=torch.uint8, device="cuda")
    hip.mxfp4_quantize(x, c, s)
    hip.mxfp4_gemm_mx(w, ws, c, _bytes_at_end(torch, s), y)
    return y, mx_ref.values(c, s)


# the second half's scales begin at byte 8 of rows of 16 (K = 512), or off 16 bytes
@pytest.mark.parametrize("M,O,K", [(512, 4096, 512), (640, 4090, 512), (513, 8190, 512), (1024, 2048, 512),
                                   (1000, 4090, 1536), (2040, 2048, 1536), (1000, 4096, 2560)])
@pytest.mark.parametrize("mx", [False, True])
def test_scales_of_the_second_half(hip, M, O, K, mx):
    import torch
    print(f"[mx] halves M={M} O={O} K={K} mx={mx}", flush=True)
    g = _gen(torch, M + O + K)
    x = mx_ref.normal(g, M, K)
    w, ws = mx_ref.quantize(mx_ref.normal(g, O, K, scale=K ** -0.5))
    # (each block of a scale of its own)
    ws = ws - 8 + torch.randint(0, 17, ws.shape, generator=g, device="cuda").to(torch.uint8)
    ws = _bytes_at_end(torch, ws)
    y, xv = _product(hip, torch, w, ws, x, mx)
    r, b = mx_ref.gemm(mx_ref.values(w, ws), xv)
    mx_ref.check(y, r, b, f"halves mx={mx}")


# outputs that end before the second (2 x 16 a workgroup) or before one of the last
# tiles (4 x 16), rows before the last of 3 or 4 tiles; K of many steps
@pytest.mark.parametrize("M,O,K", [(3, 8200, 4128), (30, 12353, 2080), (65, 130, 4096), (97, 517, 2208),
                                   (60, 12305, 2080), (113, 8211, 1056), (129, 40, 1568)])
@pytest.mark.parametrize("mx", [False, True])
def test_tiles_with_nothing_in_them(hip, M, O, K, mx):
    import torch
    print(f"[mx] empty tiles M={M} O={O} K={K} mx={mx}", flush=True)
    g = _gen(torch, M + O + K)
    x = mx_ref.normal(g, M, K)
    w, ws = mx_ref.quantize(mx_ref.normal(g, O, K, scale=K ** -0.5))
    y, xv = _product(hip, torch, _bytes_at_end(torch, w), _bytes_at_end(torch, ws), x, mx)
    r, b = mx_ref.gemm(mx_ref.values(w, ws), xv)
    mx_ref.check(y, r, b, f"empty tiles mx={mx}")


# K that ends in the middle of a stage, the stages odd in number: one half has a stage
# less than the other, and what it brings past its end counts nowhere
HALVES = [(513, 4104, 288), (900, 2050, 544), (513, 4100, 160), (1000, 4090, 2080), (700, 4096, 1056),
          (513, 4104, 320), (1000, 4090, 2112)]


@pytest.mark.parametrize("M,O,K", HALVES)
@pytest.mark.parametrize("mx", [False, True])
def test_halves_smallest_scales(hip, M, O, K, mx):
    """Weight scales 2^-127 .. 2^-125: what is no part of the sum shows at any scale."""
    import torch
    print(f"[mx] halves, smallest scales M={M} O={O} K={K} mx={mx}", flush=True)
    g = _gen(torch, M + K)
    w, _ = mx_ref.quantize(mx_ref.normal(g, O, K))
    ws = torch.randint(0, 3, (O, K // 32), generator=g, device="cuda").to(torch.uint8)
    x = mx_ref.normal(g, M, K, scale=2.0 ** 115)
    y, xv = _product(hip, torch, w, ws, x, mx)
    r, b = mx_ref.gemm(mx_ref.values(w, ws), xv)
    mx_ref.check(y, r, b, f"halves, smallest scales mx={mx}")


# (beside the halves: few rows, with 16, 32 and 64 outputs a workgroup, and tiles of 128 x 128, of
# 256 x 128 and of 256 x 256, also with the last of them in quarters)
@pytest.mark.parametrize("M,O,K", HALVES + [(3, 40, 96), (4, 8200, 160), (60, 12305, 160), (300, 2500, 288),
                                            (2050, 2049, 160), (2300, 6001, 544), (2048, 8192, 1056),
                                            (4100, 4090, 1056), (4090, 4100, 4128)])
def test_infinities(hip, M, O, K):
    """One infinite activation a row, in every place of it: y is infinite with the sign
    of its weight, NaN where that is zero."""
    import torch
    print(f"[mx] infinities M={M} O={O} K={K}", flush=True)
    g = _gen(torch, M + K)
    w, ws = mx_ref.quantize(mx_ref.normal(g, O, K, scale=K ** -0.5))
    x = mx_ref.normal(g, M, K)
    at = torch.arange(M, device="cuda")
    for first in (0, K // 2, K - min(M, K)):
        xi = x.clone()
        xi[at, (first + at) % K] = float("inf")
        y, _ = _product(hip, torch, w, ws, xi, False)
        wv = mx_ref.values(w, ws)[:, (first + at) % K].t()
        assert torch.equal(y.isnan(), wv == 0)
        assert torch.equal(y == float("inf"), wv > 0) and torch.equal(y == -float("inf"), wv < 0)
