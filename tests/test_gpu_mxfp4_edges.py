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
