"""GPU parity: MXFP4 quantisation (bit for bit) and products (within the
bound that fp32 accumulation and one bf16 rounding allow) against plain
64-bit implementations."""
import pytest

import mx_ref

pytestmark = pytest.mark.gpu


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _quantize(hip, torch, x):
    M, K = x.shape
    c = torch.full((M, K // 2), 0xAA, dtype=torch.uint8, device="cuda")
    s = torch.full((M, K // 32), 0xAA, dtype=torch.uint8, device="cuda")
    hip.mxfp4_quantize(x, c, s)
    return c, s


@pytest.mark.parametrize("M,K,pad", [(1, 32, 0), (1, 2048, 0), (3, 96, 8), (37, 4096, 72),
                                     (1000, 160, 0), (2049, 1056, 24), (20000, 32, 0)])
def test_quantize(hip, M, K, pad):
    import torch
    print(f"[mx] quantize M={M} K={K} pad={pad}", flush=True)
    g = _gen(torch, M + K)
    wide = mx_ref.normal(g, M, K + pad)
    wide *= torch.exp2(torch.randint(-20, 21, (M, 1), generator=g, device="cuda")).to(torch.bfloat16)
    x = wide[:, pad:]
    c, s = _quantize(hip, torch, x)
    rc, rs = mx_ref.quantize(x)
    assert torch.equal(s, rs) and torch.equal(c, rc)
    buf = torch.full((M, K + pad), 7.0, dtype=torch.bfloat16, device="cuda")
    hip.mxfp4_dequantize(c, s, buf[:, pad:])
    assert torch.equal(buf[:, pad:].double(), mx_ref.values(c, s))
    assert bool((buf[:, :pad] == 7.0).all())


def test_quantize_every_code(hip):
    """Every bf16 code at the position that sets its block's scale, and below
    block maxima of every exponent: subnormals, both zeros, the smallest and
    largest scales, infinities and NaN."""
    import torch
    codes = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16)
    x = torch.zeros(65536, 32, dtype=torch.int16, device="cuda")
    x[:, 5] = codes
    x[:, 6] = 1                                            # the smallest subnormal
    lead = torch.arange(256, device="cuda") << 7           # 2^(e - 127), 0 and infinity
    y = torch.zeros(256, 256, 32, dtype=torch.int16, device="cuda")
    y[:, :, 0] = lead.to(torch.int16)[:, None]
    y[:, :, 1:] = (torch.arange(256 * 31, device="cuda").view(1, 256, 31) * 2115 % 65536).to(torch.int16)
    for t in (x, y.view(-1, 32)):
        v = t.view(torch.bfloat16)
        c, s = _quantize(hip, torch, v)
        rc, rs = mx_ref.quantize(v)
        assert torch.equal(s, rs)
        assert torch.equal(c, rc)


def test_dequantize_every_scale(hip):
    import torch
    s = torch.arange(256, device="cuda", dtype=torch.int32).to(torch.uint8).view(256, 1)
    c = (torch.arange(16, device="cuda") | (torch.arange(16, device="cuda").flip(0) << 4))
    c = c.to(torch.uint8).repeat(256, 1)
    x = torch.empty(256, 32, dtype=torch.bfloat16, device="cuda")
    hip.mxfp4_dequantize(c, s, x)
    assert torch.equal(torch.nan_to_num(x.double(), nan=1.5),
                       torch.nan_to_num(mx_ref.values(c, s).to(torch.bfloat16).double(), nan=1.5))


# one row to many, row and output counts off every tile, K of one block, of a
# part of a step, of many steps; slices of wider buffers on both sides
SHAPES = [(1, 12352, 2048, 0, 0), (1, 1, 32, 0, 0), (2, 17, 96, 8, 3), (15, 517, 160, 0, 0),
          (16, 64, 128, 8, 8), (17, 2048, 4096, 64, 0), (37, 33, 2080, 0, 1), (64, 2048, 4096, 0, 0),
          (65, 130, 544, 8, 0), (130, 1000, 288, 0, 24), (257, 300, 1056, 40, 1),
          (300, 4160, 2048, 0, 0), (1025, 513, 96, 0, 0), (2300, 1100, 64, 0, 0),
          (1500, 2112, 1088, 8, 8), (640, 12352, 512, 0, 0), (4096, 516, 32, 0, 0)]


def _operands(torch, M, O, K, px, seed):
    g = _gen(torch, seed)
    x = mx_ref.normal(g, M, K + px)[:, px:]
    w, ws = mx_ref.quantize(mx_ref.normal(g, O, K, scale=K ** -0.5))
    return x, w, ws


@pytest.mark.parametrize("M,O,K,px,py", SHAPES)
def test_gemm(hip, M, O, K, px, py):
    import torch
    print(f"[mx] gemm M={M} O={O} K={K} px={px} py={py}", flush=True)
    x, w, ws = _operands(torch, M, O, K, px, M * 7 + O + K)
    buf = torch.full((M + 1, O + py), 7.0, dtype=torch.bfloat16, device="cuda")
    y = buf[:M, py:]
    hip.mxfp4_gemm(w, ws, x, y)
    r, b = mx_ref.gemm(mx_ref.values(w, ws), x.double())
    mx_ref.check(y, r, b, "gemm")
    assert bool((buf[:, :py] == 7.0).all()) and bool((buf[M] == 7.0).all())


@pytest.mark.parametrize("M,O,K,px,py", SHAPES)
def test_gemm_mx(hip, M, O, K, px, py):
    import torch
    print(f"[mx] gemm_mx M={M} O={O} K={K} py={py}", flush=True)
    x, w, ws = _operands(torch, M, O, K, px, M * 5 + O + K)
    c, s = _quantize(hip, torch, x)
    buf = torch.full((M + 1, O + py), 7.0, dtype=torch.bfloat16, device="cuda")
    y = buf[:M, py:]
    hip.mxfp4_gemm_mx(w, ws, c, s, y)
    r, b = mx_ref.gemm(mx_ref.values(w, ws), mx_ref.values(c, s))
    mx_ref.check(y, r, b, "gemm_mx")
    assert bool((buf[:, :py] == 7.0).all()) and bool((buf[M] == 7.0).all())


@pytest.mark.parametrize("M,O,K", [(3, 40, 192), (200, 700, 320), (1100, 1300, 192)])
@pytest.mark.parametrize("mx", [False, True])
def test_gemm_wide_range(hip, M, O, K, mx):
    """Scales from 2^-40 to 2^40 in weights and activations: a block's scale
    meets its own elements only."""
    import torch
    g = _gen(torch, M + O)
    pw = torch.exp2(torch.randint(-40, 41, (O, K // 32), generator=g, device="cuda")).repeat_interleave(32, 1)
    w, ws = mx_ref.quantize((torch.randn(O, K, generator=g, device="cuda") * pw).to(torch.bfloat16))
    pxs = torch.exp2(torch.randint(-40, 41, (M, K // 32), generator=g, device="cuda")).repeat_interleave(32, 1)
    x = (torch.randn(M, K, generator=g, device="cuda") * pxs).to(torch.bfloat16)
    y = torch.empty(M, O, dtype=torch.bfloat16, device="cuda")
    if mx:
        c, s = _quantize(hip, torch, x)
        hip.mxfp4_gemm_mx(w, ws, c, s, y)
        xv = mx_ref.values(c, s)
    else:
        hip.mxfp4_gemm(w, ws, x, y)
        xv = x.double()
    r, b = mx_ref.gemm(mx_ref.values(w, ws), xv)
    mx_ref.check(y, r, b, f"wide range mx={mx}")


@pytest.mark.parametrize("M,O,K", [(5, 70, 160), (300, 600, 160), (1100, 1300, 160)])
@pytest.mark.parametrize("mx", [False, True])
def test_gemm_nan_rows(hip, M, O, K, mx):
    """A NaN in one activation row and a NaN block in one weight row spoil
    that row and that column of y, nothing else."""
    import torch
    x, w, ws = _operands(torch, M, O, K, 0, M)
    x = x.contiguous()
    y0, y1 = (torch.empty(M, O, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def run(x, ws, y):
        if mx:
            hip.mxfp4_gemm_mx(w, ws, *_quantize(hip, torch, x), y)
        else:
            hip.mxfp4_gemm(w, ws, x, y)

    run(x, ws, y0)
    xb, wb = x.clone(), ws.clone()
    xb[M - 1, K - 3] = float("nan")
    wb[O - 1, 1] = 255
    run(xb, wb, y1)
    assert bool(y1[M - 1].isnan().all()) and bool(y1[:, O - 1].isnan().all())
    assert torch.equal(y1[:M - 1, :O - 1], y0[:M - 1, :O - 1])


def test_empty_calls(hip):
    """No rows, no outputs: nothing is written. K = 0: zeros."""
    import torch
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")
    bf = lambda *s: torch.full(s, 7.0, dtype=torch.bfloat16, device="cuda")
    hip.mxfp4_quantize(bf(0, 64), u8(0, 32), u8(0, 2))
    hip.mxfp4_quantize(bf(3, 0), u8(3, 0), u8(3, 0))
    hip.mxfp4_dequantize(u8(0, 32), u8(0, 2), bf(0, 64))
    hip.mxfp4_gemm(u8(5, 32), u8(5, 2), bf(0, 64), bf(0, 5))
    hip.mxfp4_gemm(u8(0, 32), u8(0, 2), bf(4, 64), bf(4, 0))
    hip.mxfp4_gemm_mx(u8(5, 32), u8(5, 2), u8(0, 32), u8(0, 2), bf(0, 5))
    y = bf(4, 9)
    hip.mxfp4_gemm(u8(5, 0), u8(5, 0), bf(4, 0), y[:, 2:7])
    assert not bool(y[:, 2:7].any()) and bool((y[:, :2] == 7).all()) and bool((y[:, 7:] == 7).all())


@pytest.mark.parametrize("M,O,K", [(4, 256, 512), (700, 1100, 256)])
def test_graph_replays(hip, M, O, K):
    """Quantise and multiply, captured on a stream of their own and replayed
    with other activations, with eager work between the replays."""
    import torch
    st = torch.cuda.Stream()
    x, w, ws = _operands(torch, M, O, K, 0, 3)
    x = x.contiguous()
    c = torch.empty(M, K // 2, dtype=torch.uint8, device="cuda")
    s = torch.empty(M, K // 32, dtype=torch.uint8, device="cuda")
    y, z, e = (torch.empty(M, O, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    st.wait_stream(torch.cuda.current_stream())
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            hip.set_stream(torch.cuda.current_stream().cuda_stream)
            hip.mxfp4_quantize(x, c, s)
            hip.mxfp4_gemm_mx(w, ws, c, s, y)
            hip.mxfp4_gemm(w, ws, x, z)
    finally:
        hip.set_stream(0)
    for i in range(4):
        x.copy_(mx_ref.normal(_gen(torch, 50 + i), M, K))
        graph.replay()
        torch.cuda.synchronize()
        hip.mxfp4_gemm(w, ws, x, e)
        assert torch.equal(z, e)
        ec, es = _quantize(hip, torch, x)
        hip.mxfp4_gemm_mx(w, ws, ec, es, e)
        assert torch.equal(c, ec) and torch.equal(s, es) and torch.equal(y, e)


def test_python_refusals(hip):
    import torch
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        hip.mxfp4_quantize(bf(4, 64), u8(4, 31), u8(4, 2))             # codes of another shape
    with pytest.raises(ValueError):
        hip.mxfp4_quantize(bf(64, 4).t(), u8(4, 32), u8(4, 2))         # columns contiguous
    with pytest.raises(ValueError):
        hip.mxfp4_gemm(u8(5, 32), u8(5, 2), torch.zeros(4, 64), bf(4, 5))      # a CPU tensor
    with pytest.raises(ValueError):
        hip.mxfp4_gemm(u8(5, 32), u8(5, 2), bf(4, 64), bf(3, 5))       # rows of y
    with pytest.raises(ValueError):
        hip.mxfp4_gemm(u8(5, 32), u8(5, 2), bf(4, 96), bf(4, 5))       # another K
    with pytest.raises(ValueError):                                    # another 2-byte type
        hip.mxfp4_quantize(bf(4, 64).half(), u8(4, 32), u8(4, 2))
    with pytest.raises(ValueError):
        hip.mxfp4_gemm(u8(5, 32), u8(5, 2), bf(4, 64), bf(4, 5).half())
    with pytest.raises(hip.ApusHipError) as e:                         # not whole blocks
        hip.mxfp4_quantize(bf(4, 48), u8(4, 24), u8(4, 1))
    assert e.value.code == 1
    x = bf(4, 1).expand(4, 64).contiguous()[:1].expand(4, 64)          # rows on top of each other
    with pytest.raises(hip.ApusHipError) as e:
        hip.mxfp4_gemm(u8(5, 32), u8(5, 2), x, bf(4, 5))
    assert e.value.code == 3
    b = bf(4, 128)
    with pytest.raises(hip.ApusHipError) as e:                         # y over x
        hip.mxfp4_gemm(u8(65, 32), u8(65, 2), b[:, :64], b[:, 63:])
    assert e.value.code == 3
    hip.mxfp4_gemm(u8(64, 32), u8(64, 2), b[:, :64], b[:, 64:])        # beside x in one buffer


# the forms of the product: shapes that the estimates give to each (few rows in
# tiles of 1 to 4 x 16 with 16, 32 and 64 outputs, 128-wide tiles, also with K in two
# halves, 256-wide tiles, also with the last of them in quarters), with row, output
# and K edges in each; K past one pair of steps a wavefront, K of 4096 and more, odd
# numbers of blocks
@pytest.mark.parametrize("M,O,K", [(4, 12345, 2080), (5, 8200, 4128), (31, 9000, 96), (33, 520, 8192),
                                   (47, 20000, 224), (50, 12352, 160), (64, 4100, 2144), (100, 12360, 1056),
                                   (250, 6001, 2208), (513, 4104, 288), (2050, 2049, 4192), (4100, 4090, 8224),
                                   (2048, 8192, 4096), (900, 2050, 320), (1000, 4090, 2080), (2000, 2041, 544),
                                   (4096, 12345, 2080), (4096, 12345, 4128),
                                   (60, 12345, 2080), (120, 8190, 1056), (45, 12401, 2080)])
@pytest.mark.parametrize("mx", [False, True])
def test_gemm_forms(hip, M, O, K, mx):
    import torch
    print(f"[mx] forms M={M} O={O} K={K} mx={mx}", flush=True)
    x, w, ws = _operands(torch, M, O, K, 0, M + O + K)
    x = x.contiguous()
    y = torch.empty(M, O, dtype=torch.bfloat16, device="cuda")
    if mx:
        c, s = _quantize(hip, torch, x)
        hip.mxfp4_gemm_mx(w, ws, c, s, y)
        xv = mx_ref.values(c, s)
    else:
        hip.mxfp4_gemm(w, ws, x, y)
        xv = x.double()
    r, b = mx_ref.gemm(mx_ref.values(w, ws), xv)
    mx_ref.check(y, r, b, f"forms mx={mx}")


@pytest.mark.parametrize("M,O,K", [(3, 40, 192), (200, 700, 320), (1100, 1300, 192), (4096, 2048, 1024)])
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("lo", [0, 247])
def test_gemm_ends_of_the_scales(hip, M, O, K, mx, lo):
    """Weight scales 2^-127 .. 2^-120, whose values and bf16 forms are subnormal
    or next to it, and 2^120 .. 2^127, with activations that bring the products
    back into range. A weight of 2^128 and more is infinite where it meets bf16
    activations, as it is for mxfp4_dequantize."""
    import torch
    g = _gen(torch, M + O + lo)
    w, _ = mx_ref.quantize(mx_ref.normal(g, O, K))
    ws = (torch.randint(lo, lo + 8, (O, K // 32), generator=g, device="cuda")).to(torch.uint8)
    x = (torch.randn(M, K, generator=g, device="cuda") * 2.0 ** (110 if lo == 0 else -115)).to(torch.bfloat16)
    y = torch.empty(M, O, dtype=torch.bfloat16, device="cuda")
    if mx:
        c, s = _quantize(hip, torch, x)
        hip.mxfp4_gemm_mx(w, ws, c, s, y)
        xv = mx_ref.values(c, s)
    else:
        hip.mxfp4_gemm(w, ws, x, y)
        xv = x.double()
    wv = mx_ref.values(w, ws)
    if not mx:                                             # (past bf16's range: infinite)
        wv = wv.to(torch.bfloat16).double()
    r, b = mx_ref.gemm(wv, xv)
    fin = r.isfinite()
    assert torch.equal(y.isnan(), r.isnan()) and torch.equal(y[r.isinf()].double(), r[r.isinf()])
    assert mx or lo == 0 or not bool(fin.all())
    mx_ref.check(y[fin], r[fin], b[fin], f"ends of the scales mx={mx}")


@pytest.mark.parametrize("M,O,K", [(3, 40, 192), (300, 520, 1056), (4096, 2300, 544)])
def test_gemm_scales_of_any_alignment(hip, M, O, K):
    import torch
    x, w, ws = _operands(torch, M, O, K, 0, M)
    x = x.contiguous()
    c, s = _quantize(hip, torch, x)
    ys = []
    for off in (0, 1, 3):
        a, b = (torch.empty(t.numel() + 4, dtype=torch.uint8, device="cuda")[off:off + t.numel()].view(t.shape).copy_(t)
                for t in (ws, s))
        y, z = (torch.empty(M, O, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        hip.mxfp4_gemm(w, a, x, y)
        hip.mxfp4_gemm_mx(w, a, c, b, z)
        ys.append((y, z))
    for y, z in ys[1:]:
        assert torch.equal(y, ys[0][0]) and torch.equal(z, ys[0][1])
    r, bound = mx_ref.gemm(mx_ref.values(w, ws), x.double())
    mx_ref.check(ys[0][0], r, bound, "alignment")
