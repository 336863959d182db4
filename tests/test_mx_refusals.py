"""CPU checks: the MXFP4 and mixture-of-experts entry points refuse bad
arguments before they look for a device (addresses here are never read), and
with APUS_HIP_DISABLE set return "disabled" whatever they are given."""
import ctypes as C
import os
import subprocess
import sys

import pytest

import apus_hip

SZ = C.c_size_t
A, B, D, E = (C.c_void_p(n << 32) for n in (1, 2, 3, 4))   # 16-byte aligned, far apart
ARG, UNS = 3, 1


def off(p, n):
    return C.c_void_p(p.value + n)


def quant(x=A, ldx=64, c=B, s=D, M=4, K=64, f="quantize"):
    lib = apus_hip.load()
    if f == "quantize":
        return lib.apus_hip_mxfp4_quantize(x, SZ(ldx), c, s, SZ(M), SZ(K))
    return lib.apus_hip_mxfp4_dequantize(c, s, x, SZ(ldx), SZ(M), SZ(K))


def gemm(w=A, ws=B, x=D, ldx=64, y=E, ldy=10, M=4, O=10, K=64):
    return apus_hip.load().apus_hip_mxfp4_gemm_dev(w, ws, x, SZ(ldx), y, SZ(ldy), SZ(M), SZ(O), SZ(K))


def gemm_mx(w=A, ws=B, x=D, xs=off(D, 1 << 20), y=E, ldy=10, M=4, O=10, K=64):
    return apus_hip.load().apus_hip_mxfp4_gemm_mx_dev(w, ws, x, xs, y, SZ(ldy), SZ(M), SZ(O), SZ(K))


@pytest.mark.parametrize("f", ["quantize", "dequantize"])
def test_quantize_refusals(f):
    assert quant(f=f, K=48) == UNS                         # not whole blocks
    assert quant(f=f, ldx=63) == ARG                       # rows on top of each other
    assert quant(f=f, ldx=68) == UNS                       # rows off 16 bytes
    assert quant(f=f, x=off(A, 8)) == UNS
    assert quant(f=f, c=off(B, 4)) == UNS
    for n in ("x", "c", "s"):
        assert quant(f=f, **{n: None}) == ARG
    assert quant(f=f, c=off(A, 16)) == ARG                 # codes inside x
    assert quant(f=f, s=off(A, 4 * 128 - 1)) == ARG
    assert quant(f=f, M=1 << 31) == UNS
    assert quant(f=f, K=(1 << 21) + 32, ldx=1 << 22) == UNS
    assert quant(f=f, M=1 << 30, ldx=1 << 21) == UNS       # past 2^40 elements
    assert quant(f=f, ldx=1 << 62) == UNS


def test_gemm_refusals():
    assert gemm(K=40) == UNS
    assert gemm(ldx=56) == ARG
    assert gemm(ldx=68) == UNS
    assert gemm(ldy=9) == ARG
    assert gemm(x=off(D, 2)) == UNS
    assert gemm(w=off(A, 8)) == UNS
    assert gemm(y=off(E, 1)) == ARG
    for n in ("w", "ws", "x", "y"):
        assert gemm(**{n: None}) == ARG
    assert gemm(O=1 << 31) == UNS
    assert gemm(K=(1 << 21) + 32, ldx=1 << 22) == UNS
    assert gemm(ldx=(1 << 21) + 8) == UNS                  # offsets past 32 bits in a tile
    assert gemm(ldy=1 << 39) == UNS and gemm(ldy=1 << 62) == UNS
    # y among x's rows: in their columns, or with another pitch
    assert gemm(ldx=128, y=off(D, 2 * 63), ldy=128) == ARG
    assert gemm(ldx=128, y=off(D, 2 * 119), ldy=128) == ARG        # wraps into the next row
    assert gemm(ldx=128, y=off(D, 2 * 64), ldy=136) == ARG
    assert gemm(ldx=128, y=C.c_void_p(D.value - 2 * 5), ldy=128) == ARG


def test_gemm_mx_refusals():
    assert gemm_mx(K=40) == UNS
    assert gemm_mx(ldy=9) == ARG
    assert gemm_mx(x=off(D, 8)) == UNS
    for n in ("w", "ws", "x", "xs", "y"):
        assert gemm_mx(**{n: None}) == ARG
    assert gemm_mx(y=off(D, 64)) == ARG
    assert gemm_mx(y=off(D, (1 << 20) + 2)) == ARG


def layer(**kw):
    d = dict(hidden=64, inter=32, experts=8, topk=2, shared_inter=0, norm_topk=1, mxfp4=0,
             w_router=A.value, w_gate_up=B.value, w_down=D.value)
    d.update(kw)
    return apus_hip.MoeLayer(**d)


def work(L, T=4, out=True):
    h = C.c_void_p()
    return apus_hip.load().apus_hip_moe_work_create(C.byref(L) if L else None, SZ(T),
                                                    C.byref(h) if out else None)


def test_moe_refusals():
    assert work(None) == ARG
    assert work(layer(), out=False) == ARG
    assert work(layer(topk=0)) == ARG and work(layer(topk=9)) == ARG and work(layer(experts=0)) == ARG
    assert work(layer(experts=1025)) == UNS and work(layer(experts=64, topk=33)) == UNS
    for n in ("hidden", "inter", "shared_inter"):
        assert work(layer(**{n: 48})) == UNS
        assert work(layer(**{n: 1 << 21})) == UNS
    assert work(layer(hidden=0)) == UNS and work(layer(inter=0)) == UNS
    assert work(layer(inter=1 << 19), T=1024) == UNS       # 4 GiB of h
    assert work(layer(hidden=1 << 20), T=1024) == UNS
    assert work(layer(), T=0) == UNS and work(layer(), T=1025) == UNS
    lib = apus_hip.load()
    L = layer()
    assert lib.apus_hip_moe_layer_decode(C.byref(L), None, SZ(1), A, B) == ARG
    assert lib.apus_hip_moe_layer_decode(None, None, SZ(1), A, B) == ARG
    assert lib.apus_hip_moe_work_destroy(None) == 0


def test_disabled_first():
    code = ("import sys; sys.path.insert(0, %r); sys.path.insert(0, %r)\n"
            "import test_mx_refusals as t\n"
            "print(t.quant(K=48), t.quant(f='d', x=None), t.gemm(w=None), t.gemm_mx(xs=None), t.work(None))"
            % (os.path.dirname(apus_hip.__file__), os.path.dirname(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                       env=dict(os.environ, APUS_HIP_DISABLE="1"))
    assert r.returncode == 0 and r.stdout.split() == ["2"] * 5, (r.stdout, r.stderr)


def last_error():
    b = C.create_string_buffer(512)
    apus_hip.load().apus_hip_last_error(b, SZ(512))
    return b.value.decode()


def test_gemm_output_over_weights():
    """y among the codes or scales of the weights: from the first byte to the last, by
    any of its rows. Between y's rows there is room for them."""
    ld = 1 << 12                                           # rows of y 8 KiB apart, 20 bytes each
    for f in (gemm, gemm_mx):
        for k, p, n in (("w", A, 320), ("ws", B, 20)):     # 10 rows of 64
            for kw in (dict(y=p), dict(y=off(p, n - 2)), dict(y=off(p, -2 * 9)),
                       dict(y=off(p, n - 2 - 3 * 2 * ld), ldy=ld), {k: off(E, 3 * 2 * ld + 16), "ldy": ld},
                       {k: off(E, 2 * ld - 16), "ldy": ld}):
                assert f(**kw) == ARG and last_error() == "the output overlaps the weights", kw
            # (the next check is reached: x among y's rows)
            for kw in (dict(y=off(p, n), x=off(p, (n + 15) // 16 * 16)), dict(y=off(p, -80), x=off(p, -64)),
                       {k: off(E, 2 * ld + 32), "ldy": ld, "x": E}):
                assert f(**kw) == ARG and last_error() == "the output overlaps the activations", kw


def test_refused_device_is_not_kept():
    """A device that init refuses is not the one that the binding expects tensors on."""
    before = apus_hip._device
    try:
        with pytest.raises(apus_hip.ApusHipError):
            apus_hip.init(1000)
        assert apus_hip._device == before
    finally:
        try:
            apus_hip.init(before)
        except apus_hip.ApusHipError:                      # (no GPU here)
            pass


def test_moe_layer_without_a_weight():
    for w in ({}, {"w_router": None}, {"s_gate_up": None}):
        with pytest.raises(ValueError, match="w_router"):
            apus_hip.moe_layer((64, 32, 8, 2, 0), w)


def test_gemm_mx_of_a_vector():
    torch = pytest.importorskip("torch")
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    for x in (u8(32), u8(1, 1, 32)):
        with pytest.raises(ValueError):
            apus_hip.mxfp4_gemm_mx(u8(5, 32), u8(5, 2), x, u8(1, 2), torch.zeros(1, 5, dtype=torch.bfloat16))
