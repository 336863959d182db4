"""CPU checks: the 8-bit cache's, its attention's and the block norm's entry
points refuse bad arguments before they look for a device (device addresses
here are never read), and with APUS_HIP_DISABLE set return "disabled"."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import apus_hip as H

ARG, UNS = 3, 1
K, V, S, X, Y, Q, G, O, T = (n << 36 for n in range(1, 10))   # aligned, far apart


def cache(**kw):
    f = dict(k=K, v=V, scale=S, blocks=64, block_table=None, max_blocks=8, max_rows=8, row_blocks=None)
    f.update(kw)
    return H.Kv8Cache(**f)


def arr(x):
    return None if x is None else np.ascontiguousarray(x, np.int32)


def p(a):
    return None if a is None else a.ctypes.data


def rows(f, c=None, nkv=2, B=2, rows=None, cu=(0, 3, 5), pos=(0, 40), k=X, ldk=512, v=Y, ldv=512):
    c = cache() if c is None else c
    rows, cu, pos = arr(rows), arr(cu), arr(pos)
    return getattr(H.load(), "apus_hip_kv8_" + f)(C.addressof(c) if c else None, nkv, B, p(rows), p(cu), p(pos), k, ldk, v, ldv)


@pytest.mark.parametrize("f", ["append", "read"])
def test_cache_refusals(f):
    for n in ("k", "v", "scale"):
        assert rows(f, cache(**{n: None})) == ARG
    assert rows(f, c=False) == ARG
    assert rows(f, nkv=0) == UNS and rows(f, nkv=1 << 40) == UNS
    for kw in (dict(blocks=0), dict(max_blocks=0), dict(max_rows=0), dict(blocks=1 << 31), dict(max_blocks=1 << 26)):
        assert rows(f, cache(**kw)) == ARG
    assert rows(f, cache(max_rows=9)) == ARG               # flat: more rows than blocks hold
    assert rows(f, cache(k=K + 8)) == UNS and rows(f, cache(scale=S + 4)) == UNS
    assert rows(f, cache(v=K + 64 * 2 * 8192 - 16)) == ARG  # arrays on top of each other
    assert rows(f, cache(scale=V + 16)) == ARG


@pytest.mark.parametrize("f", ["append", "read"])
def test_batch_refusals(f):
    assert rows(f, cu=(1, 3, 5)) == ARG and rows(f, cu=(0, 3, 2)) == ARG
    assert rows(f, cu=None) == ARG and rows(f, pos=None) == ARG
    assert rows(f, pos=(-1, 0)) == ARG
    assert rows(f, pos=(0, 255)) == ARG                    # past the row's blocks
    assert rows(f, pos=(0, (1 << 31) - 1)) == ARG
    assert rows(f, rows=(0, 8)) == ARG and rows(f, rows=(-1, 0)) == ARG
    held = arr([1, 0, -1, 2, 0, 0, 0, 0])
    c = cache(row_blocks=p(held))
    assert rows(f, c, rows=(2, 3), pos=(0, 0)) == ARG      # not open
    assert rows(f, c, rows=(0, 3), pos=(30, 0)) == ARG     # past what it holds
    assert rows("append", rows=(3, 3)) == ARG              # one row twice
    assert rows("append", B=3, rows=(3, 1, 3), cu=(0, 1, 2, 3), pos=(0, 0, 40)) == ARG
    assert rows(f, B=1 << 25) == UNS


@pytest.mark.parametrize("f", ["append", "read"])
def test_row_refusals(f):
    for n in ("k", "v"):
        assert rows(f, **{n: None}) == ARG
        assert rows(f, **{n: X + 8}) == UNS
        assert rows(f, **{"ld" + n: 511}) == ARG
        assert rows(f, **{"ld" + n: 516}) == UNS
        assert rows(f, **{"ld" + n: 1 << 40}) == UNS
        assert rows(f, **{n: K + 1024}) == ARG             # inside the cache
        assert rows(f, **{n: V}) == ARG and rows(f, **{n: S}) == ARG
    assert rows("read", v=X + 512) == ARG                  # the outputs on top of each other


def test_work_refusals():
    L = H.AttnLayer(16, 2, 256, 64, 1e7, X, Y)
    out = C.c_void_p()
    f = H.load().apus_hip_attn_kv8_work_create
    mk = lambda layer, n, m: f(C.byref(layer), C.c_size_t(n), C.c_size_t(m), C.byref(out))     # noqa: E731
    assert mk(H.AttnLayer(16, 2, 128, 64, 1e7, X, Y), 1, 10) == UNS
    assert mk(H.AttnLayer(15, 2, 256, 64, 1e7, X, Y), 1, 10) == UNS
    assert mk(L, 0, 10) == UNS and mk(L, 1, 0) == UNS and mk(L, 1 << 25, 10) == UNS and mk(L, 1, 1 << 25) == UNS
    assert f(C.byref(L), C.c_size_t(1), C.c_size_t(1), None) == ARG
    assert f(None, C.c_size_t(1), C.c_size_t(1), C.byref(out)) == ARG
    assert not out.value


@pytest.mark.parametrize("f", ["decode", "prefill"])
def test_attention_refusals(f):
    L = H.AttnLayer(16, 2, 256, 64, 1e7, X, Y)
    c, cu, pos = cache(), arr([0, 1]), arr([0])
    call = getattr(H.load(), f"apus_hip_attn_{f}_kv8")
    assert call(C.addressof(L), None, 1, None, p(cu), p(pos), Q, None, None, C.addressof(c), O) == ARG
    assert call(None, None, 1, None, p(cu), p(pos), Q, None, None, C.addressof(c), O) == ARG


def test_pool_refusals():
    out = C.c_void_p()
    lib = H.load()
    assert lib.apus_hip_kv8_pool_cache(None, C.c_size_t(0), C.byref(cache())) == ARG
    del out


def norm(n=64, T=4, y=Y, ldy=64, h=X, ldh=64, o=O, ldo=64, x=G, ldx=64, **kw):
    f = dict(hidden=n, h_f32=0, scale=1.0, eps=1e-6, w_post=None, w_pre=K, gate=None, ld_gate=0)
    f.update(kw)
    N = H.BlockNorm(**f)
    return H.load().apus_hip_block_norm(C.addressof(N), T, y, ldy, h, ldh, o, ldo, x, ldx)


def test_norm_refusals():
    assert norm(n=0) == UNS and norm(n=16385, ldy=1 << 15, ldh=1 << 15, ldo=1 << 15, ldx=1 << 15) == UNS
    assert norm(T=1 << 25) == UNS
    assert norm(eps=-1.0) == ARG and norm(eps=float("nan")) == ARG
    assert norm(h=None) == ARG and norm(o=None) == ARG and norm(y=None, x=None) == ARG
    assert norm(w_pre=None) == ARG
    for ld in ("ldy", "ldh", "ldo", "ldx"):
        assert norm(**{ld: 63}) == ARG
        assert norm(**{ld: 1 << 62}) == UNS
    assert norm(gate=T, ld_gate=63) == ARG
    assert norm(y=Y + 1) == ARG and norm(h=X + 2, h_f32=1) == ARG and norm(w_pre=K + 1) == ARG
    assert norm(o=X + 2) == ARG and norm(o=Y) == ARG and norm(x=X) == ARG and norm(x=O) == ARG
    assert norm(o=X, ldo=72) == ARG and norm(x=Y, ldx=72) == ARG
    assert norm(o=K) == ARG and norm(x=K - 64) == ARG
    assert norm(o=T, gate=T) == ARG and norm(x=T + 64, gate=T, ld_gate=64) == ARG
    lib = H.load()
    assert lib.apus_hip_block_norm(None, 1, Y, 64, X, 64, O, 64, G, 64) == ARG


def test_disabled_first():
    code = ("import sys; sys.path.insert(0, sys.argv[1]); import ctypes as C, apus_hip as H\n"
            "l = H.load(); o = C.c_void_p()\n"
            "r = [l.apus_hip_kv8_append(None, 0, 0, None, None, None, None, 0, None, 0),\n"
            "     l.apus_hip_kv8_read(None, 0, 0, None, None, None, None, 0, None, 0),\n"
            "     l.apus_hip_attn_decode_kv8(None, None, 0, None, None, None, None, None, None, None, None),\n"
            "     l.apus_hip_attn_prefill_kv8(None, None, 0, None, None, None, None, None, None, None, None),\n"
            "     l.apus_hip_attn_layer_decode_kv8(None, None, None, 0, None, None, None, None, None, None),\n"
            "     l.apus_hip_attn_kv8_work_create(None, C.c_size_t(0), C.c_size_t(0), None),\n"
            "     l.apus_hip_attn_kv8_work_destroy(None),\n"
            "     l.apus_hip_kv8_pool_create(*[C.c_size_t(0)] * 6, None),\n"
            "     l.apus_hip_block_norm(None, 0, None, 0, None, 0, None, 0, None, 0)]\n"
            "assert r == [2] * 9, r\n")
    env = dict(os.environ, APUS_HIP_DISABLE="1")
    subprocess.run([sys.executable, "-c", code, os.path.dirname(H.__file__)], env=env, check=True)
