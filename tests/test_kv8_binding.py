"""CPU checks of the Python binding of the 8-bit cache's calls and the norms around
a block: what it hands to the library of the tensors that it is given, which here
lie in host memory (no call is made)."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import apus_hip as H


@pytest.fixture
def kv(monkeypatch):
    monkeypatch.setattr(H, "_device", -1)                  # (a host tensor's get_device())
    kv = H.Kv8Cache()
    kv.nkv = 2
    return kv


def bind(f, kv, k, v):
    return getattr(H, f + "_bound")(kv, None, [0, k.shape[0]], [0], k, v)


@pytest.mark.parametrize("f", ["kv8_append", "kv8_read"])
def test_rows_of_heads_are_the_tensors_own(kv, f):
    """Three-dimensional rows go by the tensor's own memory; those whose elements
    do not lie in a row are refused, and not copied."""
    rows = [torch.zeros(7, 2, 256, dtype=torch.bfloat16), torch.zeros(7, 5, 256, dtype=torch.bfloat16)[:, 2:4],
            torch.zeros(1, 2, 256, dtype=torch.bfloat16), torch.zeros(9, 4, 256, dtype=torch.bfloat16)[::2, 1:3]]
    for x in rows:
        a = bind(f, kv, x, x)._args
        assert a[6] == a[8] == x.data_ptr()
        assert a[7] == a[9] == (x.stride(0) if x.shape[0] > 1 else 512)
    good = rows[0]
    across = torch.zeros(256, 2, 7, dtype=torch.bfloat16).permute(2, 1, 0)         # strides 1, 7, 14
    dims_first = torch.zeros(256, 2, 256, dtype=torch.bfloat16)[:, :, :7].permute(2, 1, 0)
    assert dims_first.stride() == (1, 256, 512)
    every_other = torch.zeros(7, 512, 2, dtype=torch.bfloat16)[..., 0].unflatten(1, (2, 256))
    for bad in (across, dims_first, every_other, dims_first[:1], good.transpose(1, 2)):
        with pytest.raises(ValueError, match="k: rows"):
            bind(f, kv, bad, torch.zeros(bad.shape[0], 2, 256, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="v: rows"):
            bind(f, kv, torch.zeros(bad.shape[0], 2, 256, dtype=torch.bfloat16), bad)
    kv.nkv = 1                                             # (one head: no stride between heads)
    x = torch.zeros(7, 3, 256, dtype=torch.bfloat16)[:, 1:2]
    assert bind(f, kv, x, x)._args[6:8] == (x.data_ptr(), 768)
    with pytest.raises(ValueError, match="k: rows"):
        x = torch.zeros(256, 1, 7, dtype=torch.bfloat16).permute(2, 1, 0)
        bind(f, kv, x, x)
    none = torch.zeros(0, 1, 256, dtype=torch.bfloat16)
    bind(f, kv, none, none)


@pytest.fixture
def norm_calls(monkeypatch):
    """What block_norm hands over: (the norm as the library would see it, its address)."""
    got = []

    class Lib:
        @staticmethod
        def apus_hip_block_norm(norm, *args):
            got.append((H.BlockNorm.from_buffer_copy(C.string_at(norm, C.sizeof(H.BlockNorm))), norm))
            return 0
    monkeypatch.setattr(H, "_device", -1)
    monkeypatch.setattr(H, "load", lambda: Lib)
    return got


def test_a_norm_is_only_read(norm_calls):
    """One norm for bf16 and fp32 residuals, by turns: each call has its own type,
    and the caller's descriptor stays as it was."""
    w = torch.zeros(64, dtype=torch.bfloat16)
    norm = H.block_norm_weights(64, w_pre=w, w_post=w, scale=0.5, eps=1e-5)
    was = bytes(norm)
    y = torch.zeros(3, 64, dtype=torch.bfloat16)
    for dtype in (torch.bfloat16, torch.float32, torch.float32, torch.bfloat16, torch.float32):
        h = torch.zeros(3, 64, dtype=dtype)
        H.block_norm(norm, y, h, h, torch.empty_like(y))
        seen = norm_calls[-1][0]
        assert seen.h_f32 == (dtype == torch.float32) and bytes(norm) == was
        assert (seen.hidden, seen.scale, seen.w_pre, seen.w_post) == (64, 0.5, w.data_ptr(), w.data_ptr())
    norm.scale, norm.h_f32 = 2.0, 1                        # (what the caller changes counts from the next call on)
    for dtype in (torch.float32, torch.bfloat16):
        h = torch.zeros(3, 64, dtype=dtype)
        H.block_norm(norm, y, h, h, torch.empty_like(y))
        assert norm_calls[-1][0].scale == 2.0 and norm_calls[-1][0].h_f32 == (dtype == torch.float32)


def test_two_threads_with_one_norm(norm_calls, monkeypatch):
    """A call that waits inside the library keeps its type while another thread
    calls with the other."""
    w = torch.zeros(64, dtype=torch.bfloat16)
    norm = H.block_norm_weights(64, w_pre=w)
    inside, go, types = threading.Event(), threading.Event(), {}

    class Lib:
        @staticmethod
        def apus_hip_block_norm(at, *args):
            first = threading.current_thread().name == "first"
            if first:
                inside.set()
                assert go.wait(30)
            types[first] = H.BlockNorm.from_buffer_copy(C.string_at(at, C.sizeof(H.BlockNorm))).h_f32
            return 0
    monkeypatch.setattr(H, "load", lambda: Lib)
    call = lambda dtype: H.block_norm(norm, None, torch.zeros(2, 64, dtype=dtype), None,             # noqa: E731
                                      torch.zeros(2, 64, dtype=torch.bfloat16))
    t = threading.Thread(target=call, args=(torch.float32,), name="first")
    t.start()
    assert inside.wait(30)
    call(torch.bfloat16)
    go.set()
    t.join(30)
    assert types == {True: 1, False: 0}


def test_bound_offsets_stay_in_the_tensors(kv, monkeypatch):
    """Offsets changed in place after a call was bound: up to the tensors' rows."""
    calls = []
    x = torch.zeros(7, 512, dtype=torch.bfloat16)
    layer = H.AttnLayer(16, 2, 256, 64, 1e7)
    work = type("Work", (), {"h": None})
    cu = np.array([0, 3, 7], np.int32)
    pos = np.zeros(2, np.int32)
    y = torch.zeros(7, 16 * 256, dtype=torch.bfloat16)
    qg = torch.zeros(7, 16, 512, dtype=torch.bfloat16)
    bound = [H.kv8_append_bound(kv, None, cu, pos, x, x), H.kv8_read_bound(kv, None, cu, pos, x, x.clone()),
             H.attn_decode_kv8_bound(layer, work, None, cu, pos, qg, x, x, kv, y),
             H.attn_prefill_kv8_bound(layer, work, None, cu, pos, qg, None, None, kv, y)]
    for b in bound:
        monkeypatch.setattr(b, "_f", lambda *a: calls.append(a) or 0)
    for last, fits in ((7, True), (8, False), (5, True), (1 << 30, False), (7, True)):
        cu[-1] = last
        for b in bound:
            calls.clear()
            if fits:
                b()
            else:
                with pytest.raises(ValueError, match="cu: "):
                    b()
            assert len(calls) == fits
