"""CPU checks of the Python binding of the 8-bit cache's calls: what it hands to
the library of the tensors that it is given, which here lie in host memory (no
call is made)."""
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
