"""GPU: edges of the mixture-of-experts layer that its parity tests do not meet."""
import pytest

import mx_ref

pytestmark = pytest.mark.gpu


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _layer(hip, w, topk, norm=True):
    E, I2, _ = w["w_gate_up"].shape
    H = w["w_router"].shape[1]
    Is = w["w_shared_gate_up"].shape[0] // 2 if "w_shared_gate_up" in w else 0
    return hip.moe_layer((H, I2 // 2, E, topk, Is), w, norm_topk=norm)


@pytest.mark.parametrize("mx", [False, True])
def test_output_over_weights_is_refused(hip, mx):
    import torch
    g = _gen(torch, 5)
    T, H, I, E, k, Is = 2, 256, 64, 8, 2, 64
    w = mx_ref.moe_weights(g, H, I, E, Is, True, mx)
    L = _layer(hip, w, k)
    work = hip.MoeWork(L, T)
    x = mx_ref.normal(g, T, H)
    before = {n: t.clone() for n, t in w.items()}
    for n, t in w.items():
        v = t.view(-1).view(torch.bfloat16) if t.dtype == torch.uint8 else t.view(-1)
        if v.numel() < T * H:                              # (no room for y)
            continue
        for y in (v[:T * H], v[-T * H:]):
            with pytest.raises(hip.ApusHipError) as e:
                hip.moe_layer_decode(L, work, x, y.view(T, H))
            assert e.value.code == 3, n
    torch.cuda.synchronize()
    assert all(torch.equal(before[n].view(torch.uint8), t.view(torch.uint8)) for n, t in w.items())
    # beside a weight, in one buffer with it
    both = torch.empty(w["w_router"].numel() + T * H, dtype=torch.bfloat16, device="cuda")
    r = both[:-T * H].view(E, H).copy_(w["w_router"])
    y, y1 = both[-T * H:].view(T, H), torch.empty_like(x)
    hip.moe_layer_decode(L, work, x, y1)
    hip.moe_layer_decode(_layer(hip, dict(w, w_router=r), k), work, x, y)
    assert torch.equal(y, y1)
    work.destroy()


@pytest.mark.parametrize("mx", [False, True])
def test_layer_without_a_weight_is_refused(hip, mx):
    import torch
    w = mx_ref.moe_weights(_gen(torch, 6), 64, 32, 8, 32, True, mx)
    _layer(hip, {n: t for n, t in w.items() if n != "w_shared_gate"}, 2)         # (may be left out)
    for n in set(w) - {"w_shared_gate", "s_gate_up"}:
        for v in ({m: t for m, t in w.items() if m != n}, dict(w, **{n: None})):
            with pytest.raises(ValueError, match=n):
                hip.moe_layer((64, 32, 8, 2, 32), v)
    if mx:                                                 # (codes are no bf16 weights)
        with pytest.raises(ValueError, match="w_gate_up"):
            hip.moe_layer((64, 32, 8, 2, 32), {m: t for m, t in w.items() if m != "s_gate_up"})
        with pytest.raises(ValueError, match="s_gate_up"):
            hip.moe_layer((64, 32, 8, 2, 32), dict(w, s_gate_up=None))
