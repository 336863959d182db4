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


# k_moe_down_few, _down, _down_stream and _down_walk
@pytest.mark.parametrize("T,H,I,E,k", [(1, 256, 64, 8, 2), (13, 256, 64, 8, 2), (64, 1024, 64, 64, 8),
                                       (64, 1024, 544, 64, 8), (300, 1024, 64, 16, 4)])
@pytest.mark.parametrize("kind", ["bf16", "mx", "overflow"])
def test_infinite_down_weights(hip, T, H, I, E, k, kind):
    """Inner values of few bits (64 times a number of e2m1), or past fp32, and one
    infinite weight an output, or all of them: y is infinite with its sign."""
    import torch
    mx = kind == "mx"
    g = _gen(torch, T + I)
    w = mx_ref.moe_weights(g, H, I, E, 0, False, False)
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 1
    gu = w["w_gate_up"]
    gu[:] = 0
    gu[:, :I, 0] = 64 if kind != "overflow" else 2.0 ** 100
    gu[:, I:, 0] = torch.tensor([1, 2, 3, 4, 6, 1.5, 0.5, 1], device="cuda").repeat(I // 8).to(torch.bfloat16) * (
        1 if kind != "overflow" else 2.0 ** 60)
    o = torch.arange(H, device="cuda")
    sign = (1 - 2 * (o % 2)).to(torch.bfloat16)
    if kind == "overflow":
        w["w_down"][:] = sign[None, :, None] * float("inf")
    elif not mx:
        w["w_down"][:, o, o % I] = sign * float("inf")
    else:
        for n in ("gate_up", "down"):
            w["w_" + n], w["s_" + n] = mx_ref.quantize(w["w_" + n])
        at = o % I                                         # the element's block: one code of 6, at 2^127
        w["s_down"][:, o, at // 32] = 254
        blocks = w["w_down"].view(E, H, I // 32, 16)
        blocks[:, o, at // 32] = 0
        blocks[:, o, at // 32, at % 32 // 2] = torch.where(at % 2 == 0, 7, 7 << 4).to(torch.uint8) | torch.where(
            sign < 0, torch.where(at % 2 == 0, 8, 8 << 4), torch.zeros_like(at)).to(torch.uint8)
        assert torch.equal(mx_ref.values(w["w_down"], w["s_down"])[0].to(torch.bfloat16).isinf().sum(1), torch.ones_like(o))
    L = _layer(hip, w, k)
    work = hip.MoeWork(L, T)
    y = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    hip.moe_layer_decode(L, work, x, y)
    assert torch.equal(y, (sign * float("inf")).expand(T, H))
    work.destroy()


# k_moe_down_few, _down, and _down_stream: inner values in one chunk and in several, slots of 16 rows and of 32
@pytest.mark.parametrize("T,H,I,E", [(1, 256, 64, 8), (2, 64, 1184, 3), (13, 256, 64, 8), (40, 96, 2080, 3), (64, 1024, 64, 64),
                                     (64, 1056, 544, 64), (100, 1024, 1152, 40), (1000, 1024, 512, 40),
                                     (1000, 1056, 1056, 16)])
@pytest.mark.parametrize("mx", [False, True])
def test_inner_values_of_24_bits(hip, T, H, I, E, mx):
    """Inner values that are integers of 24 bits (times 64), of which each output takes the
    difference of two with the same 16 leading bits: all in fp32, and exact."""
    import torch
    g = _gen(torch, T + I)
    n = torch.randint(1 << 23, 1 << 24, (E, I // 2, 1), generator=g, device="cuda") & ~255
    n = (n + torch.randint(0, 256, (E, I // 2, 2), generator=g, device="cuda")).view(E, I)
    bit = torch.arange(24, device="cuda")
    w = dict(w_router=mx_ref.normal(g, E, H, scale=0.5), w_gate_up=torch.zeros(E, 2 * I, H, dtype=torch.bfloat16, device="cuda"),
             w_down=torch.zeros(E, H, I, dtype=torch.bfloat16, device="cuda"))
    w["w_router"][:, :40] = 0
    w["w_gate_up"][:, :I, 32] = 64                         # silu(64) = 64 in fp32
    w["w_gate_up"][:, I:, :24] = (n.unsqueeze(-1) >> bit & 1).to(torch.bfloat16)
    o = torch.arange(H, device="cuda")
    w["w_down"][:, o, 2 * o % I] = 1
    w["w_down"][:, o, 2 * o % I + 1] = -1
    if mx:
        for m in ("gate_up", "down"):
            w["w_" + m], w["s_" + m] = mx_ref.quantize(w["w_" + m])
    x = mx_ref.normal(g, T, H)
    x[:, :40] = 0
    x[:, :24] = torch.exp2(bit.float()).to(torch.bfloat16)
    x[:, 32] = 1
    r, _, gap = mx_ref.moe(x, w, 1, True, mx)
    assert float((r - 64 * torch.round(r / 64)).abs().max()) < 1e-9 and 0 < float(r.abs().max()) <= 64 * 255
    L = _layer(hip, w, 1)
    work = hip.MoeWork(L, T)
    y = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    hip.moe_layer_decode(L, work, x, y)
    ok = gap > 0                                           # (the choice no fp32 sum's error can change)
    assert int(ok.sum()) >= T - T // 10
    assert torch.equal(y[ok].double(), torch.round(r[ok]))
    work.destroy()


# one and two tokens: one round of k_moe_down_few's loads, several, and past what it takes of two tokens
@pytest.mark.parametrize("T,H,I,E,k,Is", [(1, 96, 1184, 9, 5, 544), (1, 2080, 5600, 4, 2, 32), (2, 288, 512, 40, 8, 512),
                                          (2, 544, 672, 40, 8, 0), (2, 1056, 1184, 12, 4, 2080), (2, 96, 4128, 5, 2, 64)])
@pytest.mark.parametrize("mx", [False, True])
def test_one_and_two_tokens(hip, T, H, I, E, k, Is, mx):
    import torch
    g = _gen(torch, T + H + I)
    w = mx_ref.moe_weights(g, H, I, E, Is, True, mx)
    x = mx_ref.safe_tokens(g, w, T, k, H)
    r, b, _ = mx_ref.moe(x, w, k, True, mx)
    L = _layer(hip, w, k)
    work = hip.MoeWork(L, T)
    y = torch.empty_like(x)
    hip.moe_layer_decode(L, work, x, y)
    mx_ref.check(y, r, b, "one and two tokens")
    work.destroy()


# the last slot of the one popular expert has 2 rows, of 5, and of 1 (of 16 or of 32)
@pytest.mark.parametrize("T,H,I", [(66, 5472, 2112), (85, 4128, 4192), (994, 1056, 2112), (993, 1056, 544)])
@pytest.mark.parametrize("mx", [False, True])
def test_all_to_one_expert_of_long_rows(hip, T, H, I, mx):
    """One expert gets every token, in slots that are full but for the last; inner sizes of
    several chunks, each form of a slot."""
    import torch
    print(f"[moe] all to one T={T} H={H} I={I} mx={mx}", flush=True)
    g = _gen(torch, T + I)
    w = mx_ref.moe_weights(g, H, I, 2, 0, False, mx)
    x = mx_ref.normal(g, T, H)
    x[:, 0] = 1
    w["w_router"][0, 0] = 40
    r, b, gap = mx_ref.moe(x, w, 1, True, mx)
    assert float(gap.min()) > 0
    L = _layer(hip, w, 1)
    work = hip.MoeWork(L, T)
    ys = []
    for _ in range(3):                                     # (the order within the slots is no matter)
        y = torch.full_like(x, 7.0)
        hip.moe_layer_decode(L, work, x, y)
        ys.append(y)
    mx_ref.check(ys[0], r, b, "all to one")
    assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])
    work.destroy()


@pytest.mark.parametrize("T,H,I,E,k,Is", [(64, 1024, 512, 24, 4, 96), (150, 288, 160, 6, 2, 64), (400, 1056, 640, 12, 3, 0)])
@pytest.mark.parametrize("mx", [False, True])
def test_outputs_repeat(hip, T, H, I, E, k, Is, mx):
    """The choices come to their experts' slots in any order: a token's output is the
    same bits, whatever the order of the tokens."""
    import torch
    g = _gen(torch, T + H)
    w = mx_ref.moe_weights(g, H, I, E, Is, True, mx)
    x = mx_ref.safe_tokens(g, w, T, k, H)
    L = _layer(hip, w, k)
    work = hip.MoeWork(L, T)
    y = torch.empty_like(x)
    hip.moe_layer_decode(L, work, x, y)
    for i in range(8):
        at = torch.randperm(T, generator=g, device="cuda")
        z = torch.empty_like(x)
        hip.moe_layer_decode(L, work, x[at].contiguous(), z)
        assert torch.equal(z, y[at]), i
    work.destroy()
