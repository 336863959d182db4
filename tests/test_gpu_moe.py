"""GPU parity: the mixture-of-experts layer against a plain 64-bit
implementation, within the bound of its fp32 arithmetic and one rounding."""
import pytest

import mx_ref

pytestmark = pytest.mark.gpu


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _layer(hip, w, topk, norm):
    E, I2, _ = w["w_gate_up"].shape
    H = w["w_router"].shape[1]
    Is = w["w_shared_gate_up"].shape[0] // 2 if "w_shared_gate_up" in w else 0
    return hip.moe_layer((H, I2 // 2, E, topk, Is), w, norm_topk=norm)


def _run(hip, torch, w, x, topk, norm, work=None):
    L = _layer(hip, w, topk, norm)
    own = work is None
    if own:
        work = hip.MoeWork(L, max(1, x.shape[0]))
    y = torch.full((x.shape[0] + 1, x.shape[1]), 7.0, dtype=torch.bfloat16, device="cuda")
    hip.moe_layer_decode(L, work, x, y[:-1])
    torch.cuda.synchronize()
    assert bool((y[-1] == 7.0).all())                      # the row behind the last token
    if own:
        work.destroy()
    return y[:-1]


# T, H, I, E, topk, Is, gate, norm
CASES = [(1, 2048, 512, 256, 8, 512, True, True),
         (1, 32, 32, 1, 1, 0, False, True),
         (1, 96, 64, 5, 5, 32, False, False),
         (2, 288, 160, 20, 3, 96, True, False),
         (5, 1056, 224, 60, 4, 0, False, True),
         (13, 1056, 224, 20, 3, 0, False, False),
         (16, 64, 32, 300, 8, 64, True, True),
         (17, 160, 96, 7, 7, 160, True, True),
         (33, 512, 256, 64, 6, 128, False, True),
         (40, 2048, 512, 128, 8, 512, True, True),
         (64, 544, 96, 1000, 32, 0, False, True),
         (130, 256, 128, 16, 2, 256, True, False),
         (325, 320, 64, 48, 8, 64, True, True),
         (513, 96, 32, 4, 2, 32, True, True),
         (1024, 64, 32, 40, 4, 0, False, True)]


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T,H,I,E,topk,Is,gate,norm", CASES)
def test_moe(hip, T, H, I, E, topk, Is, gate, norm, mx):
    import torch
    print(f"[moe] T={T} H={H} I={I} E={E} topk={topk} Is={Is} norm={norm} mx={mx}", flush=True)
    g = _gen(torch, T + H + E)
    w = mx_ref.moe_weights(g, H, I, E, Is, gate, mx)
    x = mx_ref.safe_tokens(g, w, T, topk, H)
    r, b, gap = mx_ref.moe(x, w, topk, norm, mx)
    assert float(gap.min()) > 0
    mx_ref.check(_run(hip, torch, w, x, topk, norm), r, b, "moe")


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T", [3, 50, 200])
def test_moe_all_to_few(hip, T, mx):
    """Every token goes to the same experts, most experts get none."""
    import torch
    g = _gen(torch, T)
    H, I, E, k = 256, 64, 40, 3
    w = mx_ref.moe_weights(g, H, I, E, 64, True, mx)
    x = mx_ref.safe_tokens(g, w, T, k, H)
    u = x.float().mean(0)
    x = (x.float() * 0.1 + u / u.norm() * 8).to(torch.bfloat16)
    w["w_router"][[7, 21, 39]] = (u / u.norm() * torch.tensor([[2.0], [1.5], [1.0]], device="cuda")).to(torch.bfloat16)
    r, b, gap = mx_ref.moe(x, w, k, True, mx)
    assert float(gap.min()) > 0
    mx_ref.check(_run(hip, torch, w, x, k, True), r, b, "all to few")


@pytest.mark.parametrize("T", [1, 6, 100])
def test_moe_ties_lowest_index(hip, T):
    """Router weights and activations of small integers: logits are exact and
    many are equal; the lowest indices are chosen. All equal: experts 0 .. k-1."""
    import torch
    g = _gen(torch, T + 1)
    H, I, E, k = 64, 32, 70, 6
    w = mx_ref.moe_weights(g, H, I, E, 0)
    w["w_router"] = torch.randint(-1, 2, (E, H), generator=g, device="cuda").to(torch.bfloat16)
    w["w_router"][:, 6:] = 0
    w["w_router"][3] = -0.0
    x = torch.randint(-2, 3, (T, H), generator=g, device="cuda").to(torch.bfloat16)
    x[0] = 0                                               # every logit zero, of both signs
    r, b, _ = mx_ref.moe(x, w, k, True, False)
    mx_ref.check(_run(hip, torch, w, x, k, True), r, b, "ties")


@pytest.mark.parametrize("T", [2, 70])
def test_moe_nan_stays_in_its_token(hip, T):
    import torch
    g = _gen(torch, T)
    H, I, E, k = 128, 64, 24, 4
    w = mx_ref.moe_weights(g, H, I, E, 64)
    x = mx_ref.safe_tokens(g, w, T, k, H)
    y0 = _run(hip, torch, w, x, k, True)
    for bad in (float("nan"), float("inf")):
        xb = x.clone()
        xb[T - 1, 5] = bad
        y = _run(hip, torch, w, xb, k, True)
        assert bool(y[T - 1].isnan().all())
        assert torch.equal(y[:T - 1], y0[:T - 1])
    wb = dict(w, w_router=w["w_router"].clone())           # an expert whose logit is NaN
    wb["w_router"][E - 1, 0] = float("nan")
    assert bool(_run(hip, torch, wb, x, k, True).isnan().all())


def test_moe_one_token_in_any_batch(hip):
    """Calls of any size fit one workspace, one after the other, and leave
    nothing behind for the next."""
    import torch
    g = _gen(torch, 9)
    H, I, E, k = 256, 96, 32, 4
    w = mx_ref.moe_weights(g, H, I, E, 64, True, True)
    x = mx_ref.safe_tokens(g, w, 200, k, H)
    work = hip.MoeWork(_layer(hip, w, k, True), 200)
    r, b, _ = mx_ref.moe(x, w, k, True, True)
    for n in (200, 1, 7, 64, 0, 33, 1, 200):
        mx_ref.check(_run(hip, torch, w, x[:n], k, True, work), r[:n], b[:n], f"T={n}")
    work.destroy()


def test_moe_in_place(hip):
    import torch
    g = _gen(torch, 4)
    w = mx_ref.moe_weights(g, 256, 64, 16, 64)
    for T in (1, 30):
        x = mx_ref.safe_tokens(g, w, T, 4, 256)
        y = _run(hip, torch, w, x, 4, True)
        L = _layer(hip, w, 4, True)
        work = hip.MoeWork(L, T)
        hip.moe_layer_decode(L, work, x, x)
        torch.cuda.synchronize()
        assert torch.equal(x, y)
        work.destroy()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T", [1, 48])
def test_moe_graphs(hip, T, mx):
    """Two captured calls with a workspace each, replayed at once on two
    streams with inputs of their own, several times, against eager calls."""
    import torch
    g = _gen(torch, 11)
    H, I, E, k = 512, 128, 32, 4
    w = mx_ref.moe_weights(g, H, I, E, 128, True, mx)
    L = _layer(hip, w, k, True)
    xs, ys, graphs, works, streams = [], [], [], [], []
    for i in range(2):
        x = mx_ref.safe_tokens(g, w, T, k, H)
        y = torch.empty_like(x)
        work, st, graph = hip.MoeWork(L, T), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        st.wait_stream(torch.cuda.current_stream())
        try:
            with torch.cuda.graph(graph, stream=st):
                hip.set_stream(torch.cuda.current_stream().cuda_stream)
                hip.moe_layer_decode(L, work, x, y)
        finally:
            hip.set_stream(0)
        for a, v in ((xs, x), (ys, y), (graphs, graph), (works, work), (streams, st)):
            a.append(v)
    for n in range(4):
        for i in range(2):
            xs[i].copy_(mx_ref.safe_tokens(_gen(torch, 100 + 2 * n + i), w, T, k, H))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(ys[i], _run(hip, torch, w, xs[i], k, True)), (n, i)
    del graphs
    for work in works:
        work.destroy()


def test_moe_refusals(hip):
    import torch
    g = _gen(torch, 2)
    w = mx_ref.moe_weights(g, 64, 32, 8, 32)
    L = _layer(hip, w, 2, True)
    work = hip.MoeWork(L, 4)
    x = mx_ref.normal(g, 5, 64)
    with pytest.raises(hip.ApusHipError) as e:             # more tokens than the workspace holds
        hip.moe_layer_decode(L, work, x, torch.empty_like(x))
    assert e.value.code == 3
    other = _layer(hip, w, 3, True)                        # a layer of another shape
    with pytest.raises(hip.ApusHipError) as e:
        hip.moe_layer_decode(other, work, x[:1], torch.empty_like(x[:1]))
    assert e.value.code == 3
    with pytest.raises(ValueError):                        # y of another shape
        hip.moe_layer_decode(L, work, x[:2], torch.empty_like(x))
    with pytest.raises(ValueError):                        # weights of another shape
        hip.moe_layer((64, 64, 8, 2, 32), w)
    with pytest.raises(ValueError):                        # another 2-byte type
        hip.moe_layer((64, 32, 8, 2, 32), dict(w, w_router=w["w_router"].half()))
    with pytest.raises(ValueError):
        hip.moe_layer_decode(L, work, x[:2].half(), torch.empty_like(x[:2]))
    for T in (0, 1025):
        with pytest.raises(hip.ApusHipError) as e:
            hip.MoeWork(L, T)
        assert e.value.code == 1
    work.destroy()
    with pytest.raises(hip.ApusHipError) as e:             # no workspace any more
        hip.moe_layer_decode(L, work, x[:1], torch.empty_like(x[:1]))
    assert e.value.code == 3


# the forms that rules on sizes choose between: slots and row blocks on either
# side of the streaming kernels' thresholds, inner sizes past what they hold,
# several rounds of K, slots of more than 16 and several slots of one expert
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T,H,I,E,topk,Is", [(5, 2048, 512, 40, 8, 512), (8, 1056, 544, 64, 8, 96),
                                             (20, 4128, 96, 32, 6, 64), (100, 544, 512, 24, 8, 544),
                                             (200, 2080, 160, 12, 4, 32), (300, 256, 1056, 10, 5, 0),
                                             (70, 2048, 480, 100, 8, 1056), (1000, 96, 64, 130, 2, 64),
                                             (3, 4128, 1184, 9, 5, 2080), (400, 1056, 480, 20, 5, 96),
                                             (40, 1056, 672, 60, 4, 1056), (9, 4128, 640, 40, 6, 32),
                                             (500, 1056, 768, 16, 4, 640), (90, 2080, 2112, 5, 2, 64)])
def test_moe_forms(hip, T, H, I, E, topk, Is, mx):
    import torch
    print(f"[moe] forms T={T} H={H} I={I} E={E} topk={topk} Is={Is} mx={mx}", flush=True)
    g = _gen(torch, T + H + I)
    w = mx_ref.moe_weights(g, H, I, E, Is, True, mx)
    x = mx_ref.safe_tokens(g, w, T, topk, H)
    r, b, gap = mx_ref.moe(x, w, topk, True, mx)
    assert float(gap.min()) > 0
    mx_ref.check(_run(hip, torch, w, x, topk, True), r, b, "forms")


@pytest.mark.parametrize("T", [1, 12, 100])
def test_moe_scales_of_any_alignment(hip, T):
    """Scales are bytes: a tensor of them may begin at any address."""
    import torch
    g = _gen(torch, T)
    H, I, E, k = 1024, 512, 24, 4
    w = mx_ref.moe_weights(g, H, I, E, 512, True, True)
    x = mx_ref.safe_tokens(g, w, T, k, H)
    y = _run(hip, torch, w, x, k, True)
    for off in (1, 2, 3):
        v = dict(w)
        for n in [n for n in w if n.startswith("s_")]:
            b = torch.empty(w[n].numel() + 4, dtype=torch.uint8, device="cuda")
            v[n] = b[off:off + w[n].numel()].view(w[n].shape).copy_(w[n])
            assert v[n].data_ptr() % 4 == off
        assert torch.equal(_run(hip, torch, v, x, k, True), y)
