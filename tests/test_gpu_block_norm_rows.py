"""The norms around a block for as many rows as a call may have."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    """The largest case takes 69 GB, which the tests after it may need."""
    yield
    torch.cuda.empty_cache()


def bf16(*shape, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(shape[-1])
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


@pytest.mark.parametrize("n,T", [(1032, 1 << 24), (1032, (1 << 22) + 1), (509, (1 << 22) + 5)])
def test_many_rows(hip, n, T):
    """Rows that repeat every 61, so in every launch's share: x is that of the
    first of them, bit for bit, and the row behind the last stays as it was."""
    few = bf16(61, n)
    norm = hip.block_norm_weights(n, w_pre=bf16(n, scale=0.1))
    want = torch.empty_like(few)
    hip.block_norm(norm, None, few, None, want)
    h = torch.empty(T, n, dtype=torch.bfloat16, device="cuda")
    whole = T // 61 * 61
    h[:whole].view(-1, 61, n).copy_(few.expand(whole // 61, 61, n))
    h[whole:].copy_(few[:T - whole])
    x = torch.full((T + 1, n), 7.0, dtype=torch.bfloat16, device="cuda")
    hip.block_norm(norm, None, h, None, x[:T])
    step = 61 << 14
    for r in range(0, whole, step):
        part = x[r:min(r + step, whole)].view(-1, 61, n)
        assert torch.equal(part, want.expand(part.shape)), r
    assert torch.equal(x[whole:T], want[:T - whole]) and (x[T] == 7.0).all()


def test_many_rows_of_every_operand(hip):
    """The same with a block's output, a gate a row and fp32 residuals."""
    n, T = 16, (1 << 22) + 9
    y, gate, h = (bf16(61, n).repeat(T // 61 + 1, 1)[:T] for _ in range(3))
    h = h.float()
    w = bf16(n, scale=0.1)
    want = [torch.empty(61, n, device="cuda"), torch.empty(61, n, dtype=torch.bfloat16, device="cuda")]
    hip.block_norm(hip.block_norm_weights(n, w, w, gate[:61].contiguous()), y[:61], h[:61], *want)
    got = [torch.empty(T, n, device="cuda"), torch.empty(T, n, dtype=torch.bfloat16, device="cuda")]
    hip.block_norm(hip.block_norm_weights(n, w, w, gate), y, h, *got)
    for a, b in zip(got, want):
        assert torch.equal(a, b.repeat(T // 61 + 1, 1)[:T])
