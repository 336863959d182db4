"""The 8-bit KV cache on the GPU where its calls are at their limits."""
import pytest

from test_gpu_kv8 import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ctx,new", [
    ([0, 4080], [0, 16]), ([0, 700], [0, 500]), ([0, 5000, 40], [0, 20, 20]), ([5000, 0, 40, 30000], [20, 0, 20, 0]),
    ([0, 0, 9000], [0, 0, 7])])
def test_prefill_split_beside_idle_rows(hip, ctx, new):
    """Keys in parts, beside sequences without tokens or cached positions."""
    s = Setup(hip, 110 + len(ctx) + new[-1], 2, ctx, new, True)
    s.check(s.call(hip.attn_prefill_kv8))
