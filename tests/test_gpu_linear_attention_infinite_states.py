"""Linear attention whose states are infinite: they stay so with their sign, in their
column, until a reset, and so do the outputs that read them."""
import pytest
import torch

import attention_reference as plain
import sequence_reference as ref
from portdnn_amd import ops
from test_gpu_linear_attention import TYPES, _cuda, _make, _wide

pytestmark = pytest.mark.gpu

INF = float("inf")
# batch, steps, heads, key_heads, keys, values: up to 12 steps
SIZES = [(1, 5, 2, 2, 24, 40), (2, 12, 2, 2, 100, 72)]
KEY, VALUE = 7, 11


def _others(n):
    return [c for c in range(n) if c != VALUE]


def _signs(got, by, sign):
    """got is infinite with the sign of by."""
    want = sign * INF * torch.sign(by.float())
    assert (by != 0).all()
    assert torch.equal(got.float().cpu(), want)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("decay", [None, -INF])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_initial_states(size, dtype, decay, sign):
    t, _ = _make(size, dtype)
    if decay is not None:
        t["decay"][:] = decay
    t["q"][t["q"] == 0] = 1.0
    bad = {**t, "initial_state": t["initial_state"].clone()}
    bad["initial_state"][:, :, KEY, VALUE] = sign * INF
    for reset in (None, 3, size[1] - 2):
        for x in (t, bad):
            x["resets"] = torch.zeros(size[:2], dtype=torch.uint8)
            if reset is not None:
                x["resets"][:, reset] = 1
        o, last = ops.linear_attention(**_cuda(bad))
        want = plain.attention(dtype=dtype, **_wide(t))
        count = plain.operations(max(size[4:]), dtype)
        _signs(o[:, :reset, :, VALUE], t["q"][:, :reset, :, KEY], sign)
        part = [x[..., _others(size[5])] for x in want[0]]
        ref.check(o[..., _others(size[5])], part, count)
        got = last.cpu()
        if reset is None:
            assert (got[:, :, KEY, VALUE] == sign * INF).all()
            got[:, :, KEY, VALUE] = want[1][0][:, :, KEY, VALUE].float()
        else:
            ref.check(o[:, reset:], [x[:, reset:] for x in want[0]], count)
        ref.check(got, want[1], plain.state_operations(max(size[4:]), dtype))
