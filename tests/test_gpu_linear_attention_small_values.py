"""Linear attention in binary16 where values are far from one: states are fp32 and
keep their bits, whatever the size of the values that make them."""
import pytest
import torch

import attention_reference as plain
import sequence_reference as ref
from portdnn_amd import ops
from test_gpu_linear_attention import _cuda, _make, _wide

pytestmark = pytest.mark.gpu

# batch, steps, heads, key_heads, keys, values: each way into LDS, four waves and
# eight, whole sequences and pieces
SIZES = [(2, 200, 4, 2, 40, 72), (2, 130, 2, 2, 64, 64), (2, 130, 3, 1, 37, 53),
         (1, 450, 2, 1, 128, 128), (2, 100, 2, 2, 128, 48), (1, 130, 1, 1, 256, 256),
         (2, 90, 2, 1, 200, 50), (1, 2000, 1, 1, 64, 128)]
F16 = torch.float16


def _state(pair, most, steps, k, v, weight=1.0):
    """The bound without what values below binary16's smallest lose: a weighted
    value is the sum of two of binary16, after its column of a block was brought to
    2^14 at least: half of 2^-24 there is 2^-39 of the column's largest."""
    value, size = pair
    count = plain.state_operations(most, F16)
    lost = steps * k.abs().max() * v.abs().max() * weight * 2.0 ** -39
    return (value, size + lost / (count * ref.F32)), count


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("factor", [1e-3, 1e-4, 1e-5, 2e4])
@pytest.mark.parametrize("state", [False, True])
def test_states_of_values(size, factor, state):
    t, _ = _make(size, F16, resets=True, state=state)
    t["v"] = (t["v"].float() * factor).clamp(-65504, 65504).to(F16)
    if state:
        t["initial_state"] *= factor
    o, last = ops.linear_attention(scale=0.1, **_cuda(t))
    # (float32: the magnitude alone)
    want = plain.attention(scale=0.1, dtype=torch.float32, **_wide(t))[1]
    pair, count = _state(want, max(size[4:]), size[1], t["k"].double(),
                         t["v"].double())
    ref.check(last, pair, count)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("factor,scale", [(1e-3, 0.1), (1e-4, 0.1), (1e-5, 0.1),
                                          (1.0, 1e-4), (1.5e4, 8.0)])
def test_states_of_gradients(size, factor, scale):
    """The last: scale times a value of the gradient is beyond 65504."""
    t, (do, _) = _make(size, F16, resets=True, state=False)
    do = (do.float() * factor).clamp(-65504, 65504).to(F16)
    got = ops.linear_attention_grad(do.cuda(), scale=scale, **_cuda(t))
    want = plain.attention_grad(do.double(), scale=scale, dtype=torch.float32,
                                **_wide(t))["initial_state"]
    pair, count = _state(want, max(size[4:]), size[1], t["q"].double(),
                         do.double(), scale)
    ref.check(got["initial_state"], pair, count)


@pytest.mark.parametrize("factor", [1e-4, 2e-7])
def test_states_of_keys(factor):
    """Keys are an operand as they are, those below 2^-14 too."""
    size = (2, 150, 2, 2, 64, 72)
    t, _ = _make(size, F16, state=False)
    t["k"] = (t["k"].float() * factor).to(F16)
    _, last = ops.linear_attention(**_cuda(t))
    want = plain.attention(dtype=torch.float32, **_wide(t))[1]
    pair, count = _state(want, 72, 150, t["k"].double(), t["v"].double())
    ref.check(last, pair, count)


@pytest.mark.parametrize("factor", [100.0, 10.0])
def test_a_block_of_small_values_behind_large_ones(factor):
    """Small values join a state of large ones, and after a reset are all of it.  A
    column of the first factor's is infinite up to there."""
    size = (2, 200, 2, 2, 40, 72)
    t, _ = _make(size, F16, state=False)
    t["v"][:, :64] *= 1000.0
    t["v"][:, 64:] *= 1e-4
    t["v"][..., 5] *= factor
    infinite = bool(t["v"].isinf().any())
    assert infinite == (factor == 100.0)
    for reset in (False, True):
        if reset:
            t["resets"] = torch.zeros(2, 200, dtype=torch.uint8)
            t["resets"][:, 70] = 1
        _, last = ops.linear_attention(**_cuda(t))
        want = plain.attention(dtype=torch.float32, **_wide(t))[1]
        columns = torch.ones(72, dtype=torch.bool)
        if infinite and not reset:
            assert not torch.isfinite(last[..., 5]).any()
            columns[5] = False
        # (values in front of a reset are left out before the range is taken)
        part = t["v"].double()[:, 70 if reset else 0:][..., columns]
        pair, count = _state(tuple(x[..., columns] for x in want), 72, 200,
                             t["k"].double(), part)
        ref.check(last.cpu()[..., columns], pair, count)
