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
# batch, steps, heads, key_heads, keys, values: up to 12 steps, blocks, pieces; each
# way into LDS, four waves and eight
SIZES = [(1, 5, 2, 2, 24, 40), (2, 12, 2, 2, 100, 72), (1, 200, 2, 2, 24, 40),
         (2, 130, 2, 2, 37, 53), (1, 450, 1, 1, 64, 128), (1, 385, 1, 1, 128, 48),
         (1, 130, 1, 1, 256, 256), (2, 90, 1, 1, 200, 40), (1, 450, 1, 1, 128, 128)]
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


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients(size, dtype):
    """A state in front that is infinite has it in a channel of q's gradient, the
    gradient of the state behind in one of k's, one of v's and its own."""
    t, (do, ds) = _make(size, dtype)
    for x in (t["k"], t["v"], do):
        x[x == 0] = 1.0
    bad = {**t, "initial_state": t["initial_state"].clone()}
    bad["initial_state"][:, :, KEY, VALUE] = INF
    bad_ds = ds.clone()
    bad_ds[:, :, KEY, VALUE] = -INF
    got = ops.linear_attention_grad(do.cuda(), grad_final_state=bad_ds.cuda(),
                                    **_cuda(bad))
    want = plain.attention_grad(do.double(), grad_final_state=ds.double(),
                                dtype=dtype, **_wide(t))
    _signs(got["q"][..., KEY], do[..., VALUE], 1.0)
    _signs(got["k"][..., KEY], t["v"][..., VALUE], -1.0)
    _signs(got["v"][..., VALUE], t["k"][..., KEY], -1.0)
    assert (got["initial_state"][:, :, KEY, VALUE] == -INF).all()
    most = max(size[4:])
    for name, at in (("q", KEY), ("k", KEY), ("v", VALUE)):
        part = [c for c in range(got[name].shape[3]) if c != at]
        ref.check(got[name][..., part], [x[..., part] for x in want[name]],
                  plain.operations(most, dtype), name)
    first = got["initial_state"].cpu()
    first[:, :, KEY, VALUE] = want["initial_state"][0][:, :, KEY, VALUE].float()
    ref.check(first, want["initial_state"], plain.state_operations(most, dtype))


@pytest.mark.parametrize("steps", [5, 12, 13, 70, 200, 900])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keys,values", [(1, 5), (1, 64), (3, 72), (65, 9), (130, 130)])
def test_values(steps, dtype, keys, values):
    """Queries and keys above zero and an infinite value: keys that pad a head take
    nothing from it."""
    g = torch.Generator().manual_seed(steps + keys)
    q = (0.5 + torch.rand(1, steps, 1, keys, generator=g)).to(dtype)
    k = (0.5 + torch.rand(1, steps, 1, keys, generator=g)).to(dtype)
    v = torch.randn(1, steps, 1, values, generator=g).to(dtype)
    at = steps // 2
    v[0, at, 0, 2] = -INF
    o, last = ops.linear_attention(q.cuda(), k.cuda(), v.cuda(),
                                   torch.tensor([-0.02]).cuda())
    o, last = o.float().cpu(), last.cpu()
    assert (o[0, at:, 0, 2] == -INF).all()
    assert (last[0, 0, :, 2] == -INF).all()
    o[0, at:, 0, 2] = 0.0
    last[0, 0, :, 2] = 0.0
    assert torch.isfinite(o).all() and torch.isfinite(last).all()


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [3.4e38, -3.3999e38])
def test_states_that_rounding_would_make_infinite(size, dtype, value):
    """fp32 values beyond the largest of bfloat16."""
    t, _ = _make(size, dtype)
    t["initial_state"][:, :, KEY, VALUE] = value
    # (at most 1e34 of a state that large, in front of the scale)
    t["q"][..., KEY] = (t["q"][..., KEY].float() * 1e-5).to(dtype)
    o, last = ops.linear_attention(scale=0.5, **_cuda(t))
    want = plain.attention(scale=0.5, dtype=dtype, **_wide(t))
    most = max(size[4:])
    ref.check(o, want[0], plain.operations(most, dtype))
    ref.check(last, want[1], plain.state_operations(most, dtype))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_states_of_nothing_else(size, dtype):
    """All of a column but one key is zero, and decays take what there was from all
    others: a range that small times a decay may be no number above zero."""
    t, _ = _make(size, dtype)
    t["decay"][:] = -2.0
    t["q"][..., KEY] = 1.0
    t["initial_state"].zero_()
    t["initial_state"][:, :, KEY, VALUE] = INF
    t["v"][..., VALUE] = 0.0
    o, last = ops.linear_attention(scale=1e-3, **_cuda(t))
    o = o.float().cpu()
    assert (o[..., VALUE] == INF).all()
    assert torch.isfinite(o[..., _others(size[5])]).all()
    assert (last[:, :, KEY, VALUE] == INF).all()
