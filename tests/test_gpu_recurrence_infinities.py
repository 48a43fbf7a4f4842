"""Infinite states, inputs and gradients in divided sequences: the same as in the walk
step by step, and as 64 bits say."""
import pytest
import torch

import sequence_reference as ref
from portdnn_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


def _kinds(t):
    """0: finite, 1: inf, 2: -inf, 3: NaN."""
    t = t.detach().cpu().double()
    kind = torch.zeros(t.shape, dtype=torch.int64)
    kind[t == INF], kind[t == -INF], kind[t.isnan()] = 1, 2, 3
    return kind


def _make(dtype, steps, channels, logit, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = {"x": torch.randn(2, steps, channels, generator=g),
         "forget": torch.randn(2, steps, channels, generator=g) + logit}
    return g, {k: v.to(dtype) for k, v in t.items()}


def _both_ways(t, dtype, dh, d_last):
    """(outputs with the recommended workspace, without one), as dicts."""
    gpu = {k: v.cuda() for k, v in t.items()}
    found = []
    for workspace in (None, torch.empty(0, dtype=dtype, device="cuda")):
        h, last = ops.linear_recurrence(**gpu, workspace=workspace)
        # (the gradients of the same h)
        first = h if not found else found[0]["h"]
        got = ops.linear_recurrence_grad(
            dh.cuda(), h=first, grad_final_state=d_last.cuda(),
            workspace=workspace, **gpu)
        found.append({"h": h, "last": last,
                      **{"d_" + k: v for k, v in got.items()}})
    return found


def _same_kinds(divided, whole, what):
    for name, v in divided.items():
        apart = _kinds(v) != _kinds(whole[name])
        assert not apart.any(), (what, name, int(apart.sum()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("logit", [3.0, -1.0, -9.0])
def test_infinities_go_through_products_that_are_too_small(dtype, gated, logit):
    """(The product of 144 gates of a logit of -1 is 1e-82, of twelve of -9 1e-47.)"""
    steps, channels = 700, 72
    g, t = _make(dtype, steps, channels, logit)
    if gated:
        t["input_gate"] = torch.randn(2, steps, channels, generator=g).to(dtype)
    state = torch.randn(2, channels, generator=g)
    state[0, 3], state[0, 4], state[1, 70] = INF, -INF, INF
    t["initial_state"] = state
    t["x"][0, 20, 7], t["x"][1, 500, 8] = INF, -INF
    t["x"][0, 600, 3] = -INF  # meets the state's infinity
    dh = torch.randn(2, steps, channels, generator=g).to(dtype)
    dh[0, 650, 11], dh[1, 200, 12] = INF, -INF
    d_last = torch.randn(2, channels, generator=g)
    d_last[0, 13], d_last[1, 14] = INF, -INF
    divided, whole = _both_ways(t, dtype, dh, d_last)
    _same_kinds(divided, whole, "logit %g" % logit)
    want_h, want_last = ref.recurrence(
        t["x"].double(), t["forget"].double(),
        t["input_gate"].double() if gated else None, h0=state.double())
    assert torch.equal(_kinds(divided["h"]), _kinds(want_h[0]))
    assert torch.equal(_kinds(divided["last"]), _kinds(want_last[0]))
    assert (_kinds(divided["h"])[0, :, 4] == 2).all()
    assert (_kinds(divided["h"])[0, 20:, 7] == 1).all()
    assert (_kinds(divided["last"])[0, 3] == 3)
    # the gradient's infinity reaches every step before it, and the state's
    assert (_kinds(divided["d_x"])[0, :651, 11] == 1).all()
    assert (_kinds(divided["d_x"])[0, :, 13] == 1).all()
    assert _kinds(divided["d_initial_state"])[1, 12] == 2
    # channels without one are the same to rounding
    clean = torch.ones(channels, dtype=torch.bool)
    clean[[3, 4, 7, 8, 11, 12, 13, 14, 70]] = False
    for name, v in divided.items():
        a, b = (d[name][..., clean.cuda()].double().cpu()
                for d in (divided, whole))
        assert a.isfinite().all()
        # (64 operations in a row, and the rounding of the type)
        near = 2 * (64 * ref.F32 + ref.ROUND[v.dtype])
        assert ((a - b).abs() <= near * a.abs() + 64 * ref.F32 * 16).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_shut_gates_and_resets_behind_infinities(dtype):
    """A sigmoid is above zero, also where fp32 has no value for it; a reset forgets."""
    steps, channels = 700, 40
    g, t = _make(dtype, steps, channels, -2.0, seed=2)
    state = torch.randn(2, channels, generator=g)
    state[0, 5], state[1, 6] = INF, -INF
    t["initial_state"] = state
    t["x"][0, 100, 9] = INF
    t["forget"][0, 400], t["forget"][0, 101, 9] = -200.0, -95.0
    t["resets"] = torch.zeros(2, steps, dtype=torch.uint8)
    t["resets"][0, 550] = 1
    t["resets"][1, 300] = 1
    dh = torch.randn(2, steps, channels, generator=g).to(dtype)
    dh[0, 540, 20], dh[0, 660, 21] = INF, INF
    d_last = torch.randn(2, channels, generator=g)
    divided, whole = _both_ways(t, dtype, dh, d_last)
    _same_kinds(divided, whole, "shut gates")
    want_h, want_last = ref.recurrence(
        t["x"].double(), t["forget"].double(), resets=t["resets"],
        h0=state.double())
    kinds = _kinds(divided["h"])
    assert torch.equal(kinds, _kinds(want_h[0]))
    assert torch.equal(_kinds(divided["last"]), _kinds(want_last[0]))
    assert (kinds[0, :550, 5] == 1).all() and (kinds[0, 100:550, 9] == 1).all()
    assert not kinds[0, 550:].any() and not kinds[1, 300:].any()
    assert (_kinds(divided["d_initial_state"])[0] != 0).nonzero().tolist() == [[20]]


@pytest.mark.parametrize("dtype", TYPES)
def test_the_largest_finite_states_are_forgotten(dtype):
    """Products too small for fp32 leave next to nothing of 1e38."""
    steps, channels = 700, 64
    g, t = _make(dtype, steps, channels, -3.0, seed=3)
    t["initial_state"] = torch.full((2, channels), 1e38)
    h, last = ops.linear_recurrence(**{k: v.cuda() for k, v in t.items()})
    want_h, want_last = ref.recurrence(
        t["x"].double(), t["forget"].double(),
        h0=t["initial_state"].double())
    # (two units of the smallest value times the state)
    for got, (value, size) in ((h[:, 300:], [v[:, 300:] for v in want_h]),
                               (last, want_last)):
        off = (got.cpu().double() - value).abs()
        near = (2.0 ** -148 * 1e38 + ref.ROUND[got.dtype] * value.abs() +
                ref.LEAST[got.dtype] + 2 * 64 * ref.F32 * size)
        assert (off <= near).all()
