"""The 64-bit references of the sequence operators' tests: their gradients are
the differences of their forward values."""
import pytest
import torch

import sequence_reference as ref


def _difference(f, v, direction, step=1e-6):
    return (f(v + step * direction) - f(v - step * direction)) / (2 * step)


def _agree(f, v, gradient, g, scale=1.0):
    """f's change along a random direction against its gradient.  The error of
    a central difference is step^2 of the third derivative and 1e-16 / step of
    f, both far below 1e-6 of these sums."""
    d = torch.randn(v.shape, generator=g, dtype=torch.float64)
    want = _difference(f, v, d)
    got = (gradient * d).sum()
    size = (gradient * d).abs().sum() + scale
    assert abs(got - want) <= 1e-6 * size


@pytest.mark.parametrize("kind", ref.ACTIVATIONS)
def test_matmul_gradients_are_differences(kind):
    g = torch.Generator().manual_seed(1)
    a, b, c, dy = (torch.randn(s, generator=g, dtype=torch.float64)
                   for s in ((5, 7), (7, 4), (4,), (5, 4)))
    z = a @ b + c
    da, db, dc = ref.matmul_grad(dy, a, b, z, kind, torch.float32)

    def loss(a, b, c):
        return (dy * ref.matmul(a, b, c, kind=kind)[0][0]).sum()

    _agree(lambda v: loss(v, b, c), a, da[0], g)
    _agree(lambda v: loss(a, v, c), b, db[0], g)
    _agree(lambda v: loss(a, b, v), c, dc[0], g)


@pytest.mark.parametrize("post", ["NONE", "RMS", "LAYER"])
@pytest.mark.parametrize("pre", ["RMS", "LAYER"])
@pytest.mark.parametrize("gate_op,gate_rows",
                         [("VALUE", 1), ("SIGMOID", 3), ("SILU", 2)])
def test_norm_gradients_are_differences(post, pre, gate_op, gate_rows):
    g = torch.Generator().manual_seed(2)
    rows, channels = 5, 6

    def normal(*shape):
        return torch.randn(shape, generator=g, dtype=torch.float64)

    t = {"x": normal(rows, channels), "residual": normal(rows, channels),
         "gate": normal(-(-rows // gate_rows), channels),
         "scale": normal(channels), "pre_weight": normal(channels),
         "pre_bias": normal(channels)}
    if post != "NONE":
        t["post_weight"], t["post_bias"] = normal(channels), normal(channels)
    kinds = {"post": post, "pre": pre, "gate_op": gate_op,
             "gate_rows": gate_rows, "eps": 1e-3}
    dy, du = normal(rows, channels), normal(rows, channels)
    (y, _), _, stats = ref.residual_norm(**t, **kinds)
    given = {k: v for k, v in t.items() if k != "residual"}
    got = ref.residual_norm_grad(y=y, stats=stats, dy=dy, du=du, **given,
                                 **kinds)
    for name in t:
        def loss(v):
            (y, _), (u, _), _ = ref.residual_norm(**{**t, name: v}, **kinds)
            return (dy * y).sum() + (du * u).sum()
        _agree(loss, t[name], got[name][0], g)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_recurrence_gradients_are_differences(gated, masked):
    g = torch.Generator().manual_seed(3)
    batch, steps, channels = 3, 9, 4

    def normal(*shape):
        return torch.randn(shape, generator=g, dtype=torch.float64)

    t = {"x": normal(batch, steps, channels),
         "f": normal(batch, steps, channels), "h0": normal(batch, channels)}
    if gated:
        t["i"] = normal(batch, steps, channels)
    masks = {}
    if masked:
        masks = {"resets": (torch.rand(batch, steps, generator=g) < 0.3),
                 "lengths": torch.tensor([0, 5, 9])}
    dh, d_last = normal(batch, steps, channels), normal(batch, channels)
    (h, _), _ = ref.recurrence(**t, **masks)
    got = ref.recurrence_grad(dh, h=h, d_last=d_last, **t, **masks)
    names = {"x": "x", "f": "forget", "i": "input_gate", "h0": "initial_state"}
    for name in t:
        def loss(v):
            (h, _), (last, _) = ref.recurrence(**{**t, name: v}, **masks)
            return (dh * h).sum() + (d_last * last).sum()
        _agree(loss, t[name], got[names[name]][0], g)
