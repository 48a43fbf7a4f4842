"""The activations and their slopes far out, against 64 bits.

A product of one term with a factor of one is the value itself, so that the
forward call returns act(z) of an exact z; the bias's gradient of a single row is
the slope at z, in fp32 and rounded once.

Bounds, relative to what the value would be if its terms had one sign.  An
exponential of an argument w that is itself rounded a few times is off by some
units of |w| 2^-24: eight of them (the argument's rounding, three products in front
of it, the hardware's product with log2(e), and as much again); sixteen more
operations of 2^-24 around it.  What is below 1e-37 may be a zero.
"""
import math

import pytest
import torch

from portdnn_amd import ops
from portdnn_amd.ops import ACTIVATION

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
         torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 1e-37, torch.float16: 2.0 ** -25,
         torch.bfloat16: 1e-37}
C = math.sqrt(8.0 / math.pi)


def _terms(z, kind):
    """(value, magnitude, |argument of the exponential|) of act and of its slope."""
    one, zero = torch.ones_like(z), torch.zeros_like(z)
    if kind == "NONE":
        return (z, z.abs(), zero), (one, one, zero)
    if kind == "RELU":
        on = (z > 0).double()
        return (z * on, z.abs() * on, zero), (on, on, zero)
    if kind == "GELU":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        density = torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
        w = 0.5 * z * z
        return ((z * phi, z.abs() * phi, w),
                (phi + z * density, phi + z.abs() * density, w))
    w = z if kind == "SILU" else C * (z + 0.044715 * z ** 3)
    dw = one if kind == "SILU" else C * (1.0 + 0.134145 * z * z)
    s, rest = torch.sigmoid(w), torch.sigmoid(-w)
    slope = z * (s * rest) * dw
    return ((z * s, z.abs() * s, w.abs()),
            (s + slope, s + slope.abs(), w.abs()))


def _check(got, terms, what):
    value, magnitude, w = terms
    got_type = got.dtype
    got = got.cpu().double().flatten()
    # (an exponential that is nothing has no error)
    error = (16.0 + 8.0 * torch.clamp(w, max=200.0)) * F32 * magnitude
    bound = (ROUND[got_type] * value.abs() + LEAST[got_type] +
             (1.0 + ROUND[got_type]) * error)
    off = (got - value).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, [
        (got[i].item(), value[i].item(), bound[i].item())
        for i in bad.nonzero().flatten()[:5].tolist()])


def _values(dtype):
    far = [0.0, 1e-3, 0.5, 1.0, 2.0, 3.0, 4.0, 5.0, 6.0, 8.0, 9.3, 12.0, 13.0,
           16.0, 20.0, 40.0, 64.0, 89.0, 104.0, 1e3, 1e4, 6e4]
    if dtype != torch.float16:
        far += [1e6, 1e12, 1.8e19, 1.9e19, 1e20, 1e25, 1e30, 3e38]
    z = torch.cat([torch.tensor(far), -torch.tensor(far),
                   torch.linspace(-14.0, 14.0, 1801)])
    return z.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["NONE", "RELU", "GELU", "GELU_TANH", "SILU"])
def test_values_and_slopes_far_out(dtype, kind):
    z = _values(dtype)
    act = getattr(ACTIVATION, kind)
    one = torch.ones(1, 1, dtype=dtype, device="cuda")
    row = z.cuda()[None]
    y, kept = ops.matmul_bias_act(one, row, activation=act,
                                  keep_pre_activation=True)
    assert torch.equal(kept, row)
    value, slope = _terms(z.double(), kind)
    _check(y, value, kind)
    dy = torch.ones_like(row)
    _, _, bias = ops.matmul_bias_act_grad(dy, one, row, row, activation=act,
                                          need_a=False, need_b=False)
    _check(bias, slope, kind + " slope")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["GELU", "GELU_TANH", "SILU"])
def test_one_value_far_out_spoils_no_gradient(dtype, kind):
    """Rows and columns of the products beside it are as if it were merely large."""
    act = getattr(ACTIVATION, kind)
    g = torch.Generator().manual_seed(1)
    a, b, dy, z = (torch.randn(s, generator=g).to(dtype) for s in
                   ((40, 24), (24, 72), (40, 72), (40, 72)))
    for sign in (1.0, -1.0):
        both = []
        for far in (100.0, 1e30):
            z[3, 5] = sign * far
            both.append(ops.matmul_bias_act_grad(
                dy.cuda(), a.cuda(), b.cuda(), z.cuda(), activation=act))
        for large, far_out in zip(*both):
            assert far_out.isfinite().all() and torch.equal(large, far_out)
