"""Gated products and their input's gradients that reach every kernel, in both orders
of the weights in memory, with copies in front and shares of the reduction, against 64
bits.  What surrounds the operands is NaN.  A product of k terms is a chain of k + a few
fp32 operations; the gradients' factors are rounded to the data type once."""
import pytest
import torch

import attention_reference as plain
import sequence_reference as ref
from gated_kernel_cases import CASES
from portdnn_amd import ops
from portdnn_amd.ops import ACTIVATION
from test_gated_plans import TYPES, kernel_of, planned
from test_gpu_matmul_every_kernel import _placed

pytestmark = pytest.mark.gpu

EXTRA = 64  # operations of the epilogue and of joining shares


def _check(got, pair, operations, what):
    ref.check(got, tuple(x.cpu() for x in pair), operations, what)


@pytest.mark.parametrize("at", range(len(CASES)))
def test_case(at):
    c = CASES[at]
    kind = ref.ACTIVATIONS[at % 5]
    act = getattr(ACTIVATION, kind)
    for dtype in TYPES[c.type]:
        assert kernel_of(planned(c, dtype)) == c.kernel
        g = torch.Generator().manual_seed(at)

        def normal(*shape, size=1.0):
            return (size * torch.randn(shape, generator=g)).to(dtype)

        stored = (c.n, c.k) if c.trans_b else (c.k, c.n)
        x = normal(c.m, c.k)
        weights = [normal(*stored, size=c.k ** -0.5) for _ in range(2)]
        placed = [_placed(x, c.pad_a, c.aligned)] + [
            _placed(w, c.pad_b, c.aligned) for w in weights]
        # (the references in 64 bits as well, where the products are quick)
        X, G, U = (t.double().cuda() for t in [x] + weights)
        if c.trans_b:
            G, U = G.T, U.T
        if c.product == 0:
            biases = [normal(c.n), normal(c.n)] if at % 3 else [None, None]
            got = ops.gated_matmul(
                *placed, *(b if b is None else b.cuda() for b in biases),
                activation=act, trans_b=c.trans_b, keep_pre_activation=True,
                workspace=None if c.workspace else
                torch.empty(0, dtype=dtype, device="cuda"))
            want = plain.gated(
                X, G, U, *(b if b is None else b.double().cuda() for b in biases),
                kind)
            for name, y, pair in zip(("out", "gate", "up"), got, want):
                _check(y, pair, c.k + EXTRA, "%s %s" % (c, name))
            continue
        dy, z, u = (normal(c.m, c.n).cuda() for _ in range(3))
        got = ops.gated_matmul_grad(dy, *placed, z, u, activation=act,
                                    trans_b=c.trans_b)
        want = plain.gated_grad(dy.double(), X, G, U, z.double(), u.double(), kind)
        lost = 1.01 * plain.per_rounding(dtype) + EXTRA
        terms = {"x": 2 * c.n, "gate": c.m, "up": c.m, "bias_gate": c.m,
                 "bias_up": c.m}
        # A factor d is taken as d (1 + e) + s, where e is half a step of the type and s
        # half of its smallest step, 2^-25 in binary16 (0 in the others): a product of
        # it with w is off by |w| 2^-25 more.  (First seen with a factor of 6e-7.)
        small = 2.0 ** -25 if dtype is torch.float16 else 0.0
        more = {"x": small * (G.abs() + U.abs()).sum(1),
                "gate": small * X.abs().sum(0)[:, None]}
        more["up"] = more["gate"]
        for y, (name, (value, size)) in zip(got, want.items()):
            operations = terms[name] + lost
            size = size + more.get(name, 0.0) / (operations * ref.F32)
            if c.trans_b and name in ("gate", "up"):
                value, size = value.T, size.T
            _check(y, (value, size), operations, "%s d%s" % (c, name))
