"""Products that reach every kernel of matmul_bias_act, in all orders of their operands
in memory, with copies in front and shares of the reduction, against 64 bits.  What
surrounds the operands is NaN.  A product of k terms is a chain of k + a few fp32
operations."""
import pytest
import torch

import sequence_reference as ref
from matmul_kernel_cases import CASES
from portdnn_amd import ops
from portdnn_amd.ops import ACTIVATION
from test_matmul_plans import TYPES, planned

pytestmark = pytest.mark.gpu

EXTRA = 64  # operations of the epilogue and of joining shares


def _placed(t, pad, aligned):
    """t on the GPU, `pad` values between its rows, from a multiple of 16 bytes on or
    a value behind one."""
    rows, cols = t.shape
    step = cols + pad
    flat = torch.full((rows * step + 64,), float("nan"), dtype=t.dtype,
                      device="cuda")
    view = flat[0 if aligned else 1:].as_strided((rows, cols), (step, 1))
    view.copy_(t)
    assert (view.data_ptr() % 16 == 0) == bool(aligned)
    return view


@pytest.mark.parametrize("at", range(len(CASES)))
def test_case(at):
    c = CASES[at]
    for dtype in TYPES[c.type]:
        p = planned(c, dtype)
        assert (p["tile_rows"], p["tile_cols"], p["shared"], p["any_address"],
                p["pair"]) == c.kernel
        g = torch.Generator().manual_seed(at)
        a = torch.randn((c.k, c.m) if c.trans_a else (c.m, c.k),
                        generator=g).to(dtype)
        b = (torch.randn((c.n, c.k) if c.trans_b else (c.k, c.n), generator=g) *
             c.k ** -0.5).to(dtype)
        bias = torch.randn(c.n, generator=g).to(dtype)
        add = torch.randn(c.m, c.n, generator=g).to(dtype)
        kind = ref.ACTIVATIONS[at % 5]
        y, z = ops.matmul_bias_act(
            _placed(a, c.pad_a, c.aligned), _placed(b, c.pad_b, c.aligned),
            bias=bias.cuda(), residual=add.cuda(),
            activation=getattr(ACTIVATION, kind), trans_a=c.trans_a,
            trans_b=c.trans_b, keep_pre_activation=True,
            workspace=None if c.workspace else
            torch.empty(0, dtype=dtype, device="cuda"))
        a, b = a.double(), b.double()
        want_y, want_z = ref.matmul(a.t() if c.trans_a else a,
                                    b.t() if c.trans_b else b, bias.double(),
                                    add.double(), kind)
        ref.check(z, want_z, c.k + EXTRA, "%s z" % (c,))
        ref.check(y, want_y, c.k + EXTRA, "%s" % (c,))
