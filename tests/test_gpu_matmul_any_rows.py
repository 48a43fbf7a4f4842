"""Products of operands whose rows start anywhere, in tiles by way of registers:
ends of the reduction and of the rows inside a tile, surroundings that are NaN,
against 64 bits.  A product of k terms is a chain of k + a few fp32 operations."""
import pytest
import torch

import sequence_reference as ref
from portdnn_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# whole chunks, one value more or less, one chunk, a few values, several tiles
SHAPES = [(1025, 130, 513), (641, 129, 1001), (700, 127, 1003), (1023, 33, 777),
          (513, 8, 2049), (2049, 9, 515), (385, 575, 899), (1153, 64, 639)]


def _surrounded(t, shift):
    rows, cols = t.shape
    wide = torch.full((rows + 2, cols + 5), float("nan"), dtype=t.dtype,
                      device="cuda")
    view = wide[1:-1, shift:shift + cols]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans_a,trans_b", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_at_any_address(dtype, trans_a, trans_b, shape):
    m, k, n = shape
    g = torch.Generator().manual_seed(m + k)
    a = torch.randn((k, m) if trans_a else (m, k), generator=g).to(dtype)
    b = torch.randn((n, k) if trans_b else (k, n), generator=g).to(dtype)
    bias = torch.randn(n, generator=g).to(dtype)
    got = ops.matmul_bias_act(_surrounded(a, 1), _surrounded(b, 3),
                              bias=bias.cuda(), trans_a=trans_a,
                              trans_b=trans_b)
    a, b = a.double(), b.double()
    want, _ = ref.matmul(a.t() if trans_a else a, b.t() if trans_b else b,
                         bias.double())
    ref.check(got, want, k + 64, "%dx%dx%d" % shape)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_room_for_copies(dtype):
    g = torch.Generator().manual_seed(1)
    a, b = (torch.randn(1500, 1001, generator=g).to(dtype),
            torch.randn(1001, 703, generator=g).to(dtype))
    none = torch.empty(0, dtype=dtype, device="cuda")
    got = ops.matmul_bias_act(a.cuda(), b.cuda(), workspace=none)
    want, _ = ref.matmul(a.double(), b.double())
    ref.check(got, want, 1001 + 64)
