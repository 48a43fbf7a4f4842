"""Positions by rotation against 64 bits: two products and their sum, of sines and
cosines that are off by a few units of an angle that far positions leave 2^-24
turns of."""
import pytest
import torch

import attention_reference as plain
import sequence_reference as ref
from portdnn_amd import ops
from portdnn_amd.ops import ROTARY, ROTARY_SCALING

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
OPERATIONS = 64
# batch, steps, heads, channels, turned
SIZES = [(1, 1, 1, 2, 2), (2, 3, 2, 16, 16), (3, 5, 4, 64, 64), (2, 7, 3, 36, 20),
         (2, 33, 2, 128, 64), (1, 100, 5, 17, 10), (64, 1, 8, 128, 128),
         (1, 65, 1, 255, 254), (2, 4, 40, 256, 8)]


def _normal(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(shape, generator=g).to(dtype)


def _check(x, table, at, layout, positions=None, **kinds):
    y = ops.rotary(x.cuda(), table.cuda(), positions=positions, layout=layout,
                   **kinds)
    want = plain.rotary(x.double(), table, at, layout == ROTARY.HALVES, **kinds)
    ref.check(y, want, OPERATIONS, "%s" % (tuple(x.shape),))
    n = 2 * table.numel()
    assert torch.equal(y[..., n:].cpu(), x[..., n:])
    return y


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", [ROTARY.HALVES, ROTARY.PAIRS])
def test_sizes(size, dtype, layout):
    batch, steps, heads, channels, turned = size
    x = _normal(size[:4], dtype)
    table = plain.frequencies(turned)
    at = torch.arange(steps).expand(batch, steps)
    y = _check(x, table, at, layout)
    # back again, where each of the two roundings counts
    back = ops.rotary(y, table.cuda(), layout=layout, inverse=True)
    want = plain.rotary(y.cpu().double(), table, at, layout == ROTARY.HALVES,
                        inverse=True)
    ref.check(back, want, OPERATIONS)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", [ROTARY.HALVES, ROTARY.PAIRS])
def test_positions(dtype, layout):
    batch, steps = 4, 9
    x = _normal((batch, steps, 3, 40), dtype)
    table = plain.frequencies(32)
    first = torch.tensor([0, -5, 131072, 2 ** 31 - 10], dtype=torch.int32)
    at = first.long()[:, None] + torch.arange(steps)
    _check(x, table, at, layout, positions=first.cuda(), magnitude=1.25)
    g = torch.Generator().manual_seed(3)
    each = torch.randint(-2 ** 31, 2 ** 31 - 1, (batch, steps), generator=g)
    each[0] = 0
    each[1, :2] = torch.tensor([2 ** 31 - 1, -2 ** 31])
    _check(x, table, each, layout, positions=each.int().cuda(), magnitude=-0.5,
           inverse=True)


@pytest.mark.parametrize("scaling", ["NONE", "POSITIONS", "BASE", "BANDS"])
def test_tables(scaling):
    kinds = dict(base=50000.0, factor=8.0, context=1024.0, low=1.0, high=32.0)
    for turned in (2, 4, 64, 250):
        got = ops.rotary_frequencies(turned, scaling=getattr(ROTARY_SCALING,
                                                             scaling), **kinds)
        want = plain.frequencies(turned, scaling=scaling, **kinds)
        assert got.is_cuda and got.dtype is torch.float64
        # (a power and a handful of operations in 64 bits)
        torch.testing.assert_close(got.cpu(), want, rtol=1e-13, atol=0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", [ROTARY.HALVES, ROTARY.PAIRS])
def test_in_place_and_slices(dtype, layout):
    """Slices of a projection, in place, at addresses that are a multiple of
    nothing; what is around them stays."""
    batch, steps, heads, channels = 2, 21, 3, 48
    x = _normal((batch, steps, heads, channels), dtype).cuda()
    table = plain.frequencies(32).cuda()
    want = ops.rotary(x, table, layout=layout)
    n = heads * channels
    for first in (0, 8, 5):
        p = torch.full((batch, steps, n + 16), 3.0, dtype=dtype, device="cuda")
        part = p[..., first:first + n].unflatten(2, (heads, channels))
        part.copy_(x)
        assert torch.equal(ops.rotary(part, table, layout=layout), want)
        got = ops.rotary(part, table, layout=layout, out=part)
        assert got is part and torch.equal(part, want)
        assert (p[..., :first] == 3.0).all() and (p[..., first + n:] == 3.0).all()
    out = torch.full((batch, steps, n + 16), 3.0, dtype=dtype, device="cuda")
    part = out[..., 8:8 + n].unflatten(2, (heads, channels))
    ops.rotary(x, table, layout=layout, out=part)
    assert torch.equal(part, want)
    assert (out[..., :8] == 3.0).all() and (out[..., 8 + n:] == 3.0).all()


def test_values_that_are_not_finite():
    """They stay in their pair."""
    x = _normal((1, 4, 2, 16), torch.float32)
    table = plain.frequencies(12).cuda()
    want = ops.rotary(x.cuda(), table)
    bad = x.clone()
    bad[0, 1, 0, 2] = float("nan")
    bad[0, 2, 1, 7] = float("inf")
    bad[0, 3, 1, 15] = float("inf")  # is not turned
    got = ops.rotary(bad.cuda(), table)
    hit = torch.zeros(x.shape, dtype=torch.bool)
    hit[0, 1, 0, [2, 8]] = True
    hit[0, 2, 1, [1, 7]] = True
    hit[0, 3, 1, 15] = True
    assert torch.equal(torch.isfinite(got).cpu(), ~hit)
    assert torch.equal(got.cpu()[~hit], want.cpu()[~hit])


def test_streams_and_graphs():
    x = _normal((2, 50, 4, 64), torch.bfloat16).cuda()
    other = x.flip(1).contiguous()
    table = plain.frequencies(64).cuda()
    at = torch.tensor([3, 70], dtype=torch.int32).cuda()
    want = [ops.rotary(t, table, positions=at) for t in (x, other)]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = ops.rotary(x, table, positions=at)
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    t = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary(t, table, positions=at)
    for turn in (0, 1, 0):
        t.copy_((x, other)[turn])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[turn])
        ops.rotary(other, table)


def test_more_than_31_bits_of_elements():
    """1100 steps of 2^21 channels: the last rows are the same as by themselves."""
    batch, steps, heads, channels = 1, 1100, 8192, 256
    x = torch.empty(batch, steps, heads, channels, dtype=torch.bfloat16,
                    device="cuda")
    x.normal_()
    table = plain.frequencies(256).cuda()
    y = ops.rotary(x, table)
    tail = x[:, -2:].contiguous()
    first = torch.tensor([steps - 2], dtype=torch.int32).cuda()
    assert torch.equal(y[:, -2:], ops.rotary(tail, table, positions=first))
