"""The gated product and its gradients against 64 bits.  A result is a sum of k
products in fp32, an activation that is off by a few units and a handful of
operations more; the gradients' factors are rounded to the data type once."""
import pytest
import torch

import attention_reference as plain
import sequence_reference as ref
from portdnn_amd import ops
from portdnn_amd.ops import ACTIVATION

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZES = [(1, 1, 1), (1, 64, 96), (1, 1024, 512), (3, 17, 5), (16, 128, 64),
         (17, 200, 130), (40, 96, 257), (64, 512, 128), (100, 33, 100),
         (129, 65, 127), (200, 136, 264), (300, 64, 520), (260, 1000, 72)]


def _make(m, k, n, dtype, trans_b=False, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed + m + k + n)

    def normal(*shape, size=1.0):
        return (size * torch.randn(shape, generator=g)).to(dtype)

    t = [normal(m, k)] + [
        normal(n, k, size=k ** -0.5) if trans_b else normal(k, n, size=k ** -0.5)
        for _ in range(2)]
    t += [normal(n), normal(n)] if bias else [None, None]
    return t, normal(m, n)


def _wide(t, trans_b):
    return [None if x is None else x.double().T if trans_b and i in (1, 2)
            else x.double() for i, x in enumerate(t)]


def _cuda(t):
    return [None if x is None else x.cuda() for x in t]


def _check(t, dy, trans_b, kind, what=""):
    dtype, (m, k) = t[0].dtype, t[0].shape
    n = dy.shape[1]
    act = getattr(ACTIVATION, kind)
    gpu = _cuda(t)
    out, z, u = ops.gated_matmul(*gpu, activation=act, trans_b=trans_b,
                                 keep_pre_activation=True)
    want = plain.gated(*_wide(t, trans_b), kind)
    for name, got, pair in zip(("out", "gate", "up"), (out, z, u), want):
        ref.check(got, pair, k + 32, "%s %s" % (what, name))
    # the gradients are those of the factors that the forward call left
    got = ops.gated_matmul_grad(dy.cuda(), *gpu[:3], z, u, activation=act,
                                trans_b=trans_b)
    want = plain.gated_grad(dy.double(), *_wide(t, trans_b)[:3],
                            z.cpu().double(), u.cpu().double(), kind)
    # (the factors are rounded, and each is off by some operations before)
    lost = 1.01 * plain.per_rounding(dtype) + 32
    terms = {"x": 2 * n, "gate": m, "up": m, "bias_gate": m, "bias_up": m}
    for g, (name, (value, size)) in zip(got, want.items()):
        if trans_b and name in ("gate", "up"):
            value, size = value.T, size.T
        ref.check(g, (value, size), terms[name] + lost,
                  "%s d%s" % (what, name))
    # a call that keeps nothing is the same
    assert torch.equal(out, ops.gated_matmul(*gpu, activation=act,
                                             trans_b=trans_b))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans_b", [False, True])
def test_sizes(size, dtype, trans_b):
    t, dy = _make(*size, dtype, trans_b)
    _check(t, dy, trans_b, "SILU", str(size))


@pytest.mark.parametrize("kind", ref.ACTIVATIONS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(5, 64, 48), (150, 72, 140)])
def test_activations(kind, dtype, size):
    t, dy = _make(*size, dtype, bias=False)
    _check(t, dy, False, kind, kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 20, 150])
def test_slices(dtype, m):
    """Both weights are halves of one matrix, the rows slices of a wider one, also
    at addresses that are a multiple of nothing; the output is a slice as well."""
    k, n = 96, 72
    t, dy = _make(m, k, n, dtype)
    gpu = _cuda(t)
    want = ops.gated_matmul(*gpu)
    for first in (0, 8, 3):
        a = torch.full((m, k + 16), 2.0, dtype=dtype, device="cuda")
        a[:, first:first + k] = gpu[0]
        both = torch.full((k, 2 * n + 16), 2.0, dtype=dtype, device="cuda")
        both[:, first:first + n] = gpu[1]
        both[:, first + n:first + 2 * n] = gpu[2]
        halves = (both[:, first:first + n], both[:, first + n:first + 2 * n])
        out = torch.full((m, n + 16), 2.0, dtype=dtype, device="cuda")
        got = ops.gated_matmul(a[:, first:first + k], *halves, *gpu[3:],
                               out=out[:, first:first + n])
        pair = plain.gated(*_wide(t, False))[0]
        ref.check(got, pair, k + 32)
        assert (out[:, :first] == 2.0).all() and (out[:, first + n:] == 2.0).all()
        if first == 0:
            assert torch.equal(got, want)
        rows = torch.zeros(m, n + 16, dtype=dtype, device="cuda")
        rows[:, first:first + n] = dy.cuda()
        _, z, u = ops.gated_matmul(*gpu, keep_pre_activation=True)
        d = ops.gated_matmul_grad(rows[:, first:first + n], a[:, first:first + k],
                                  *halves, z, u)
        wide = plain.gated_grad(dy.double(), *_wide(t, False)[:3],
                                z.cpu().double(), u.cpu().double())
        for g, (name, pair) in zip(d, wide.items()):
            ref.check(g, pair, 2 * n + m + 1.01 * plain.per_rounding(dtype) + 32,
                      name)


@pytest.mark.parametrize("size", [(3, 2048, 8192), (30, 1024, 16384)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans_b", [False, True])
def test_weights_larger_than_all_else(size, dtype, trans_b):
    t, _ = _make(*size, dtype, trans_b)
    got = ops.gated_matmul(*_cuda(t), trans_b=trans_b)
    ref.check(got, plain.gated(*_wide(t, trans_b))[0], size[1] + 32)


@pytest.mark.parametrize("size", [(2, 512, 64), (150, 513, 130), (64, 2048, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_without_a_workspace(size, dtype):
    t, _ = _make(*size, dtype)
    room = torch.empty(0, dtype=dtype, device="cuda")
    got = ops.gated_matmul(*_cuda(t), workspace=room)
    ref.check(got, plain.gated(*_wide(t, False))[0], size[1] + 32)


def test_parts_that_are_not_wanted():
    t, dy = _make(70, 48, 56, torch.float32)
    gpu, dy = _cuda(t), dy.cuda()
    _, z, u = ops.gated_matmul(*gpu, keep_pre_activation=True)
    want = ops.gated_matmul_grad(dy, *gpu[:3], z, u)
    for kinds in (dict(need_a=False), dict(need_b=False), dict(bias=False),
                  dict(need_a=False, need_b=False), dict(need_b=False, bias=False)):
        got = ops.gated_matmul_grad(dy, *gpu[:3], z, u, **kinds)
        for g, w in zip(got, want):
            assert g is None or torch.equal(g, w)


@pytest.mark.parametrize("m", [4, 200])
def test_values_that_are_not_finite(m):
    """A row or a column with one has it for itself."""
    t, _ = _make(m, 100, 90, torch.bfloat16)
    want = ops.gated_matmul(*_cuda(t))
    bad = [x.clone() for x in t]
    bad[0][1, 7] = float("inf")
    bad[0][2, 99] = float("nan")
    bad[1][50, 3] = float("nan")
    got = ops.gated_matmul(*_cuda(bad))
    assert torch.isnan(got[2].float()).all()
    assert not torch.isfinite(got[:, 3].float()).any()
    rows = [r for r in range(m) if r not in (1, 2)]
    cols = [c for c in range(90) if c != 3]
    assert torch.equal(got[rows][:, cols], want[rows][:, cols])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [2, 150])
def test_streams_and_graphs(dtype, m):
    a, dy = _make(m, 520, 136, dtype)
    b, _ = _make(m, 520, 136, dtype, seed=9)
    both, dy = [_cuda(a), _cuda(b)], dy.cuda()

    def run(t):
        out, z, u = ops.gated_matmul(*t, keep_pre_activation=True)
        return [out, z, u] + list(ops.gated_matmul_grad(dy, *t[:3], z, u))

    want = [[x.clone() for x in run(t)] for t in both]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s, t in zip(streams, both):
        with torch.cuda.stream(s):
            got.append(run(t))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g, w))
    t = [x.clone() for x in both[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(t)
    for turn in (0, 1, 0, 1):
        for x, y in zip(t, both[turn]):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want[turn]))
        run(both[1 - turn])
