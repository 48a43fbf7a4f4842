"""Calls of more work-groups than one dimension of a grid holds work-items for: rows,
sequences and columns by the hundred million, of a few values each.  The first ones,
the last ones and those around the 2^20-th work-group are compared with 64 bits, the
others are zero and stay so."""
import pytest
import torch

import sequence_reference as ref
from portdnn_amd import ops
from portdnn_amd.ops import NORM

pytestmark = pytest.mark.gpu

F16 = torch.float16


def _places(n, around):
    return [slice(0, 40), slice(around - 20, around + 20), slice(n - 40, n)]


def _filled(shape, places, seed, dim=0):
    """Zeros but for random values at the places, and those on the CPU."""
    g = torch.Generator().manual_seed(seed)
    t = torch.zeros(shape, dtype=F16, device="cuda")
    parts = []
    for p in places:
        size = list(shape)
        size[dim] = p.stop - p.start
        part = torch.randn(size, generator=g).to(F16)
        t.narrow(dim, p.start, p.stop - p.start).copy_(part)
        parts.append(part)
    return t, parts


def _only_there(t, places, dim=0):
    """Whether t is zero everywhere else."""
    begin = 0
    for p in places + [slice(t.shape[dim], None)]:
        if t.narrow(dim, begin, p.start - begin).any():
            return False
        begin = p.stop
    return True


def test_norms_of_many_short_rows():
    rows, channels = (1 << 26) + 45, 8
    places = _places(rows, 4 << 20)
    x, parts = _filled((rows, channels), places, 0)
    kinds = {"post": "LAYER", "pre": "RMS", "eps": 1e-5}
    own = {"post": NORM.LAYER, "pre": NORM.RMS, "eps": 1e-5}
    y, u, stats = ops.residual_norm(x, residual=x, keep_stats=True, **own)
    dy, grads = _filled((rows, channels), places, 1)
    got = ops.residual_norm_grad(x, y, stats, grad_sum=dy, grad_normed=dy, **own)
    for p, part, d in zip(places, parts, grads):
        v = part.double()
        want_y, want_u, _ = ref.residual_norm(v, residual=v, **kinds)
        ref.check(y[p], want_y, 128)
        ref.check(u[p], want_u, 128)
        want = ref.residual_norm_grad(
            v, y[p].cpu().double(), stats[p].cpu().double(), d.double(),
            d.double(), **kinds)
        ref.check(got["x"][p], want["x"], 128)
        ref.check(got["residual"][p], want["residual"], 128)
    for t in (y, u, got["x"], got["residual"]):
        assert _only_there(t, places)


def test_many_short_sequences():
    batch, channels = (1 << 26) + 43, 4
    places = _places(batch, 4 << 20)
    x, xs = _filled((batch, 1, channels), places, 2)
    f, fs = _filled((batch, 1, channels), places, 3)
    h, last = ops.linear_recurrence(x, f)
    dh, ds = _filled((batch, 1, channels), places, 4)
    got = ops.linear_recurrence_grad(dh, x, f, h)
    for p, a, b, d in zip(places, xs, fs, ds):
        want_h, want_last = ref.recurrence(a.double(), b.double())
        ref.check(h[p], want_h, 64)
        ref.check(last[p], want_last, 64)
        want = ref.recurrence_grad(d.double(), a.double(), b.double(),
                                   h[p].cpu().double())
        for name, v in got.items():
            ref.check(v[p], want[name], 64, name)
    for t in (h, last, *got.values()):
        assert _only_there(t, places)


def test_products_of_many_columns():
    m, k, n = 3, 3, (1 << 28) + 41
    places = _places(n, 16 << 20)
    b, parts = _filled((k, n), places, 5, dim=1)
    a = torch.randn(m, k, generator=torch.Generator().manual_seed(6)).to(F16)
    y = ops.matmul_bias_act(a.cuda(), b)
    for p, part in zip(places, parts):
        want, _ = ref.matmul(a.double(), part.double())
        ref.check(y[:, p], want, k + 64)
    assert _only_there(y, places, dim=1)


def test_sums_of_many_columns():
    m, n = 2, (1 << 28) + 40
    places = _places(n, 64 << 20)
    dy, parts = _filled((m, n), places, 7, dim=1)
    a, b = torch.zeros(m, 1, dtype=F16).cuda(), torch.zeros(1, n, dtype=F16).cuda()
    _, _, bias = ops.matmul_bias_act_grad(dy, a, b, need_a=False, need_b=False)
    for p, part in zip(places, parts):
        v = part.double()
        ref.check(bias[p], (v.sum(0), v.abs().sum(0)), 64)
    assert _only_there(bias, places)


def test_sums_over_many_rows():
    """More rows than 2^30, of one channel: x + scale y and its gradients."""
    rows = (1 << 30) + 75
    places = _places(rows, 1 << 29)
    x, xs = _filled((rows, 1), places, 8)
    dy, ds = _filled((rows, 1), places, 9)
    scale = torch.tensor([0.75], dtype=F16, device="cuda")
    y, _, _ = ops.residual_norm(x, residual=x, scale=scale)
    got = ops.residual_norm_grad(x, y, None, grad_sum=dy, scale=scale)
    for p, part, d in zip(places, xs, ds):
        v, w = part.double(), d.double()
        ref.check(y[p], (1.75 * v, 1.75 * v.abs()), 8)
        ref.check(got["x"][p], (0.75 * w, 0.75 * w.abs()), 8)
        assert torch.equal(got["residual"][p].cpu(), d)
    assert _only_there(y, places) and _only_there(got["x"], places)
    each = torch.cat([v.double() * w.double() for v, w in zip(xs, ds)])
    # (120 terms that are not zero, added along 2^18 rows a wave and joined)
    ref.check(got["scale"], (each.sum(0), each.abs().sum(0)), 256)
