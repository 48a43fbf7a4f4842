"""The norms around a block with its gate and residual scale, and their
gradients, against 64 bits.  A row's sums are trees of at most 16 values per
lane and 10 levels; a statistic and what follows it stay below 128 operations."""
import itertools

import pytest
import torch

import sequence_reference as ref
from portdnn_amd import ops
from portdnn_amd.ops import GATE, NORM

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
OPERATIONS = 128


def _make(rows, channels, dtype, post, pre, gate_op, gate_rows, scale=True,
          residual=True, affine=True, seed=0):
    g = torch.Generator().manual_seed(seed + rows + channels)

    def normal(*shape, mean=0.0, std=1.0):
        return (torch.randn(shape, generator=g) * std + mean).to(dtype)

    t = {"x": normal(rows, channels, mean=0.5)}
    if residual:
        t["residual"] = normal(rows, channels, std=2.0)
    if gate_op != "NONE":
        t["gate"] = normal(-(-rows // gate_rows), channels)
    if scale:
        t["scale"] = normal(channels)
    if affine and post != "NONE":
        t["post_weight"], t["post_bias"] = normal(channels), normal(channels)
    if affine and pre != "NONE":
        t["pre_weight"], t["pre_bias"] = normal(channels), normal(channels)
    kinds = {"post": post, "pre": pre, "gate_rows": gate_rows, "eps": 1e-5}
    return g, t, kinds


def _gpu(t, kinds, gate_op):
    return ({k: v.cuda() for k, v in t.items()},
            {**kinds, "post": getattr(NORM, kinds["post"]),
             "pre": getattr(NORM, kinds["pre"]),
             "gate_op": getattr(GATE, gate_op)})


def _double(t):
    return {k: v.double() for k, v in t.items()}


def _check(rows, channels, dtype, post, pre, gate_op, gate_rows, **options):
    what = "%dx%d %s %s %s/%d" % (rows, channels, post, pre, gate_op, gate_rows)
    g, t, kinds = _make(rows, channels, dtype, post, pre, gate_op, gate_rows,
                        **options)
    gpu, gpu_kinds = _gpu(t, kinds, gate_op)
    y, u, stats = ops.residual_norm(**gpu, **gpu_kinds, keep_stats=True)
    want_y, want_u, want_stats = ref.residual_norm(**_double(t), **kinds,
                                                   gate_op=gate_op)
    ref.check(y, want_y, OPERATIONS, what + " sum")
    if pre == "NONE":
        assert u is None
    else:
        ref.check(u, want_u, OPERATIONS, what + " normed")
    # mean and deviation of x, whose values are exact
    x, m, r = t["x"].double(), want_stats[:, :1], want_stats[:, 1:2]
    size = x.abs() + x.abs().mean(1, keepdim=True)
    ref.check(stats[:, :1], (m, x.abs().mean(1, keepdim=True)), OPERATIONS,
              what + " mean")
    ref.check(stats[:, 1:2],
              (r, r * (1 + r * r * ((x - m).abs() * size).mean(1, keepdim=True))),
              OPERATIONS, what + " deviation")

    dy = torch.randn(rows, channels, generator=g).to(dtype)
    du = torch.randn(rows, channels, generator=g).to(dtype)
    if pre == "NONE":
        du = None
    given = {k: v for k, v in gpu.items() if k != "residual"}
    got = ops.residual_norm_grad(
        sum=y, stats=stats, grad_sum=dy.cuda(),
        grad_normed=None if du is None else du.cuda(), **given, **gpu_kinds)
    given = {k: v.double() for k, v in t.items() if k != "residual"}
    want = ref.residual_norm_grad(
        y=y.cpu().double(), stats=stats.cpu().double(), dy=dy.double(),
        du=None if du is None else du.double(), gate_op=gate_op, **given,
        **kinds)
    assert set(got) == set(given) | {"residual"}
    for name, v in got.items():
        over_rows = name not in ("x", "residual") and not (
            name == "gate" and gate_rows == 1)
        ref.check(v, want[name], OPERATIONS + (rows if over_rows else 0),
                  what + " " + name)


CHANNELS = [1, 7, 64, 200, 512, 513, 1000, 1024, 1600, 2048, 4096, 4100, 6000,
            8192, 9000, 16384]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", CHANNELS)
def test_row_lengths(dtype, channels):
    for rows, post, pre, gate_op, gate_rows in (
            (1, "RMS", "LAYER", "SILU", 1), (37, "LAYER", "RMS", "SIGMOID", 9),
            (5, "NONE", "RMS", "VALUE", 5)):
        if channels == 1 and "LAYER" in (post, pre):
            continue  # (one value less its mean is rounding and nothing else)
        _check(rows, channels, dtype, post, pre, gate_op, gate_rows)


@pytest.mark.parametrize("post,pre", itertools.product(
    ["NONE", "RMS", "LAYER"], repeat=2))
@pytest.mark.parametrize("gate_op,gate_rows", [
    ("NONE", 1), ("VALUE", 1), ("SIGMOID", 1), ("SILU", 1), ("VALUE", 4),
    ("SILU", 100), ("SIGMOID", 7)])
def test_kinds(post, pre, gate_op, gate_rows):
    for dtype in TYPES:
        for channels in (96, 1040):
            _check(53, channels, dtype, post, pre, gate_op, gate_rows)


@pytest.mark.parametrize("dtype", TYPES)
def test_absent_operands(dtype):
    for scale, residual, affine in itertools.product([0, 1], repeat=3):
        _check(11, 264, dtype, "RMS", "LAYER", "NONE", 1, scale=scale,
               residual=residual, affine=affine)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_and_gates(dtype):
    _check(3001, 40, dtype, "RMS", "RMS", "VALUE", 2)
    _check(2100, 520, dtype, "LAYER", "RMS", "SILU", 1000)
    _check(4111, 130, dtype, "RMS", "LAYER", "SIGMOID", 4111)
    _check(5000, 64, dtype, "NONE", "RMS", "SILU", 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_strides_and_alignments(dtype, shift):
    """x and the gate as slices of one projection's output."""
    for channels in (128, 131, 1024):
        g, t, kinds = _make(9, channels, dtype, "RMS", "RMS", "SILU", 1)
        both = torch.full((9, 2 * channels + 8), float("nan"), dtype=dtype,
                          device="cuda")
        gpu, gpu_kinds = _gpu(t, kinds, "SILU")
        want = ops.residual_norm(**gpu, **gpu_kinds, keep_stats=True)
        for i, name in enumerate(("x", "gate")):
            view = both[:, shift + i * channels:shift + (i + 1) * channels]
            view.copy_(gpu[name])
            gpu[name] = view
        got = ops.residual_norm(**gpu, **gpu_kinds, keep_stats=True)
        dy = torch.randn(9, channels, generator=g).to(dtype).cuda()
        del gpu["residual"]
        grads = ops.residual_norm_grad(sum=got[0], stats=got[2], grad_sum=dy,
                                       grad_normed=dy, **gpu, **gpu_kinds)
        ref_y, ref_u, _ = ref.residual_norm(**_double(t), **kinds,
                                            gate_op="SILU")
        ref.check(got[0], ref_y, OPERATIONS)
        ref.check(got[1], ref_u, OPERATIONS)
        del t["residual"]
        back = ref.residual_norm_grad(
            y=got[0].cpu().double(), stats=got[2].cpu().double(),
            dy=dy.cpu().double(), du=dy.cpu().double(), gate_op="SILU",
            **_double(t), **kinds)
        for name, v in grads.items():
            ref.check(v, back[name], OPERATIONS + 9, name)
        assert want[0].shape == got[0].shape


@pytest.mark.parametrize("dtype", TYPES)
def test_sum_in_place(dtype):
    for channels in (72, 640):
        _, t, kinds = _make(33, channels, dtype, "RMS", "RMS", "VALUE", 33)
        for name in ("x", "residual"):
            gpu, gpu_kinds = _gpu(t, kinds, "VALUE")
            want = ops.residual_norm(**gpu, **gpu_kinds)
            got = ops.residual_norm(**gpu, **gpu_kinds, out=gpu[name])
            assert got[0] is gpu[name]
            assert torch.equal(got[0], want[0])
            assert torch.equal(got[1], want[1])


def test_only_normed_only_one_gradient():
    _, t, kinds = _make(21, 256, torch.float16, "NONE", "RMS", "NONE", 1,
                        scale=False, residual=False)
    gpu, gpu_kinds = _gpu(t, kinds, "NONE")
    want = ops.residual_norm(**gpu, **gpu_kinds)
    none, u, _ = ops.residual_norm(**gpu, **gpu_kinds, keep_sum=False)
    assert none is None and torch.equal(u, want[1])
    _, t, kinds = _make(21, 256, torch.float16, "RMS", "RMS", "SILU", 1)
    gpu, gpu_kinds = _gpu(t, kinds, "SILU")
    y, u, stats = ops.residual_norm(**gpu, **gpu_kinds, keep_stats=True)
    given = {k: v for k, v in gpu.items() if k != "residual"}
    zero = torch.zeros_like(y)
    d = torch.randn_like(y)
    for a, b in (((d, None), (d, zero)), ((None, d), (zero, d))):
        one = ops.residual_norm_grad(sum=y, stats=stats, grad_sum=a[0],
                                     grad_normed=a[1], **given, **gpu_kinds)
        two = ops.residual_norm_grad(sum=y, stats=stats, grad_sum=b[0],
                                     grad_normed=b[1], **given, **gpu_kinds)
        assert all(torch.equal(v, two[name]) for name, v in one.items())


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_infinities_and_nans_stay_to_themselves(dtype):
    for channels in (80, 1032):
        _, t, kinds = _make(12, channels, dtype, "RMS", "LAYER", "SIGMOID", 1)
        gpu, gpu_kinds = _gpu(t, kinds, "SIGMOID")
        clean = ops.residual_norm(**gpu, **gpu_kinds)
        gpu["x"][3, 5], gpu["x"][7, channels - 1] = float("nan"), float("inf")
        gpu["x"][9] = 0
        got = ops.residual_norm(**gpu, **gpu_kinds)
        keep = [i for i in range(12) if i not in (3, 7, 9)]
        for a, b in zip(clean[:2], got[:2]):
            assert torch.equal(a[keep], b[keep])
            assert b[3].isnan().all() and b[9].isfinite().all()
        # a normalised infinity is none: all else in its row becomes its zero
        assert got[0][7, channels - 1].isnan()


def test_large_values_and_offsets():
    """A row of one value and noise: the squares come from what is left when
    the mean is out."""
    x = 1000.0 + torch.randn(4, 512, generator=torch.Generator().manual_seed(3))
    want = ref.residual_norm(x.double(), pre="LAYER")
    u = ops.residual_norm(x.cuda(), pre=NORM.LAYER)[1]
    ref.check(u, want[1], OPERATIONS)


def test_tensors_beyond_two_gigabytes():
    rows, channels = (1 << 20) + 11, 2056
    x = torch.zeros((rows, channels), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(3)
    tail = torch.randn(50, channels, generator=g).bfloat16()
    x[-50:] = tail.cuda()
    y, u, stats = ops.residual_norm(x, residual=x, post=NORM.RMS, pre=NORM.RMS,
                                    eps=1e-5, keep_stats=True)
    want_y, want_u, _ = ref.residual_norm(tail.double(), tail.double(),
                                          post="RMS", pre="RMS", eps=1e-5)
    ref.check(y[-50:], want_y, OPERATIONS)
    ref.check(u[-50:], want_u, OPERATIONS)
    assert not u[:100].any()
    got = ops.residual_norm_grad(x, y, stats, grad_sum=y, post=NORM.RMS,
                                 pre=NORM.RMS, eps=1e-5)
    want = ref.residual_norm_grad(
        tail.double(), y[-50:].cpu().double(), stats[-50:].cpu().double(),
        dy=y[-50:].cpu().double(), post="RMS", pre="RMS", eps=1e-5)
    ref.check(got["x"][-50:], want["x"], OPERATIONS)


def test_another_stream_a_graph_and_the_same_bits_again():
    _, t, kinds = _make(777, 520, torch.bfloat16, "RMS", "LAYER", "SILU", 100)
    gpu, gpu_kinds = _gpu(t, kinds, "SILU")
    given = {k: v for k, v in gpu.items() if k != "residual"}
    d = torch.randn(777, 520, device="cuda").bfloat16()

    def run():
        y, u, stats = ops.residual_norm(**gpu, **gpu_kinds, keep_stats=True)
        return [y, u, stats, *ops.residual_norm_grad(
            sum=y, stats=stats, grad_sum=d, grad_normed=u, **given,
            **gpu_kinds).values()]

    eager = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = run()
    stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(3):
        for v in captured:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = run()
        assert all(torch.equal(x, y) for x, y in zip(captured, again))
