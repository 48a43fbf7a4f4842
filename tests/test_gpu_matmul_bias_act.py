"""Matrix products with bias, activation and residual, and their gradients,
against 64 bits.  A product of k terms is a chain of k + a few fp32 operations."""
import pytest
import torch

import sequence_reference as ref
from portdnn_amd import capi, ops
from portdnn_amd.ops import ACTIVATION

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
EXTRA = 64  # operations of the epilogue and of joining shares


def _normal(g, *shape, std=1.0, dtype):
    return (torch.randn(shape, generator=g) * std).to(dtype)


def _wide(t, pad, shift=0):
    """t on the GPU as rows of a wider matrix, `shift` elements into it."""
    rows, cols = t.shape
    wide = torch.full((rows, cols + pad + shift), float("nan"), dtype=t.dtype,
                      device="cuda")
    view = wide[:, shift:shift + cols]
    view.copy_(t)
    return view


def _operands(m, k, n, dtype, trans_a, trans_b, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = _normal(g, *((k, m) if trans_a else (m, k)), dtype=dtype)
    b = _normal(g, *((n, k) if trans_b else (k, n)), std=k ** -0.5,
                dtype=dtype)
    return g, a, b


def _double(t, trans=False):
    t = t.double()
    return t.t() if trans else t


SHAPES = [(1, 1, 1), (1, 64, 128), (1, 777, 300), (1, 2048, 512), (3, 5, 7),
          (16, 128, 256), (17, 64, 129), (24, 1024, 264), (64, 72, 136),
          (65, 200, 64), (100, 1000, 24), (128, 128, 128), (130, 70, 257),
          (257, 129, 300), (300, 136, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans_a,trans_b", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_products(dtype, trans_a, trans_b):
    for m, k, n in SHAPES:
        g, a, b = _operands(m, k, n, dtype, trans_a, trans_b, m + k)
        bias, add = _normal(g, n, dtype=dtype), _normal(g, m, n, dtype=dtype)
        kind = ref.ACTIVATIONS[(m + n) % 5]
        y, z = ops.matmul_bias_act(
            a.cuda(), b.cuda(), bias=bias.cuda(), residual=add.cuda(),
            activation=getattr(ACTIVATION, kind), trans_a=trans_a,
            trans_b=trans_b, keep_pre_activation=True)
        want_y, want_z = ref.matmul(
            _double(a, trans_a), _double(b, trans_b), bias.double(),
            add.double(), kind)
        what = "%dx%dx%d %s" % (m, k, n, kind)
        ref.check(z, want_z, k + EXTRA, what + " z")
        ref.check(y, want_y, k + EXTRA, what)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("trans_a,trans_b", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_products_of_many_large_tiles(dtype, trans_a, trans_b):
    m, k, n = 4088, 168, 3080
    g, a, b = _operands(m, k, n, dtype, trans_a, trans_b)
    bias = _normal(g, n, dtype=dtype)
    y = ops.matmul_bias_act(a.cuda(), b.cuda(), bias=bias.cuda(),
                            activation=ACTIVATION.SILU, trans_a=trans_a,
                            trans_b=trans_b)
    want, _ = ref.matmul(_double(a, trans_a), _double(b, trans_b),
                         bias.double(), kind="SILU")
    ref.check(y, want, k + EXTRA)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ref.ACTIVATIONS)
@pytest.mark.parametrize("with_bias,with_residual,keep",
                         [(0, 0, 0), (1, 0, 1), (0, 1, 0)])
def test_epilogues(dtype, kind, with_bias, with_residual, keep):
    for m, k, n in ((5, 96, 40), (90, 64, 72), (150, 33, 51)):
        g, a, b = _operands(m, k, n, dtype, 0, 0, 7)
        bias = _normal(g, n, dtype=dtype) if with_bias else None
        add = _normal(g, m, n, dtype=dtype) if with_residual else None
        got = ops.matmul_bias_act(
            a.cuda(), b.cuda(), bias=bias.cuda() if with_bias else None,
            residual=add.cuda() if with_residual else None,
            activation=getattr(ACTIVATION, kind), keep_pre_activation=keep)
        y, z = got if keep else (got, None)
        want_y, want_z = ref.matmul(
            a.double(), b.double(), bias.double() if with_bias else None,
            add.double() if with_residual else None, kind)
        ref.check(y, want_y, k + EXTRA)
        if keep:
            ref.check(z, want_z, k + EXTRA)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans_a,trans_b", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (8, 1), (16, 8)])
def test_strides_and_alignments(dtype, trans_a, trans_b, pad, shift):
    """Rows of wider matrices, whose other values are NaN and stay as they are."""
    for m, k, n in ((1, 136, 136), (40, 72, 144), (144, 136, 200)):
        g, a, b = _operands(m, k, n, dtype, trans_a, trans_b, 3)
        add = _normal(g, m, n, dtype=dtype)
        out = _wide(torch.zeros(m, n, dtype=dtype), pad, shift)
        y = ops.matmul_bias_act(
            _wide(a, pad, shift), _wide(b, pad, shift),
            residual=_wide(add, pad, shift), trans_a=trans_a, trans_b=trans_b,
            out=out)
        assert y.data_ptr() == out.data_ptr()
        want, _ = ref.matmul(_double(a, trans_a), _double(b, trans_b),
                             residual=add.double())
        ref.check(y, want, k + EXTRA)
        if m > 1:
            whole = out.as_strided((m, out.stride(0)), (out.stride(0), 1),
                                   out.storage_offset() - shift)
            assert whole[:, :shift].isnan().all()
            assert whole[:, shift + n:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_residual_in_place(dtype):
    for m, k, n in ((3, 512, 64), (200, 64, 72)):
        g, a, b = _operands(m, k, n, dtype, 0, 0)
        add = _normal(g, m, n, dtype=dtype)
        x = add.cuda()
        y = ops.matmul_bias_act(a.cuda(), b.cuda(), residual=x, out=x)
        assert y is x
        ref.check(x, ref.matmul(a.double(), b.double(),
                                residual=add.double())[0], k + EXTRA)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_reductions_repeat_and_do_without_workspace(dtype):
    for m, k, n in ((1, 4096, 256), (30, 4096, 136), (100, 3000, 128)):
        g, a, b = _operands(m, k, n, dtype, 0, 1)
        want, _ = ref.matmul(a.double(), b.double().t())
        a, b = a.cuda(), b.cuda()
        first = ops.matmul_bias_act(a, b, trans_b=True)
        for _ in range(3):
            again = ops.matmul_bias_act(a, b, trans_b=True)
            assert torch.equal(first, again)
        ref.check(first, want, k + EXTRA)
        none = torch.empty(0, dtype=dtype, device="cuda")
        ref.check(ops.matmul_bias_act(a, b, trans_b=True, workspace=none),
                  want, k + EXTRA)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans_a,trans_b", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_gradients(dtype, trans_a, trans_b):
    for m, k, n, kind in ((1, 64, 128, "SILU"), (7, 33, 5, "GELU"),
                          (50, 200, 72, "NONE"), (129, 65, 130, "GELU_TANH"),
                          (300, 136, 264, "RELU"), (520, 256, 128, "GELU")):
        g, a, b = _operands(m, k, n, dtype, trans_a, trans_b, m)
        dy, z = _normal(g, m, n, dtype=dtype), _normal(g, m, n, dtype=dtype)
        got = ops.matmul_bias_act_grad(
            dy.cuda(), a.cuda(), b.cuda(), z.cuda(),
            activation=getattr(ACTIVATION, kind), trans_a=trans_a,
            trans_b=trans_b)
        da, db, dc = ref.matmul_grad(
            dy.double(), _double(a, trans_a), _double(b, trans_b), z.double(),
            kind, dtype)
        what = "%dx%dx%d %s" % (m, k, n, kind)
        for name, t, (value, mag, extra), length, trans in (
                ("a", got[0], da, n, trans_a), ("b", got[1], db, m, trans_b)):
            mag = extra + (length + EXTRA) * mag
            if trans:
                value, mag = value.t(), mag.t()
            ref.check(t, (value, mag), 1, what + " " + name)
        ref.check(got[2], dc, m + EXTRA, what + " bias")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_of_large_tiles_and_strided_operands(dtype):
    m, k, n = 3400, 3080, 136
    g, a, b = _operands(m, k, n, dtype, 0, 0)
    dy, z = _normal(g, m, n, dtype=dtype), _normal(g, m, n, dtype=dtype)
    got = ops.matmul_bias_act_grad(
        _wide(dy, 8), _wide(a, 16, 8), _wide(b, 8), z.cuda(),
        activation=ACTIVATION.SILU)
    da, db, dc = ref.matmul_grad(dy.double(), a.double(), b.double(),
                                 z.double(), "SILU", dtype)
    for t, (value, mag, extra), length in ((got[0], da, n), (got[1], db, m)):
        ref.check(t, (value, extra + (length + EXTRA) * mag), 1)
    ref.check(got[2], dc, m + EXTRA)


def test_gradients_one_at_a_time():
    dtype = torch.float16
    g, a, b = _operands(40, 72, 56, dtype, 0, 0)
    dy, z = _normal(g, 40, 56, dtype=dtype), _normal(g, 40, 56, dtype=dtype)
    t = [v.cuda() for v in (dy, a, b, z)]
    for act in (ACTIVATION.NONE, ACTIVATION.GELU):
        whole = ops.matmul_bias_act_grad(*t, activation=act)
        for i, want in enumerate(whole):
            got = ops.matmul_bias_act_grad(
                *t, activation=act, need_a=i == 0, need_b=i == 1, bias=i == 2)
            assert torch.equal(got[i], want)
            assert all(v is None for j, v in enumerate(got) if j != i)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nans_stay_in_their_rows_and_columns(dtype):
    for m, k, n in ((4, 256, 72), (70, 40, 136), (140, 96, 130)):
        g, a, b = _operands(m, k, n, dtype, 0, 0)
        clean = ops.matmul_bias_act(a.cuda(), b.cuda())
        a[1, 3], a[2, k - 1] = float("nan"), float("inf")
        b[5, n - 1] = float("nan")
        y = ops.matmul_bias_act(a.cuda(), b.cuda(),
                                activation=ACTIVATION.RELU)
        assert y[1].isnan().all() and y[:, n - 1].isnan().all()
        # an infinity by the sign of its factors
        row = y[2, :n - 1].float().cpu()
        assert torch.equal(row.isinf(), b[k - 1, :n - 1] > 0)
        keep = [i for i in range(m) if i not in (1, 2)]
        assert torch.equal(y[keep][:, :n - 1],
                           torch.clamp(clean[keep][:, :n - 1], min=0))


def test_operands_beyond_two_gigabytes():
    """Rows behind 2^31 elements of the left operand and the output."""
    dtype = torch.bfloat16
    m, k, n = (1 << 21) + 77, 1032, 16
    a = torch.zeros((m, k), dtype=dtype, device="cuda")
    g = torch.Generator().manual_seed(5)
    tail = _normal(g, 300, k, dtype=dtype)
    b = _normal(g, k, n, dtype=dtype)
    a[-300:] = tail.cuda()
    y = ops.matmul_bias_act(a, b.cuda())
    ref.check(y[-300:], ref.matmul(tail.double(), b.double())[0], k + EXTRA)
    assert not y[:1000].any() and not y[-10000:-300].any()


def test_another_stream_and_a_graph():
    dtype = torch.float16
    cases = []
    for m, k, n in ((1, 2048, 256), (40, 264, 128), (200, 71, 90)):
        g, a, b = _operands(m, k, n, dtype, 0, 0)
        dy = _normal(g, m, n, dtype=dtype)
        cases.append([v.cuda() for v in (a, b, dy)])

    def run():
        out = []
        for a, b, dy in cases:
            y, z = ops.matmul_bias_act(a, b, activation=ACTIVATION.SILU,
                                       keep_pre_activation=True)
            out += [y, z, *ops.matmul_bias_act_grad(
                dy, a, b, z, activation=ACTIVATION.SILU)]
        return out

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
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = run()
        assert all(torch.equal(x, y) for x, y in zip(captured, again))


def test_workspace_that_is_too_small():
    dtype = torch.float16
    t = [torch.zeros(64, 64, dtype=dtype, device="cuda") for _ in range(4)]
    with pytest.raises(capi.SnnHipError, match="InsufficientWorkspace"):
        ops.matmul_bias_act_grad(
            *t, activation=ACTIVATION.GELU,
            workspace=torch.empty(8, dtype=dtype, device="cuda"))
