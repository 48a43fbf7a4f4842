"""What the operators of a residual block over sequences refuse, and their
workspace queries: decided on the host before anything is launched."""
import ctypes

import pytest
import torch

from portdnn_amd import capi, ops
from portdnn_amd.capi import (ACTIVATION, DTYPE, GATE, NORM, STATUS,
                              LinearRecurrenceParams, MatmulBiasActParams,
                              ResidualNormGradients, ResidualNormParams,
                              ResidualNormTensors)

FAKE = 0x1000  # never dereferenced: every call returns early
TYPES = ["f32", "f16", "bf16"]


def _matmul(suffix, p, lhs=FAKE, rhs=FAKE, out=FAKE, workspace=None, elems=0):
    return getattr(capi.lib(), "snn_hip_matmul_bias_act_" + suffix)(
        lhs, rhs, None, None, out, None, p and ctypes.byref(p), workspace,
        elems, None)


def _matmul_grad(suffix, p, dy=FAKE, lhs=FAKE, rhs=FAKE, z=FAKE, dl=FAKE,
                 dr=FAKE, db=FAKE, workspace=None, elems=0):
    return getattr(capi.lib(), "snn_hip_matmul_bias_act_grad_" + suffix)(
        dy, lhs, rhs, z, dl, dr, db, p and ctypes.byref(p), workspace, elems,
        None)


def _matmul_params(**kw):
    return MatmulBiasActParams(**{**dict(m=8, k=16, n=24), **kw})


BAD_MATMUL = [dict(m=0), dict(k=0), dict(n=-1), dict(activation=5),
              dict(activation=-1), dict(lhs_stride=15), dict(rhs_stride=23),
              dict(residual_stride=23), dict(output_stride=23),
              dict(lhs_stride=-16), dict(transpose_lhs=1, lhs_stride=7),
              dict(transpose_rhs=1, rhs_stride=15)]


@pytest.mark.parametrize("suffix", TYPES)
def test_matmul_refusals(suffix):
    for kw in BAD_MATMUL:
        p = _matmul_params(**kw)
        assert _matmul(suffix, p) == STATUS.INVALID_PARAMETER, kw
        assert _matmul_grad(suffix, p) == STATUS.INVALID_PARAMETER, kw
    p = _matmul_params()
    assert _matmul(suffix, None) == STATUS.INVALID_PARAMETER
    for name in ("lhs", "rhs", "out"):
        assert _matmul(suffix, p, **{name: None}) == STATUS.INVALID_PARAMETER
    assert _matmul(suffix, p, workspace=FAKE + 8) == STATUS.INVALID_PARAMETER
    assert (_matmul(suffix, _matmul_params(n=1 << 30)) ==
            STATUS.INDEX_EXCEEDED)


@pytest.mark.parametrize("suffix", TYPES)
def test_matmul_gradient_refusals(suffix):
    p = _matmul_params(activation=ACTIVATION.GELU)
    assert _matmul_grad(suffix, None) == STATUS.INVALID_PARAMETER
    for kw in (dict(dy=None), dict(z=None), dict(lhs=None), dict(rhs=None),
               dict(dl=None, dr=None, db=None), dict(workspace=FAKE + 4)):
        assert _matmul_grad(suffix, p, **kw) == STATUS.INVALID_PARAMETER, kw
    required, recommended = _sizes(
        "snn_hip_matmul_bias_act_workspace_size", p, 1,
        getattr(DTYPE, suffix.upper()))
    assert 0 < required <= recommended
    for elems in (0, required - 1):
        assert (_matmul_grad(suffix, p, workspace=FAKE, elems=elems) ==
                STATUS.INSUFFICIENT_WORKSPACE)
    assert _matmul_grad(suffix, p) == STATUS.INSUFFICIENT_WORKSPACE


def _sizes(name, p, *args):
    req, rec = ctypes.c_size_t(), ctypes.c_size_t()
    capi.check(getattr(capi.lib(), name)(ctypes.byref(p), *args,
                                         ctypes.byref(req), ctypes.byref(rec)))
    return req.value, rec.value


def _norm_params(**kw):
    return ResidualNormParams(**{**dict(
        rows=4, channels=8, post_norm=NORM.RMS, pre_norm=NORM.LAYER,
        gate=GATE.SILU, gate_rows=1, epsilon=1e-6), **kw})


def _norm(suffix, p, **kw):
    t = ResidualNormTensors(**{**dict(x=FAKE, gate=FAKE, sum=FAKE), **kw})
    return getattr(capi.lib(), "snn_hip_residual_norm_" + suffix)(
        ctypes.byref(t), p and ctypes.byref(p), None)


def _norm_grad(suffix, p, tensors=(), workspace=None, elems=0, **kw):
    t = ResidualNormTensors(**{**dict(x=FAKE, gate=FAKE, sum=FAKE, stats=FAKE),
                               **dict(tensors)})
    g = ResidualNormGradients(**{**dict(grad_sum=FAKE, grad_x=FAKE), **kw})
    return getattr(capi.lib(), "snn_hip_residual_norm_grad_" + suffix)(
        ctypes.byref(t), ctypes.byref(g), p and ctypes.byref(p), workspace,
        elems, None)


BAD_NORM = [dict(rows=0), dict(channels=0), dict(channels=16385),
            dict(post_norm=3), dict(post_norm=-1), dict(pre_norm=3),
            dict(gate=4), dict(gate=-1), dict(gate_rows=0), dict(x_stride=7),
            dict(gate_stride=7), dict(epsilon=-1.0),
            dict(epsilon=float("nan"))]


@pytest.mark.parametrize("suffix", TYPES)
def test_norm_refusals(suffix):
    bad = STATUS.INVALID_PARAMETER
    for kw in BAD_NORM:
        assert _norm(suffix, _norm_params(**kw)) == bad, kw
        assert _norm_grad(suffix, _norm_params(**kw)) == bad, kw
    p = _norm_params()
    entry = getattr(capi.lib(), "snn_hip_residual_norm_" + suffix)
    assert entry(None, ctypes.byref(p), None) == bad
    assert _norm(suffix, None) == bad
    assert _norm(suffix, p, x=None) == bad
    assert _norm(suffix, p, gate=None) == bad
    assert _norm(suffix, p, sum=None) == bad
    assert _norm(suffix, _norm_params(gate=GATE.NONE)) == bad
    assert _norm(suffix, _norm_params(pre_norm=NORM.NONE), normed=FAKE) == bad
    for name in ("post_weight", "post_bias"):
        assert _norm(suffix, _norm_params(post_norm=NORM.NONE),
                     **{name: FAKE}) == bad
    for name in ("pre_weight", "pre_bias"):
        assert _norm(suffix, _norm_params(pre_norm=NORM.NONE),
                     **{name: FAKE}) == bad


@pytest.mark.parametrize("suffix", TYPES)
def test_norm_gradient_refusals(suffix):
    bad = STATUS.INVALID_PARAMETER
    p = _norm_params()
    assert _norm_grad(suffix, p, grad_sum=None) == bad
    assert _norm_grad(suffix, p, {"stats": None}) == bad
    assert _norm_grad(suffix, p, {"sum": None}, grad_normed=FAKE) == bad
    assert _norm_grad(suffix, _norm_params(pre_norm=NORM.NONE),
                      grad_normed=FAKE) == bad
    for name in ("scale", "post_weight", "post_bias", "pre_weight", "pre_bias"):
        assert _norm_grad(suffix, p, **{"grad_" + name: FAKE}) == bad, name
    assert _norm_grad(suffix, _norm_params(gate=GATE.NONE), {"gate": None},
                      grad_gate=FAKE) == bad
    assert _norm_grad(suffix, p, {"scale": FAKE}, grad_scale=FAKE,
                      workspace=FAKE + 8, elems=1 << 20) == bad
    required, recommended = _sizes(
        "snn_hip_residual_norm_grad_workspace_size", p,
        getattr(DTYPE, suffix.upper()))
    assert 0 < required <= recommended
    for workspace, elems in ((None, required), (FAKE, 0)):
        assert _norm_grad(suffix, p, {"scale": FAKE}, grad_scale=FAKE,
                          workspace=workspace, elems=elems) == \
            STATUS.INSUFFICIENT_WORKSPACE


def _recurrence(suffix, p, x=FAKE, f=FAKE, h=FAKE, workspace=None):
    return getattr(capi.lib(), "snn_hip_linear_recurrence_" + suffix)(
        x, f, None, None, None, None, h, None, p and ctypes.byref(p), workspace,
        0, None)


def _recurrence_grad(suffix, p, dh=FAKE, x=FAKE, f=FAKE, i=None, h=FAKE,
                     dx=FAKE, df=FAKE, di=None):
    return getattr(capi.lib(), "snn_hip_linear_recurrence_grad_" + suffix)(
        dh, None, x, f, i, None, None, None, h, dx, df, di, None,
        p and ctypes.byref(p), None, 0, None)


@pytest.mark.parametrize("suffix", TYPES)
def test_recurrence_refusals(suffix):
    bad = STATUS.INVALID_PARAMETER
    for kw in (dict(batch=0), dict(steps=0), dict(channels=0),
               dict(row_stride=7), dict(grad_row_stride=7),
               dict(row_stride=-8)):
        p = LinearRecurrenceParams(**{**dict(batch=2, steps=3, channels=8),
                                      **kw})
        assert _recurrence(suffix, p) == bad, kw
        assert _recurrence_grad(suffix, p) == bad, kw
    p = LinearRecurrenceParams(batch=2, steps=3, channels=8)
    assert _recurrence(suffix, None) == bad
    assert _recurrence_grad(suffix, None) == bad
    for name in ("x", "f", "h"):
        assert _recurrence(suffix, p, **{name: None}) == bad
    for name in ("dh", "x", "f", "h", "dx", "df"):
        assert _recurrence_grad(suffix, p, **{name: None}) == bad
    assert _recurrence_grad(suffix, p, i=FAKE) == bad
    assert _recurrence_grad(suffix, p, di=FAKE) == bad
    assert _recurrence(suffix, p, workspace=FAKE + 4) == bad
    many = LinearRecurrenceParams(batch=(1 << 31) - 1, steps=1, channels=65)
    assert _recurrence(suffix, many) == STATUS.INDEX_EXCEEDED


def test_workspace_queries():
    for name, p, args in (
            ("snn_hip_matmul_bias_act_workspace_size", _matmul_params(), (0,)),
            ("snn_hip_residual_norm_grad_workspace_size", _norm_params(), ()),
            ("snn_hip_linear_recurrence_workspace_size",
             LinearRecurrenceParams(batch=1, steps=5000, channels=64), ())):
        entry = getattr(capi.lib(), name)
        n = ctypes.c_size_t()
        for dtype in (-1, 3):
            assert entry(ctypes.byref(p), *args, dtype, ctypes.byref(n),
                         ctypes.byref(n)) == STATUS.INVALID_PARAMETER
        assert entry(None, *args, 0, ctypes.byref(n),
                     ctypes.byref(n)) == STATUS.INVALID_PARAMETER
        assert entry(ctypes.byref(p), *args, 0, None,
                     ctypes.byref(n)) == STATUS.INVALID_PARAMETER
        # the same floats, in elements of the type
        f32, f16 = _sizes(name, p, *args, 0)[1], _sizes(name, p, *args, 1)[1]
        assert _sizes(name, p, *args, 2)[1] == f16
        if "matmul" not in name:
            assert f32 > 0
    # products with few tiles and a long reduction share it
    for grad in (0, 1):
        assert _sizes("snn_hip_matmul_bias_act_workspace_size",
                      _matmul_params(k=8192), grad, 1)[1] > 0
    # one step is one piece
    assert _sizes("snn_hip_linear_recurrence_workspace_size",
                  LinearRecurrenceParams(batch=1, steps=1, channels=64), 0) == \
        (0, 0)


def test_the_fused_convolution_keeps_its_activations():
    p = ops.conv_params(1, 4, 4, 4, 4, 1, 1, True)
    entry = capi.lib().snn_hip_conv2d_forward_bias_act_f32
    for act in (ACTIVATION.GELU, ACTIVATION.GELU_TANH, ACTIVATION.SILU):
        assert entry(FAKE, FAKE, None, FAKE, ctypes.byref(p), 1, act, None, 0,
                     None) == STATUS.INVALID_PARAMETER
    assert capi.lib().snn_hip_conv2d_default_algorithm_for(
        ctypes.byref(p), 0, DTYPE.BF16) == 0


def test_python_calls_check_shapes_and_types(monkeypatch):
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    a, b = torch.zeros(4, 8), torch.zeros(8, 6)
    for call in (
            lambda: ops.matmul_bias_act(a, b.t()),
            lambda: ops.matmul_bias_act(a, b.half()),
            lambda: ops.matmul_bias_act(a, b, bias=torch.zeros(5)),
            lambda: ops.matmul_bias_act(a, b, bias=torch.zeros(6).half()),
            lambda: ops.matmul_bias_act(a, b, residual=torch.zeros(6, 4)),
            lambda: ops.matmul_bias_act(a, b, out=torch.zeros(4, 7)),
            lambda: ops.matmul_bias_act(a.expand(4, 8).t(), b, trans_a=True),
            lambda: ops.matmul_bias_act(a[:1].expand(4, 8), b),
            lambda: ops.matmul_bias_act_grad(a, a, b),
            lambda: ops.matmul_bias_act_grad(
                torch.zeros(4, 6), a, b, torch.zeros(4, 5), activation=1),
            lambda: ops.residual_norm(a, residual=b, pre=NORM.RMS),
            lambda: ops.residual_norm(a, gate_op=GATE.SILU, pre=NORM.RMS),
            lambda: ops.residual_norm(a, gate=a, gate_rows=2, pre=NORM.RMS),
            lambda: ops.residual_norm(a, scale=torch.zeros(4), pre=NORM.RMS),
            lambda: ops.residual_norm(a.t(), pre=NORM.RMS),
            lambda: ops.residual_norm_grad(a, a, torch.zeros(4, 3), grad_sum=a),
            lambda: ops.linear_recurrence(a[None], a[None, :, :4]),
            lambda: ops.linear_recurrence(a[None], a[None].half()),
            lambda: ops.linear_recurrence(
                a[None], a[None], resets=torch.zeros(1, 4)),
            lambda: ops.linear_recurrence(
                a[None], a[None], lengths=torch.zeros(1, dtype=torch.int64)),
            lambda: ops.linear_recurrence(
                a[None], a[None], initial_state=torch.zeros(1, 8).half()),
            lambda: ops.linear_recurrence(
                torch.zeros(2, 3, 8).transpose(0, 1), torch.zeros(3, 2, 8)),
    ):
        with pytest.raises(AssertionError):
            call()
