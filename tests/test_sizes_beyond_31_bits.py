"""Sizes that the entry points' 31-bit counts do not hold: refused, not cut off."""
import ctypes

import pytest
import torch

from portdnn_amd import _native, capi, ops
from portdnn_amd.ops import NORM

BEYOND = [1 << 31, (1 << 32) + 4, -(1 << 31) - 1]


@pytest.mark.parametrize("value", BEYOND)
def test_parameter_records(value):
    for make in (lambda: capi.MatmulBiasActParams(m=value),
                 lambda: capi.ResidualNormParams(rows=value),
                 lambda: capi.LinearRecurrenceParams(steps=value),
                 lambda: capi.ConvParams(batch=value),
                 lambda: capi.DepthwiseParams(batch=value),
                 lambda: capi.PoolParams(batch=value)):
        with pytest.raises(OverflowError):
            make()
    least = capi.MatmulBiasActParams(m=(1 << 31) - 1, k=-(1 << 31))
    assert (least.m, least.k) == ((1 << 31) - 1, -(1 << 31))


@pytest.mark.parametrize("value", BEYOND)
def test_numbers_of_a_call(value):
    """An entry point that only counts how often it is called."""
    called = []

    def fn(*args):
        called.append(args)
        return 0

    p = ctypes.c_void_p
    norm = ctypes.CFUNCTYPE(ctypes.c_int, p, p, p)(fn)
    matmul = ctypes.CFUNCTYPE(ctypes.c_int, *[p] * 8, ctypes.c_size_t, p)(fn)
    recurrence = ctypes.CFUNCTYPE(ctypes.c_int, *[p] * 10, ctypes.c_size_t, p)(fn)

    def at(f):
        return ctypes.cast(f, p).value

    for call in (
            lambda: _native.residual_norm(
                at(norm), *[None] * 11, value, 8, 1, 1, 0, 1, 8, 8, 1e-6, 0),
            lambda: _native.matmul_bias_act(
                at(matmul), *[None] * 6, 4, value, 4, 0, 0, 0, 0, 0, 0, 0, None,
                0, 0),
            lambda: _native.linear_recurrence(
                at(recurrence), *[None] * 8, 1, 1, 8, value, 0, None, 0, 0)):
        with pytest.raises(OverflowError):
            call()
    assert not called


def test_tensors_of_more_rows(monkeypatch):
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    rows = (1 << 32) + 4
    x = torch.empty(rows, 8, dtype=torch.bfloat16, device="meta")
    w = torch.empty(8, 8, dtype=torch.bfloat16, device="meta")
    for call in (lambda: ops.residual_norm(x, pre=NORM.RMS),
                 lambda: ops.matmul_bias_act(x, w),
                 lambda: ops.matmul_bias_act(x, x, trans_a=True),
                 lambda: ops.linear_recurrence(x[None], x[None]),
                 lambda: ops.linear_recurrence(x[:, None], x[:, None])):
        with pytest.raises(OverflowError):
            call()
