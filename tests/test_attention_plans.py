"""How linear attention goes over sequences: that the calls of attention_kernel_cases
reach every kernel.  Decided on the host."""
import ctypes

import pytest
import torch

from attention_kernel_cases import CASES
from portdnn_amd import capi, ops
from portdnn_amd.capi import DTYPE, STATUS, LinearAttentionParams

TYPES = {"f32": [torch.float32], "16": [torch.float16, torch.bfloat16]}


def kernels(kind):
    """(outputs, keys, waves, blocks in the ring) of all kernels of a type."""
    got = set()
    for outputs in (0, 1):
        for keys in (64, 128, 256):
            rings = {0, 1, 2} if keys == 64 else {0, 1}
            got |= {(outputs, keys, 4, ring) for ring in rings}
            if kind == "16":
                rings = {0, 1} if keys == 256 else {0, 2 + outputs}
                got |= {(outputs, keys, 8, ring) for ring in rings}
    return got


def launches_of(case, dtype, **kinds):
    return ops.linear_attention_plan(
        case.batch, case.steps, case.heads, case.key_heads, case.keys,
        case.values, dtype, grad=case.grad, **kinds)


def kernels_of(case, dtype):
    return {(l["outputs"], l["keys"], l["waves"], l["ring"])
            for l in launches_of(case, dtype)[2]}


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("grad", [0, 1])
def test_the_cases_reach_every_kernel(kind, grad):
    for dtype in TYPES[kind]:
        got = set()
        for c in CASES:
            if (c.type, c.grad) == (kind, grad):
                got |= kernels_of(c, dtype)
        assert got == kernels(kind)


def test_rows_at_other_addresses_pass_through_registers():
    for c in CASES:
        for dtype in TYPES[c.type]:
            for kinds in (dict(aligned=False),
                          dict(v_stride=c.heads * c.values + 3)):
                for l in launches_of(c, dtype, **kinds)[2]:
                    assert l["ring"] == 0


def test_without_a_workspace_sequences_are_whole():
    for c in CASES:
        for dtype in TYPES[c.type]:
            pieces, steps, launches = launches_of(c, dtype)
            assert (pieces - 1) * steps < c.steps <= pieces * steps
            states = [l for l in launches if l["outputs"] == 0]
            assert len(states) == (pieces > 1)
            if not c.grad:
                pieces, _, launches = launches_of(c, dtype, workspace_elems=0)
                assert pieces == 1 and len(launches) == 1


def test_a_few_steps_have_no_blocks():
    assert ops.linear_attention_plan(2, 12, 2, 2, 64, 64, torch.float16) == \
        (1, 0, [])


@pytest.mark.parametrize("dtype", [DTYPE.F32, DTYPE.F16, DTYPE.BF16])
def test_refusals(dtype):
    fn = capi.lib().snn_hip_linear_attention_planned
    plan = capi.LinearAttentionPlan()
    sizes = dict(batch=1, steps=40, heads=4, key_heads=2, keys=16, values=24,
                 scale=1.0)

    def call(grad=0, kind=dtype, elems=1 << 20, to=plan, **kw):
        p = LinearAttentionParams(**{**sizes, **kw})
        return fn(ctypes.byref(p), grad, kind, 1, elems, to and ctypes.byref(to))

    assert call() == call(grad=1) == STATUS.OK
    for kw in (dict(kind=3), dict(kind=-1), dict(to=None), dict(keys=257),
               dict(heads=3)):
        assert call(**kw) == STATUS.INVALID_PARAMETER, kw
    assert fn(None, 0, dtype, 1, 0, ctypes.byref(plan)) == \
        STATUS.INVALID_PARAMETER
    assert call(grad=1, elems=0) == STATUS.INSUFFICIENT_WORKSPACE
    many = dict(heads=65536, key_heads=1, keys=256, values=16)
    assert call(grad=1, **many) == STATUS.INDEX_EXCEEDED
    assert call(**many) == STATUS.OK
