"""What the operators of a linear-attention block refuse, and their workspace
queries: decided on the host before anything is launched."""
import ctypes
import math

import pytest
import torch

import attention_reference as plain
from portdnn_amd import capi, ops
from portdnn_amd.capi import (DTYPE, ROTARY_SCALING, STATUS, GatedMatmulParams,
                              LinearAttentionParams, RotaryParams)

FAKE = 0x1000  # never dereferenced: every call returns early
TYPES = ["f32", "f16", "bf16"]
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _sizes(name, p, *args):
    req, rec = ctypes.c_size_t(), ctypes.c_size_t()
    capi.check(getattr(capi.lib(), name)(ctypes.byref(p), *args,
                                         ctypes.byref(req), ctypes.byref(rec)))
    return req.value, rec.value


# ---- the gated product ----------------------------------------------------------


def _gated_params(**kw):
    return GatedMatmulParams(**{**dict(m=8, k=16, n=24), **kw})


def _gated(suffix, p, lhs=FAKE, gate_weight=FAKE, up_weight=FAKE, out=FAKE,
           gate=None, up=None, workspace=None, elems=0):
    return getattr(capi.lib(), "snn_hip_gated_matmul_" + suffix)(
        lhs, gate_weight, up_weight, None, None, out, gate, up,
        p and ctypes.byref(p), workspace, elems, None)


def _gated_grad(suffix, p, dy=FAKE, lhs=FAKE, gate_weight=FAKE, up_weight=FAKE,
                gate=FAKE, up=FAKE, d=(FAKE,) * 5, workspace=None, elems=0):
    return getattr(capi.lib(), "snn_hip_gated_matmul_grad_" + suffix)(
        dy, lhs, gate_weight, up_weight, gate, up, *d, p and ctypes.byref(p),
        workspace, elems, None)


BAD_GATED = [dict(m=0), dict(k=0), dict(n=-1), dict(activation=5),
             dict(activation=-1), dict(lhs_stride=15), dict(rhs_stride=23),
             dict(output_stride=23), dict(lhs_stride=-16),
             dict(transpose_rhs=1, rhs_stride=15)]


@pytest.mark.parametrize("suffix", TYPES)
def test_gated_refusals(suffix):
    for kw in BAD_GATED:
        p = _gated_params(**kw)
        assert _gated(suffix, p) == STATUS.INVALID_PARAMETER, kw
        assert _gated_grad(suffix, p) == STATUS.INVALID_PARAMETER, kw
    p = _gated_params()
    assert _gated(suffix, None) == STATUS.INVALID_PARAMETER
    assert _gated_grad(suffix, None) == STATUS.INVALID_PARAMETER
    for kw in (dict(lhs=None), dict(gate_weight=None), dict(up_weight=None),
               dict(out=None), dict(gate=FAKE), dict(up=FAKE),
               dict(workspace=FAKE + 8)):
        assert _gated(suffix, p, **kw) == STATUS.INVALID_PARAMETER, kw
    for kw in (dict(dy=None), dict(gate=None), dict(up=None), dict(lhs=None),
               dict(gate_weight=None), dict(up_weight=None),
               dict(d=(None,) * 5), dict(workspace=FAKE + 4)):
        assert _gated_grad(suffix, p, **kw) == STATUS.INVALID_PARAMETER, kw
    most = (1 << 29) // SIZE[suffix]
    for name in ("m", "k", "n"):
        assert (_gated(suffix, _gated_params(**{name: most})) ==
                STATUS.INDEX_EXCEEDED)
        assert (_gated_grad(suffix, _gated_params(**{name: most})) ==
                STATUS.INDEX_EXCEEDED)
    required, recommended = _sizes("snn_hip_gated_matmul_workspace_size", p, 1,
                                   getattr(DTYPE, suffix.upper()))
    assert 0 < required <= recommended
    for elems in (0, required - 1):
        assert (_gated_grad(suffix, p, workspace=FAKE, elems=elems) ==
                STATUS.INSUFFICIENT_WORKSPACE)
    assert _gated_grad(suffix, p) == STATUS.INSUFFICIENT_WORKSPACE


def test_gated_workspace():
    name = "snn_hip_gated_matmul_workspace_size"
    entry = getattr(capi.lib(), name)
    size = ctypes.c_size_t()
    p = _gated_params()
    at, out = ctypes.byref(p), ctypes.byref(size)
    assert entry(at, 0, 3, out, out) == STATUS.INVALID_PARAMETER
    assert entry(at, 0, -1, out, out) == STATUS.INVALID_PARAMETER
    assert entry(at, 0, 0, None, out) == STATUS.INVALID_PARAMETER
    assert entry(at, 0, 0, out, None) == STATUS.INVALID_PARAMETER
    assert entry(None, 0, 0, out, out) == STATUS.INVALID_PARAMETER
    assert (entry(ctypes.byref(_gated_params(k=0)), 0, 0, out, out) ==
            STATUS.INVALID_PARAMETER)
    # the forward call requires none; few rows and a long k are split
    assert _sizes(name, p, 0, DTYPE.BF16)[0] == 0
    assert _sizes(name, _gated_params(m=1, k=8192, n=64), 0, DTYPE.BF16)[1] > 0


# ---- positions by rotation ------------------------------------------------------


def _rotary(suffix, x=FAKE, table=FAKE, positions=None, out=FAKE, **kw):
    p = RotaryParams(**{**dict(batch=2, steps=3, heads=2, channels=8, turned=6,
                               magnitude=1.0), **kw})
    return getattr(capi.lib(), "snn_hip_rotary_" + suffix)(
        x, table, positions, out, ctypes.byref(p), None)


@pytest.mark.parametrize("suffix", TYPES)
def test_rotary_refusals(suffix):
    for kw in (dict(batch=0), dict(steps=-1), dict(heads=0), dict(channels=0),
               dict(turned=0), dict(turned=3), dict(turned=10), dict(layout=2),
               dict(layout=-1), dict(positions=3), dict(positions=-1),
               dict(row_stride=15), dict(output_row_stride=15),
               dict(magnitude=float("nan")), dict(magnitude=float("inf")),
               dict(x=None), dict(table=None), dict(out=None),
               dict(output_row_stride=20), dict(row_stride=20)):
        assert _rotary(suffix, **kw) == STATUS.INVALID_PARAMETER, kw
    p = RotaryParams(batch=2, steps=3, heads=2, channels=8, turned=6, positions=1,
                     magnitude=1.0)
    entry = getattr(capi.lib(), "snn_hip_rotary_" + suffix)
    # positions without an array, and an array without them
    assert (entry(FAKE, FAKE, None, FAKE, ctypes.byref(p), None) ==
            STATUS.INVALID_PARAMETER)
    p.positions = 0
    assert (entry(FAKE, FAKE, FAKE, FAKE, ctypes.byref(p), None) ==
            STATUS.INVALID_PARAMETER)
    assert entry(FAKE, FAKE, None, FAKE, None, None) == STATUS.INVALID_PARAMETER
    assert (_rotary(suffix, batch=1 << 16, steps=1 << 16, out=2 * FAKE) ==
            STATUS.INDEX_EXCEEDED)


def _frequencies(turned=8, base=10000.0, scaling=0, factor=1.0, context=0.0,
                 low=1.0, high=32.0, out=True):
    table = (ctypes.c_double * max(1, turned // 2))()
    return capi.lib().snn_hip_rotary_frequencies(
        turned, base, scaling, factor, context, low, high,
        ctypes.addressof(table) if out else None)


def test_frequencies():
    for kw in (dict(turned=0), dict(turned=7), dict(turned=-2), dict(out=False),
               dict(base=0.0), dict(base=-1.0), dict(base=math.inf),
               dict(scaling=4), dict(scaling=-1), dict(scaling=1, factor=0.0),
               dict(scaling=2, factor=math.nan), dict(scaling=3),
               dict(scaling=3, context=64.0, low=2.0, high=2.0),
               dict(scaling=3, context=64.0, high=math.inf)):
        assert _frequencies(**kw) == STATUS.INVALID_PARAMETER, kw
    for scaling in ("NONE", "POSITIONS", "BASE", "BANDS"):
        for turned in (2, 6, 128):
            kinds = dict(base=7000.0, factor=4.0, context=500.0, low=1.5,
                         high=20.0)
            got = ops.rotary_frequencies(
                turned, scaling=getattr(ROTARY_SCALING, scaling), device="cpu",
                **kinds)
            # (a power and a handful of operations in 64 bits)
            torch.testing.assert_close(
                got, plain.frequencies(turned, scaling=scaling, **kinds),
                rtol=1e-13, atol=0)


# ---- linear attention -----------------------------------------------------------


def _attention_params(**kw):
    return LinearAttentionParams(**{**dict(
        batch=2, steps=40, heads=4, key_heads=2, keys=16, values=24, scale=1.0),
        **kw})


def _attention(suffix, p, q=FAKE, k=FAKE, v=FAKE, decay=FAKE, out=FAKE,
               workspace=None, elems=0):
    return getattr(capi.lib(), "snn_hip_linear_attention_" + suffix)(
        q, k, v, decay, None, None, None, out, None, p and ctypes.byref(p),
        workspace, elems, None)


def _attention_grad(suffix, p, do=FAKE, q=FAKE, k=FAKE, v=FAKE, decay=FAKE,
                    d=(FAKE,) * 4, workspace=None, elems=0):
    return getattr(capi.lib(), "snn_hip_linear_attention_grad_" + suffix)(
        do, None, q, k, v, decay, None, None, None, *d, p and ctypes.byref(p),
        workspace, elems, None)


BAD_ATTENTION = [dict(batch=0), dict(steps=0), dict(heads=0), dict(key_heads=0),
                 dict(keys=0), dict(values=-1), dict(keys=257), dict(values=257),
                 dict(key_heads=3), dict(key_heads=8), dict(q_stride=31),
                 dict(k_stride=31), dict(v_stride=95), dict(v_stride=-96),
                 dict(grad_q_stride=31), dict(grad_k_stride=31),
                 dict(grad_v_stride=95), dict(scale=math.nan),
                 dict(scale=-math.inf)]
FAR_ATTENTION = [dict(steps=(1 << 30) + 1), dict(batch=1 << 19),
                 dict(q_stride=(1 << 22) + 1), dict(k_stride=(1 << 22) + 1),
                 dict(v_stride=(1 << 22) + 1), dict(grad_q_stride=(1 << 22) + 1),
                 dict(batch=1, heads=1 << 20, key_heads=1),
                 dict(batch=1, heads=1 << 20, key_heads=1 << 20, keys=1,
                      values=5)]


@pytest.mark.parametrize("suffix", TYPES)
def test_attention_refusals(suffix):
    for kw in BAD_ATTENTION:
        p = _attention_params(**kw)
        assert _attention(suffix, p) == STATUS.INVALID_PARAMETER, kw
        assert _attention_grad(suffix, p) == STATUS.INVALID_PARAMETER, kw
    for kw in FAR_ATTENTION:
        p = _attention_params(**kw)
        assert _attention(suffix, p) == STATUS.INDEX_EXCEEDED, kw
        assert _attention_grad(suffix, p) == STATUS.INDEX_EXCEEDED, kw
    p = _attention_params()
    assert _attention(suffix, None) == STATUS.INVALID_PARAMETER
    assert _attention_grad(suffix, None) == STATUS.INVALID_PARAMETER
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(decay=None),
               dict(out=None), dict(workspace=FAKE + 8)):
        assert _attention(suffix, p, **kw) == STATUS.INVALID_PARAMETER, kw
    for kw in (dict(do=None), dict(q=None), dict(k=None), dict(v=None),
               dict(decay=None), dict(d=(None,) * 4), dict(workspace=FAKE + 8)):
        assert _attention_grad(suffix, p, **kw) == STATUS.INVALID_PARAMETER, kw
    required, recommended = _sizes(
        "snn_hip_linear_attention_workspace_size", p, 1,
        getattr(DTYPE, suffix.upper()))
    # shared heads: fp32 sums of q's and k's gradients
    assert required == 2 * 2 * 40 * 4 * 16 * 4 // SIZE[suffix] <= recommended
    for elems in (0, required - 1):
        assert (_attention_grad(suffix, p, workspace=FAKE, elems=elems) ==
                STATUS.INSUFFICIENT_WORKSPACE)
    assert _attention_grad(suffix, p) == STATUS.INSUFFICIENT_WORKSPACE


@pytest.mark.parametrize("suffix", TYPES)
@pytest.mark.parametrize("heads,key_heads,keys,values", [
    (65536, 1, 256, 16), (65536, 16384, 256, 8), (32769, 1, 256, 16),
    (1 << 20, 1, 9, 1)])
def test_attention_sums_of_many_heads(suffix, heads, key_heads, keys, values):
    """A row of the sums over heads that share queries and keys holds heads * keys
    floats: beyond 2^23 of them a block's rows pass 31 bits of bytes."""
    p = _attention_params(batch=1, heads=heads, key_heads=key_heads, keys=keys,
                          values=values)
    entry = capi.lib().snn_hip_linear_attention_workspace_size
    code = getattr(DTYPE, suffix.upper())
    size = ctypes.c_size_t()
    out = ctypes.byref(size)

    def required(grad):
        return entry(ctypes.byref(p), grad, code, out, out)

    assert _attention_grad(suffix, p) == STATUS.INDEX_EXCEEDED
    assert required(1) == STATUS.INDEX_EXCEEDED
    # the forward call has no such sums
    assert required(0) == STATUS.OK
    # the largest row that is counted in 31 bits: the workspace is what is missing
    p.heads = (1 << 23) // keys // key_heads * key_heads
    assert _attention_grad(suffix, p) == STATUS.INSUFFICIENT_WORKSPACE
    assert required(1) == STATUS.OK
    if key_heads == 1:  # heads that share nothing: none
        p.heads = p.key_heads = (1 << 22) // keys
        assert required(1) == STATUS.OK


def test_attention_workspace():
    name = "snn_hip_linear_attention_workspace_size"
    entry = getattr(capi.lib(), name)
    size = ctypes.c_size_t()
    p = _attention_params()
    at, out = ctypes.byref(p), ctypes.byref(size)
    for args in ((at, 0, 3, out, out), (at, 0, -1, out, out),
                 (at, 0, 0, None, out), (at, 0, 0, out, None),
                 (None, 0, 0, out, out),
                 (ctypes.byref(_attention_params(heads=3)), 0, 0, out, out)):
        assert entry(*args) == STATUS.INVALID_PARAMETER
    for dtype in (DTYPE.F32, DTYPE.F16, DTYPE.BF16):
        # one head of a long sequence is divided, a few steps and many heads not
        long = _attention_params(batch=1, steps=8192, heads=1, key_heads=1)
        required, recommended = _sizes(name, long, 0, dtype)
        assert required == 0 < recommended
        assert _sizes(name, _attention_params(steps=16), 0, dtype) == (0, 0)
        many = _attention_params(batch=512, heads=4, key_heads=4, steps=64)
        assert _sizes(name, many, 0, dtype) == (0, 0)
        assert _sizes(name, long, 1, dtype)[0] == 0


def test_python_refusals():
    """Operands that the entry points could not tell from others."""
    def normal(*shape):
        return torch.zeros(shape)

    q, v = normal(2, 5, 2, 8), normal(2, 5, 4, 8)
    decay = normal(4)
    for bad in (dict(q=q.transpose(1, 2)), dict(q=q[..., ::2]), dict(k=q[:, 1:]),
                dict(k=q.half()), dict(decay=decay[1:]),
                dict(decay=decay.double()), dict(resets=normal(2, 5)),
                dict(resets=torch.zeros(2, 4, dtype=torch.uint8)),
                dict(lengths=torch.zeros(2, dtype=torch.int64)),
                dict(lengths=torch.zeros(3, dtype=torch.int32)),
                dict(initial_state=normal(2, 4, 8, 7)),
                dict(initial_state=normal(2, 4, 8, 8).half()),
                dict(out=normal(2, 5, 4, 9)), dict(final_state=normal(4, 8, 8))):
        with pytest.raises(AssertionError):
            ops.linear_attention(**{**dict(q=q, k=q, v=v, decay=decay), **bad})
    table = torch.zeros(4, dtype=torch.float64)
    for bad in (dict(frequencies=table.float()), dict(frequencies=table[::2]),
                dict(positions=torch.zeros(2)),
                dict(positions=torch.zeros(3, dtype=torch.int32)),
                dict(positions=torch.zeros(2, 4, dtype=torch.int32)),
                dict(out=normal(2, 5, 2, 9)), dict(x=q.transpose(0, 1))):
        with pytest.raises(AssertionError):
            ops.rotary(**{**dict(x=q, frequencies=table), **bad})
    a, w = normal(3, 4), normal(4, 5)
    for bad in (dict(w_up=normal(4, 6)), dict(w_up=w.half()), dict(a=normal(3, 5)),
                dict(bias_gate=normal(4)), dict(bias_up=normal(5).half()),
                dict(out=normal(3, 6)), dict(a=a.T),
                dict(w_up=normal(4, 10)[:, :5])):
        with pytest.raises(AssertionError):
            ops.gated_matmul(**{**dict(a=a, w_gate=w, w_up=w), **bad})


@pytest.mark.parametrize("size", [(), (2, 5, 2), (2, 5, 2, 8), (2, 5, 2, 8, 1)])
def test_positions_of_anything_but_sequences_or_tokens(size):
    """They would be read as the tokens', which one number for all is too short for."""
    x = torch.zeros(2, 5, 2, 8)
    table = torch.zeros(4, dtype=torch.float64)
    with pytest.raises(AssertionError):
        ops.rotary(x, table, positions=torch.zeros(size, dtype=torch.int32))
