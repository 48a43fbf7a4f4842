"""Torch-tensor conveniences over the C ABI, used by the tests and bench.py.

torch is plumbing here (device memory and the current HIP stream); every
computation happens in libsnn_hip.so.  There is no fallback path.
"""
import ctypes

import torch

from . import _native, capi
from .capi import ACTIVATION, ALGO, BINARY_OP, DIRECTION, DTYPE, GATE, NORM, \
    POINTWISE_OP, POOL_OP, ROTARY, ROTARY_POSITIONS, ROTARY_SCALING, STATUS, \
    ConvParams, DepthwiseParams, GatedMatmulParams, LinearAttentionParams, \
    LinearRecurrenceParams, MatmulBiasActParams, PoolParams, ResidualNormParams


def calculate_padding(inp, window, stride, same):
    """helpers::calculate_padding (include/portdnn/helpers/padding.h:51-69):
    returns (padding, output)."""
    if same:
        out = (inp + stride - 1) // stride
        needed = (out - 1) * stride + window - inp
        return int(needed / 2), out  # C++ integer division truncates
    num = inp - window + 1
    q = int(num / stride)
    return 0, (q if num < 0 else q + (1 if num % stride else 0))


def add_padding_to(params, same):
    """helpers::add_padding_to (include/portdnn/helpers/padding.h:80-92)."""
    params.pad_rows, params.out_rows = calculate_padding(
        params.in_rows, params.window_rows, params.stride_rows, same)
    params.pad_cols, params.out_cols = calculate_padding(
        params.in_cols, params.window_cols, params.stride_cols, same)
    return params


def conv_params(batch, in_rows, in_cols, channels, features, window, stride,
                same):
    return add_padding_to(ConvParams(
        channels=channels, features=features, batch=batch, in_rows=in_rows,
        in_cols=in_cols, window_rows=window, window_cols=window,
        stride_rows=stride, stride_cols=stride), same)


def depthwise_params(batch, in_rows, in_cols, channels, multiplier, window,
                     stride, same):
    return add_padding_to(DepthwiseParams(
        channels=channels, channel_multiplier=multiplier, batch=batch,
        in_rows=in_rows, in_cols=in_cols, window_rows=window,
        window_cols=window, stride_rows=stride, stride_cols=stride), same)


def pool_params(batch, in_rows, in_cols, channels, window, stride, same):
    return add_padding_to(PoolParams(
        in_rows=in_rows, in_cols=in_cols, window_rows=window,
        window_cols=window, stride_rows=stride, stride_cols=stride,
        batch=batch, channels=channels), same)


def conv_sizes(p, direction):
    """(input, filter, output) element counts, conv2d/sizes.h:166-179."""
    x = p.batch * p.in_rows * p.in_cols * p.channels
    w = p.window_rows * p.window_cols * p.channels * p.features
    y = p.batch * p.out_rows * p.out_cols * p.features
    if direction == DIRECTION.FORWARD:
        return x, w, y
    if direction == DIRECTION.INPUT_BACKPROP:
        return y, w, x
    return x, y, w


def conv_flops(p, direction):
    """bench/conv2d/base_convolution_fixture.h:81-109."""
    if direction == DIRECTION.FORWARD:
        pix = p.batch * p.out_rows * p.out_cols
    else:
        pix = p.batch * p.in_rows * p.in_cols
    return 2 * pix * p.window_rows * p.window_cols * p.channels * p.features


def _stream():
    # (torch.cuda.current_stream().cuda_stream without the object it builds)
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


# The calls below that a program makes per layer and step go through _native
# (csrc/py_native.cpp), which converts the arguments, checks the operand sizes
# and calls the entry point.  Back to back, against the same calls through
# ctypes: one small depthwise layer 7.9 -> 4.5 us, convolution + bias + ReLU
# 24.3 -> 18.0, the three directions of a small 1x1 layer 28.1 -> 20.9.
_addresses = {}


def _address(name):
    """The address of an entry point of the loaded library."""
    at = _addresses.get(name)
    if at is None:
        at = _addresses[name] = ctypes.cast(
            getattr(capi.lib(), name), ctypes.c_void_p).value
    return at


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _at(t):
    """The address for _native; a missing operand is the entry point's error."""
    return None if t is None else t.data_ptr()


def _room(workspace, t):
    """The elements of t's type that a caller's workspace, of whatever type, has
    memory for: what the entry points count a workspace in."""
    assert workspace.is_contiguous(), "a workspace that is not contiguous"
    n = workspace.numel()
    if workspace.dtype is t.dtype:
        return n
    return n * workspace.element_size() // t.element_size()


def workspace_size(p, direction, algorithm, dtype=None):
    """(required, recommended) elements; with a capi.DTYPE the element type's
    own answer (snn_hip_conv2d_workspace_size_for)."""
    req, rec = ctypes.c_size_t(), ctypes.c_size_t()
    if dtype is None:
        capi.check(capi.lib().snn_hip_conv2d_workspace_size(
            ctypes.byref(p), direction, algorithm, ctypes.byref(req),
            ctypes.byref(rec)))
    else:
        capi.check(capi.lib().snn_hip_conv2d_workspace_size_for(
            ctypes.byref(p), direction, algorithm, dtype, ctypes.byref(req),
            ctypes.byref(rec)))
    return req.value, rec.value


def default_algorithm(p, direction, dtype=None):
    """The library's default selector's choice (for a capi.DTYPE when given)."""
    if dtype is None:
        return capi.lib().snn_hip_conv2d_default_algorithm(ctypes.byref(p),
                                                           direction)
    return capi.lib().snn_hip_conv2d_default_algorithm_for(
        ctypes.byref(p), direction, dtype)


def gather_tile(p, direction, dtype):
    """(pixels, features, splits) of the gathering kernel's tile, or None where
    such a launch runs on another kernel (snn_hip_conv2d_gather_tile)."""
    pixels, features, splits = (ctypes.c_int() for _ in range(3))
    code = capi.lib().snn_hip_conv2d_gather_tile(
        ctypes.byref(p), direction, dtype, ctypes.byref(pixels),
        ctypes.byref(features), ctypes.byref(splits))
    if code == STATUS.INVALID_ALGORITHM:
        return None
    capi.check(code)
    return pixels.value, features.value, splits.value


def halves_tile(p, direction, algorithm):
    """(pixels, features) of the fp32 kernel whose operands are taken apart into
    binary16 values, or None where such a launch runs on another kernel
    (snn_hip_conv2d_halves_tile)."""
    pixels, features = ctypes.c_int(), ctypes.c_int()
    code = capi.lib().snn_hip_conv2d_halves_tile(
        ctypes.byref(p), direction, algorithm, ctypes.byref(pixels),
        ctypes.byref(features))
    if code == STATUS.INVALID_ALGORITHM:
        return None
    capi.check(code)
    return pixels.value, features.value


def filter_halves_partials(p, algorithm):
    """Partial filters of the fp32 filter gradient whose operands are taken apart into
    binary16 values, or None where such a launch runs on another kernel
    (snn_hip_conv2d_filter_halves_partials)."""
    partials = ctypes.c_int()
    code = capi.lib().snn_hip_conv2d_filter_halves_partials(
        ctypes.byref(p), algorithm, ctypes.byref(partials))
    if code == STATUS.INVALID_ALGORITHM:
        return None
    capi.check(code)
    return partials.value


def lds_form_f16(p, direction):
    """How a binary16 launch keeps its pixels in LDS, or None where it runs on
    another kernel (snn_hip_conv2d_lds_form_f16)."""
    form = ctypes.c_int()
    code = capi.lib().snn_hip_conv2d_lds_form_f16(
        ctypes.byref(p), direction, ctypes.byref(form))
    if code == STATUS.INVALID_ALGORITHM:
        return None
    capi.check(code)
    return form.value


_CONV_FN = {
    (DIRECTION.FORWARD, torch.float32): "snn_hip_conv2d_forward_f32",
    (DIRECTION.INPUT_BACKPROP, torch.float32):
        "snn_hip_conv2d_input_backprop_f32",
    (DIRECTION.FILTER_BACKPROP, torch.float32):
        "snn_hip_conv2d_filter_backprop_f32",
    (DIRECTION.FORWARD, torch.float16): "snn_hip_conv2d_forward_f16",
    (DIRECTION.INPUT_BACKPROP, torch.float16):
        "snn_hip_conv2d_input_backprop_f16",
    (DIRECTION.FILTER_BACKPROP, torch.float16):
        "snn_hip_conv2d_filter_backprop_f16",
}


def conv2d_raw(inp, fil, out, p, direction, algorithm, workspace=None):
    """Calls the entry point and returns its status code (no exception)."""
    fn = getattr(capi.lib(), _CONV_FN[(direction, inp.dtype)])
    return fn(_ptr(inp), _ptr(fil), _ptr(out), ctypes.byref(p), algorithm,
              _ptr(workspace),
              0 if workspace is None else _room(workspace, inp), _stream())


def conv2d(inp, fil, p, direction=DIRECTION.FORWARD, algorithm=ALGO.DIRECT,
           workspace=None, out=None):
    """inp / fil are flat or shaped device tensors with the operand roles of
    include/snn_hip.h; returns the flat output tensor."""
    assert inp.is_contiguous() and fil.is_contiguous()
    dtype = inp.dtype
    if out is None:
        out = torch.empty(conv_sizes(p, direction)[2], dtype=dtype,
                          device=inp.device)
    if (workspace is None and dtype == torch.float32 and
            algorithm in (ALGO.WINOGRAD, ALGO.WINOGRAD_LARGE)):
        _, rec = workspace_size(p, direction, algorithm)
        workspace = torch.empty(rec, dtype=dtype, device=inp.device)
    code = _native.conv2d(
        _address(_CONV_FN[direction, dtype]), direction, inp.data_ptr(),
        inp.numel(), fil.data_ptr(), fil.numel(), out.data_ptr(), p, algorithm,
        _at(workspace), 0 if workspace is None else _room(workspace, out),
        _stream())
    if code:
        capi.check(code)
    return out


def _bind(fn, *cargs):
    """A zero-argument callable that makes one C ABI call with arguments
    converted once: timing loops over kernels of a few microseconds would
    otherwise measure the per-call conversions of the wrappers above (6-7 us
    against 2 for the call itself).  The stream is the one current now."""
    def call():
        code = fn(*cargs)
        if code:
            capi.check(code)
    return call


def conv2d_bound(inp, fil, out, p, direction, algorithm, workspace=None):
    """conv2d with everything fixed: returns the callable that launches it."""
    n_in, n_fil, n_out = conv_sizes(p, direction)
    assert (inp.numel(), fil.numel(), out.numel()) == (n_in, n_fil, n_out)
    assert inp.is_contiguous() and fil.is_contiguous() and out.is_contiguous()
    fn = getattr(capi.lib(), _CONV_FN[(direction, inp.dtype)])
    return _bind(fn, _ptr(inp), _ptr(fil), _ptr(out), ctypes.byref(p),
                 algorithm, _ptr(workspace),
                 0 if workspace is None else _room(workspace, inp),
                 ctypes.c_void_p(_stream()))


def conv2d_prepared_bound(inp, fil, out, p, direction, algorithm, workspace):
    """conv2d_prepared with everything fixed."""
    return _bind(capi.lib().snn_hip_conv2d_prepared_f32, direction, _ptr(inp),
                 _ptr(fil), _ptr(out), ctypes.byref(p), algorithm,
                 _ptr(workspace),
                 0 if workspace is None else _room(workspace, inp),
                 ctypes.c_void_p(_stream()))


def conv2d_prepare_filter(fil, p, direction, algorithm, workspace):
    """snn_hip_conv2d_prepare_filter_f32: what the launch derives from the
    filter alone goes into `workspace`."""
    capi.check(capi.lib().snn_hip_conv2d_prepare_filter_f32(
        direction, _ptr(fil), ctypes.byref(p), algorithm, _ptr(workspace),
        0 if workspace is None else _room(workspace, fil), _stream()))


def conv2d_prepared(inp, fil, p, direction, algorithm, workspace, out=None):
    """snn_hip_conv2d_prepared_f32: the launch that trusts a prepared
    workspace."""
    _, _, n_out = conv_sizes(p, direction)
    if out is None:
        out = torch.empty(n_out, dtype=inp.dtype, device=inp.device)
    capi.check(capi.lib().snn_hip_conv2d_prepared_f32(
        direction, _ptr(inp), _ptr(fil), _ptr(out), ctypes.byref(p), algorithm,
        _ptr(workspace), 0 if workspace is None else _room(workspace, inp),
        _stream()))
    return out


def conv2d_deterministic(inp, fil, p, direction, algorithm, workspace=None,
                         out=None):
    """snn_hip_conv2d_deterministic_f32: fixed order of additions."""
    n_in, n_fil, n_out = conv_sizes(p, direction)
    assert inp.numel() == n_in and fil.numel() == n_fil
    if out is None:
        out = torch.empty(n_out, dtype=inp.dtype, device=inp.device)
    if workspace is None:
        _, rec = workspace_size(p, direction, algorithm)
        if rec:
            workspace = torch.empty(rec, dtype=inp.dtype, device=inp.device)
    capi.check(capi.lib().snn_hip_conv2d_deterministic_f32(
        direction, _ptr(inp), _ptr(fil), _ptr(out), ctypes.byref(p), algorithm,
        _ptr(workspace), 0 if workspace is None else _room(workspace, inp),
        _stream()))
    return out


def conv2d_bias_act(inp, fil, bias, p, algorithm, relu=True, workspace=None,
                    out=None):
    """snn_hip_conv2d_forward_bias_act_f32: act(conv(inp, fil) + bias)."""
    if out is None:
        out = torch.empty(conv_sizes(p, DIRECTION.FORWARD)[2], dtype=inp.dtype,
                          device=inp.device)
    if workspace is None and algorithm in (ALGO.WINOGRAD, ALGO.WINOGRAD_LARGE):
        _, rec = workspace_size(p, DIRECTION.FORWARD, algorithm)
        workspace = torch.empty(rec, dtype=inp.dtype, device=inp.device)
    code = _native.conv2d_bias_act(
        _address("snn_hip_conv2d_forward_bias_act_f32"), _at(inp), _at(fil),
        _at(bias), out.data_ptr(), p, algorithm, 1 if relu else 0,
        _at(workspace), 0 if workspace is None else _room(workspace, out),
        _stream())
    if code:
        capi.check(code)
    return out


_DW_FN = {
    (DIRECTION.FORWARD, torch.float32): "snn_hip_depthwise_conv2d_forward_f32",
    (DIRECTION.INPUT_BACKPROP, torch.float32):
        "snn_hip_depthwise_conv2d_input_backprop_f32",
    (DIRECTION.FILTER_BACKPROP, torch.float32):
        "snn_hip_depthwise_conv2d_filter_backprop_f32",
    (DIRECTION.FORWARD, torch.float16): "snn_hip_depthwise_conv2d_forward_f16",
    (DIRECTION.INPUT_BACKPROP, torch.float16):
        "snn_hip_depthwise_conv2d_input_backprop_f16",
    (DIRECTION.FILTER_BACKPROP, torch.float16):
        "snn_hip_depthwise_conv2d_filter_backprop_f16",
}


def depthwise_sizes(p, direction):
    x = p.batch * p.in_rows * p.in_cols * p.channels
    w = p.window_rows * p.window_cols * p.channels * p.channel_multiplier
    y = p.batch * p.out_rows * p.out_cols * p.channels * p.channel_multiplier
    if direction == DIRECTION.FORWARD:
        return x, w, y
    if direction == DIRECTION.INPUT_BACKPROP:
        return y, w, x
    return x, y, w


def depthwise_conv2d(inp, fil, p, direction=DIRECTION.FORWARD, out=None):
    if out is None:
        out = torch.empty(depthwise_sizes(p, direction)[2], dtype=inp.dtype,
                          device=inp.device)
    code = _native.depthwise(
        _address(_DW_FN[direction, inp.dtype]), direction, inp.data_ptr(),
        inp.numel(), fil.data_ptr(), fil.numel(), out.data_ptr(), p, _stream())
    if code:
        capi.check(code)
    return out


def depthwise_conv2d_bound(inp, fil, out, p, direction=DIRECTION.FORWARD):
    """depthwise_conv2d with everything fixed (see _bind)."""
    n_in, n_fil, n_out = depthwise_sizes(p, direction)
    assert (inp.numel(), fil.numel(), out.numel()) == (n_in, n_fil, n_out)
    fn = getattr(capi.lib(), _DW_FN[(direction, inp.dtype)])
    return _bind(fn, _ptr(inp), _ptr(fil), _ptr(out), ctypes.byref(p),
                 ctypes.c_void_p(_stream()))


def pooling_forward_bound(inp, out, p, op):
    """pooling_forward with everything fixed (see _bind)."""
    assert inp.numel() == p.batch * p.in_rows * p.in_cols * p.channels
    assert out.numel() == p.batch * p.out_rows * p.out_cols * p.channels
    name = ("snn_hip_pooling_forward_f32" if inp.dtype == torch.float32 else
            "snn_hip_pooling_forward_f16")
    return _bind(getattr(capi.lib(), name), _ptr(inp), _ptr(out),
                 ctypes.byref(p), op, ctypes.c_void_p(_stream()))


def pooling_forward(inp, p, op, out=None):
    if out is None:
        out = torch.empty(p.batch * p.out_rows * p.out_cols * p.channels,
                          dtype=inp.dtype, device=inp.device)
    code = _native.pooling_forward(
        _address("snn_hip_pooling_forward" + _suffix(inp)), inp.data_ptr(),
        inp.numel(), out.data_ptr(), p, op, _stream())
    if code:
        capi.check(code)
    return out


def pooling_max_grad(inp, out, dy, p, op=POOL_OP.MAX, dx=None):
    if dx is None:
        dx = torch.empty_like(inp)
    code = _native.pooling_max_grad(
        _address("snn_hip_pooling_max_grad" + _suffix(inp)), inp.data_ptr(),
        _at(out), _at(dy), dx.data_ptr(), p, op, _stream())
    if code:
        capi.check(code)
    return dx


def pooling_avg_grad(dy, p, dx=None):
    if dx is None:
        dx = torch.empty(p.batch * p.in_rows * p.in_cols * p.channels,
                         dtype=dy.dtype, device=dy.device)
    code = _native.pooling_avg_grad(
        _address("snn_hip_pooling_avg_grad" + _suffix(dy)), dy.data_ptr(),
        dx.data_ptr(), p, _stream())
    if code:
        capi.check(code)
    return dx


def matmul(a, b, batches, m, k, n, trans_a=False, trans_b=False, beta=0.0,
           out=None):
    assert a.numel() == batches * m * k and b.numel() == batches * k * n
    if out is None:
        out = torch.zeros(batches * m * n, dtype=a.dtype, device=a.device)
    name = ("snn_hip_matmul_f32" if a.dtype == torch.float32 else
            "snn_hip_matmul_f16")
    capi.check(getattr(capi.lib(), name)(
        _ptr(a), _ptr(b), _ptr(out), batches, m, k, n, int(trans_a),
        int(trans_b), float(beta), _stream()))
    return out


def _suffix(t):
    return "_f32" if t.dtype == torch.float32 else "_f16"


def pointwise_forward(x, op, out=None):
    """sycldnn::pointwise::launch<T, Op, Forward>; `out` may be `x`."""
    if out is None:
        out = torch.empty_like(x)
    code = _native.pointwise_forward(
        _address("snn_hip_pointwise_forward" + _suffix(x)), x.data_ptr(),
        out.data_ptr(), x.numel(), op, _stream())
    if code:
        capi.check(code)
    return out


def pointwise_forward_bound(x, out, op):
    """pointwise_forward with everything fixed (see _bind)."""
    assert out.numel() == x.numel()
    fn = getattr(capi.lib(), "snn_hip_pointwise_forward" + _suffix(x))
    return _bind(fn, _ptr(x), _ptr(out), x.numel(), op,
                 ctypes.c_void_p(_stream()))


def pointwise_grad(val, err, op, out=None):
    """sycldnn::pointwise::launch<T, Op, Gradient>: `val` is the forward
    output (the forward input for LOG), `err` the incoming gradient."""
    if out is None:
        out = torch.empty_like(val)
    fn = getattr(capi.lib(), "snn_hip_pointwise_grad" + _suffix(val))
    capi.check(fn(_ptr(val), _ptr(err), _ptr(out), val.numel(), op, _stream()))
    return out


def binaryop_raw(lhs, rhs, out, lhs_dims, rhs_dims, op):
    """Calls the entry point and returns its status code (no exception)."""
    ld = (ctypes.c_int * max(len(lhs_dims), 1))(*lhs_dims)
    rd = (ctypes.c_int * max(len(rhs_dims), 1))(*rhs_dims)
    fn = getattr(capi.lib(), "snn_hip_binaryop" + _suffix(lhs))
    return fn(_ptr(lhs), _ptr(rhs), _ptr(out), ld, len(lhs_dims), rd,
              len(rhs_dims), op, _stream())


def binaryop(lhs, rhs, lhs_dims, rhs_dims, op, out=None):
    """sycldnn::binaryop::launch<T, Op> with BinaryParams{lhs_dims, rhs_dims};
    `out` may be either operand when that operand has the output's shape."""
    if out is None:
        n = max(len(lhs_dims), len(rhs_dims), 1)
        l = [1] * (n - len(lhs_dims)) + list(lhs_dims)
        r = [1] * (n - len(rhs_dims)) + list(rhs_dims)
        size = 1
        for a, b in zip(l, r):
            size *= max(a, b)
        out = torch.empty(size, dtype=lhs.dtype, device=lhs.device)
    code = _native.binaryop(
        _address("snn_hip_binaryop" + _suffix(lhs)), lhs.data_ptr(), _at(rhs),
        out.data_ptr(), lhs_dims, rhs_dims, op, _stream())
    if code:
        capi.check(code)
    return out


# ---- a residual block over sequences -----------------------------------------
# The operators below take their sizes and strides from the tensors: a matrix is
# a 2-D tensor, a sequence a [batch, steps, channels] one, whose rows may be
# slices of wider ones.

_TYPES = {torch.float32: ("_f32", DTYPE.F32), torch.float16: ("_f16", DTYPE.F16),
          torch.bfloat16: ("_bf16", DTYPE.BF16)}


def _row_stride(t):
    """Elements from row to row of a matrix whose rows are contiguous."""
    rows, cols = t.shape
    if rows == 1:
        assert cols == 1 or t.stride(1) == 1
        return cols
    step, unit = t.stride()
    assert (unit == 1 or cols == 1) and step >= cols, "rows are not contiguous"
    return step


def _step_stride(t):
    """Elements from step to step of a [batch, steps, channels] tensor."""
    batch, steps, channels = t.shape
    outer, step, unit = t.stride()
    assert unit == 1 or channels == 1, "channels are not contiguous"
    if steps == 1:
        step = outer if batch > 1 else channels
    else:
        assert batch == 1 or outer == steps * step, \
            "sequences do not follow one another"
    assert step >= channels
    return step


def _empty_like(t):
    """A tensor of t's shape whose rows follow one another.  (Taking the layout
    over is 0.6 us faster than a shape, of small calls of 8.)"""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _vector(t, n, dtype):
    """The address of an optional vector of n values."""
    if t is None:
        return None
    assert t.dtype is dtype and t.numel() == n and t.is_contiguous()
    return t.data_ptr()


def _like(t, shape, dtype):
    """The address of an optional contiguous tensor."""
    if t is None:
        return None
    assert t.shape == shape and t.dtype == dtype and t.is_contiguous()
    return t.data_ptr()


# What a call derives from its operands' sizes, strides and types (and from
# nothing else): settled once, as small calls are bound by the interpreter.
_plans = {}
_MOST_PLANS = 4096


def _keep(key, plan):
    if len(_plans) >= _MOST_PLANS:  # (lengths that never come again)
        _plans.clear()
    _plans[key] = plan
    return plan


def _workspace(entry, params, *args):
    """The recommended elements of a workspace."""
    req, rec = ctypes.c_size_t(), ctypes.c_size_t()
    capi.check(getattr(capi.lib(), entry)(
        ctypes.byref(params), *args, ctypes.byref(req), ctypes.byref(rec)))
    return rec.value


def _matmul_plan(key, a, b, grad, activation, trans_a, trans_b):
    dtype = a.dtype
    m, k = (a.shape[1], a.shape[0]) if trans_a else a.shape
    n = b.shape[0] if trans_b else b.shape[1]
    assert (b.shape[1] if trans_b else b.shape[0]) == k and b.dtype == dtype
    suffix, code = _TYPES[dtype]
    out_stride = 0
    if grad is not None:
        assert grad.shape == (m, n) and grad.dtype == dtype
        out_stride = _row_stride(grad)
    p = MatmulBiasActParams(
        m=m, k=k, n=n, transpose_lhs=int(trans_a), transpose_rhs=int(trans_b),
        activation=activation, lhs_stride=_row_stride(a),
        rhs_stride=_row_stride(b), output_stride=out_stride)
    elems = _workspace("snn_hip_matmul_bias_act_workspace_size", p,
                       int(grad is not None), code)
    name = "snn_hip_matmul_bias_act" + ("_grad" if grad is not None else "")
    return _keep(key, (_address(name + suffix), m, k, n, p.lhs_stride,
                       p.rhs_stride, out_stride, elems))


def matmul_plan(m, k, n, dtype, product=0, activation=ACTIVATION.NONE,
                trans_a=False, trans_b=False, aligned=True, workspace_elems=None,
                **strides):
    """What a product runs on (snn_hip_matmul_bias_act_planned), a dict by the names
    of capi.MATMUL_PLAN; by default with the recommended workspace."""
    p = MatmulBiasActParams(m=m, k=k, n=n, transpose_lhs=int(trans_a),
                            transpose_rhs=int(trans_b), activation=activation,
                            **strides)
    code = _TYPES[dtype][1]
    if workspace_elems is None:
        workspace_elems = _workspace("snn_hip_matmul_bias_act_workspace_size", p,
                                     int(product > 0), code)
    plan = capi.MatmulBiasActPlan()
    capi.check(capi.lib().snn_hip_matmul_bias_act_planned(
        ctypes.byref(p), product, code, int(aligned), workspace_elems,
        ctypes.byref(plan)))
    return {name: getattr(plan, name) for name in capi.MATMUL_PLAN}


def matmul_bias_act(a, b, bias=None, residual=None,
                    activation=ACTIVATION.NONE, trans_a=False, trans_b=False,
                    keep_pre_activation=False, out=None, workspace=None):
    """snn_hip_matmul_bias_act: act(op(a) op(b) + bias) + residual.  With
    keep_pre_activation returns (output, op(a) op(b) + bias), of which the
    gradient takes the second.  `out` may be the residual."""
    dtype = a.dtype
    key = (a.shape, a.stride(), b.shape, b.stride(), dtype, b.dtype, activation,
           trans_a, trans_b)
    plan = _plans.get(key)
    if plan is None:
        plan = _matmul_plan(key, a, b, None, activation, trans_a, trans_b)
    fn, m, k, n, a_stride, b_stride, _, elems = plan
    if out is None:
        out = a.new_empty((m, n))
        out_stride = n
    else:
        assert out.shape == (m, n) and out.dtype == dtype
        out_stride = _row_stride(out)
    add, add_stride = None, 0
    if residual is not None:
        assert residual.shape == (m, n) and residual.dtype == dtype
        add, add_stride = residual.data_ptr(), _row_stride(residual)
    z = a.new_empty((m, n)) if keep_pre_activation else None
    if workspace is None:
        if elems:
            workspace = a.new_empty(elems)
    else:
        elems = _room(workspace, a)
    code = _native.matmul_bias_act(
        fn, a.data_ptr(), b.data_ptr(), _vector(bias, n, dtype), add,
        out.data_ptr(), _at(z), m, k, n, trans_a, trans_b, activation, a_stride,
        b_stride, add_stride, out_stride, _at(workspace), elems, _stream())
    if code:
        capi.check(code)
    return (out, z) if keep_pre_activation else out


def matmul_bias_act_grad(grad, a, b, pre_activation=None,
                         activation=ACTIVATION.NONE, trans_a=False,
                         trans_b=False, bias=True, need_a=True, need_b=True,
                         workspace=None):
    """snn_hip_matmul_bias_act_grad: the gradients of a, b and the bias, None
    for those that are not wanted (the residual's is `grad` itself)."""
    dtype = a.dtype
    key = (a.shape, a.stride(), b.shape, b.stride(), grad.shape, grad.stride(),
           dtype, b.dtype, grad.dtype, activation, trans_a, trans_b)
    plan = _plans.get(key)
    if plan is None:
        plan = _matmul_plan(key, a, b, grad, activation, trans_a, trans_b)
    fn, m, k, n, a_stride, b_stride, grad_stride, elems = plan
    grad_a = a.new_empty(a.shape) if need_a else None
    grad_b = a.new_empty(b.shape) if need_b else None
    grad_bias = a.new_empty(n) if bias else None
    if workspace is None:
        if elems:
            workspace = a.new_empty(elems)
    else:
        elems = _room(workspace, a)
    code = _native.matmul_bias_act_grad(
        fn, grad.data_ptr(), a.data_ptr(), b.data_ptr(),
        _like(pre_activation, (m, n), dtype), _at(grad_a), _at(grad_b),
        _at(grad_bias), m, k, n, trans_a, trans_b, activation, a_stride,
        b_stride, 0, grad_stride, _at(workspace), elems, _stream())
    if code:
        capi.check(code)
    return grad_a, grad_b, grad_bias


def _gate_operand(gate, gate_rows, rows, channels, dtype):
    assert gate.shape == (-(-rows // gate_rows), channels) and \
        gate.dtype == dtype
    return gate.data_ptr(), _row_stride(gate)


def residual_norm(x, residual=None, gate=None, scale=None, post=NORM.NONE,
                  post_weight=None, post_bias=None, pre=NORM.NONE,
                  pre_weight=None, pre_bias=None, gate_op=None, gate_rows=1,
                  eps=1e-6, keep_sum=True, keep_stats=False, out=None):
    """snn_hip_residual_norm: sum = residual + scale * gate * post_norm(x) and
    normed = pre_norm(sum).  Returns (sum, normed, stats), None for what is not
    wanted or not there; `out` takes the sum and may be x or the residual."""
    rows, channels = shape = x.shape
    dtype = x.dtype
    gate_at, gate_stride = None, 0
    if gate is None:
        assert not gate_op, "an operation without a gate"
        gate_op = GATE.NONE
    else:
        if gate_op is None:
            gate_op = GATE.VALUE
        gate_at, gate_stride = _gate_operand(gate, gate_rows, rows, channels,
                                             dtype)
    if out is None:
        if keep_sum:
            out = _empty_like(x)
        sum_at = _at(out)
    else:
        sum_at = _like(out, shape, dtype)
    normed = _empty_like(x) if pre != NORM.NONE else None
    stats = (x.new_empty((rows, 4), dtype=torch.float32) if keep_stats
             else None)
    code = _native.residual_norm(
        _address("snn_hip_residual_norm" + _TYPES[dtype][0]), x.data_ptr(),
        _like(residual, shape, dtype), gate_at, _vector(scale, channels, dtype),
        _vector(post_weight, channels, dtype),
        _vector(post_bias, channels, dtype),
        _vector(pre_weight, channels, dtype),
        _vector(pre_bias, channels, dtype), sum_at, _at(normed), _at(stats),
        rows, channels, post, pre, gate_op, gate_rows, _row_stride(x),
        gate_stride, eps, _stream())
    if code:
        capi.check(code)
    return out, normed, stats


def residual_norm_grad(x, sum, stats, grad_sum=None, grad_normed=None,
                       gate=None, scale=None, post=NORM.NONE, post_weight=None,
                       post_bias=None, pre=NORM.NONE, pre_weight=None,
                       pre_bias=None, gate_op=None, gate_rows=1, eps=1e-6,
                       workspace=None):
    """snn_hip_residual_norm_grad: a dict of the gradients of x, residual and
    of those of gate, scale, post_weight, post_bias, pre_weight and pre_bias
    that are given."""
    rows, channels = shape = x.shape
    dtype = x.dtype
    got = {"x": _empty_like(x), "residual": _empty_like(x)}
    gate_at, gate_stride = None, 0
    if gate is None:
        assert not gate_op, "an operation without a gate"
        gate_op = GATE.NONE
    else:
        if gate_op is None:
            gate_op = GATE.VALUE
        gate_at, gate_stride = _gate_operand(gate, gate_rows, rows, channels,
                                             dtype)
        got["gate"] = x.new_empty(gate.shape)
    addresses = {}
    for name, t in (("scale", scale), ("post_weight", post_weight),
                    ("post_bias", post_bias), ("pre_weight", pre_weight),
                    ("pre_bias", pre_bias)):
        addresses[name] = _vector(t, channels, dtype)
        if t is not None and (grad_normed is not None or
                              not name.startswith("pre")):
            got[name] = x.new_empty(channels)
    if workspace is None:
        key = (rows, channels, gate_op, gate_rows, dtype)
        elems = _plans.get(key)
        if elems is None:
            elems = _keep(key, _workspace(
                "snn_hip_residual_norm_grad_workspace_size",
                ResidualNormParams(rows=rows, channels=channels, gate=gate_op,
                                   gate_rows=gate_rows), _TYPES[dtype][1]))
        workspace = x.new_empty(elems)
    else:
        elems = _room(workspace, x)
    code = _native.residual_norm_grad(
        _address("snn_hip_residual_norm_grad" + _TYPES[dtype][0]),
        x.data_ptr(), None, gate_at, addresses["scale"],
        addresses["post_weight"], addresses["post_bias"],
        addresses["pre_weight"], addresses["pre_bias"],
        _like(sum, shape, dtype), None,
        _like(stats, (rows, 4), torch.float32), _like(grad_sum, shape, dtype),
        _like(grad_normed, shape, dtype), got["x"].data_ptr(),
        got["residual"].data_ptr(), _at(got.get("gate")),
        _at(got.get("scale")), _at(got.get("post_weight")),
        _at(got.get("post_bias")), _at(got.get("pre_weight")),
        _at(got.get("pre_bias")), rows, channels, post, pre, gate_op, gate_rows,
        _row_stride(x), gate_stride, eps, workspace.data_ptr(),
        elems, _stream())
    if code:
        capi.check(code)
    return got


def _recurrence_operands(x, forget, input_gate, resets, lengths):
    """The common row stride, the workspace's elements and the optional
    operands' addresses."""
    shape, stride, dtype = x.shape, x.stride(), x.dtype
    key = (shape, stride, dtype)
    plan = _plans.get(key)
    if plan is None:
        batch, steps, channels = shape
        plan = _keep(key, (_step_stride(x), _workspace(
            "snn_hip_linear_recurrence_workspace_size",
            LinearRecurrenceParams(batch=batch, steps=steps,
                                   channels=channels), _TYPES[dtype][1])))
    for t in (forget, input_gate):
        assert t is None or (t.shape == shape and t.dtype == dtype and
                             (t.stride() == stride or
                              _step_stride(t) == plan[0]))
    return plan[0], plan[1], _like(resets, shape[:2], torch.uint8), \
        _vector(lengths, shape[0], torch.int32)


def linear_recurrence(x, forget, input_gate=None, resets=None, lengths=None,
                      initial_state=None, out=None, final_state=None,
                      workspace=None):
    """snn_hip_linear_recurrence over [batch, steps, channels] tensors; resets
    is a uint8 [batch, steps] tensor, lengths an int32 [batch] one, states are
    fp32 [batch, channels].  Returns (h, final state); final_state may be
    initial_state, which is then updated in place."""
    batch, steps, channels = shape = x.shape
    dtype = x.dtype
    stride, elems, resets_at, lengths_at = _recurrence_operands(
        x, forget, input_gate, resets, lengths)
    state = (batch, channels)
    if out is None:
        out = _empty_like(x)
        out_at = out.data_ptr()
    else:
        out_at = _like(out, shape, dtype)
    initial_at = _like(initial_state, state, torch.float32)
    if final_state is None:
        final_state = x.new_empty(state, dtype=torch.float32)
        final_at = final_state.data_ptr()
    elif final_state is initial_state:
        final_at = initial_at
    else:
        final_at = _like(final_state, state, torch.float32)
    if workspace is None:
        if elems:
            workspace = x.new_empty(elems)
    else:
        elems = _room(workspace, x)
    code = _native.linear_recurrence(
        _address("snn_hip_linear_recurrence" + _TYPES[dtype][0]), x.data_ptr(),
        forget.data_ptr(), _at(input_gate), resets_at, lengths_at,
        initial_at, out_at, final_at, batch, steps, channels, stride, 0,
        _at(workspace), elems, _stream())
    if code:
        capi.check(code)
    return out, final_state


def linear_recurrence_grad(grad, x, forget, h, input_gate=None, resets=None,
                           lengths=None, initial_state=None,
                           grad_final_state=None, out=None, workspace=None):
    """snn_hip_linear_recurrence_grad: a dict of the gradients of x, forget,
    input_gate (where it is given) and initial_state.  `out` is a [batch, steps,
    channels * n] tensor, or such a slice of a wider one, that takes those of x,
    forget and input_gate side by side: the gradient of a projection that they
    are slices of."""
    batch, steps, channels = shape = x.shape
    dtype = x.dtype
    stride, elems, resets_at, lengths_at = _recurrence_operands(
        x, forget, input_gate, resets, lengths)
    names = ["x", "forget"] + (["input_gate"] if input_gate is not None else [])
    if out is None:
        got = {name: _empty_like(x) for name in names}
        grad_stride = channels
    else:
        assert out.shape == (batch, steps, channels * len(names)) and \
            out.dtype == dtype
        got = {name: out[..., i * channels:(i + 1) * channels]
               for i, name in enumerate(names)}
        grad_stride = _step_stride(out)
    got["initial_state"] = x.new_empty((batch, channels), dtype=torch.float32)
    if workspace is None:
        if elems:
            workspace = x.new_empty(elems)
    else:
        elems = _room(workspace, x)
    state = (batch, channels)
    code = _native.linear_recurrence_grad(
        _address("snn_hip_linear_recurrence_grad" + _TYPES[dtype][0]),
        _like(grad, shape, dtype),
        _like(grad_final_state, state, torch.float32), x.data_ptr(),
        forget.data_ptr(), _at(input_gate), resets_at, lengths_at,
        _like(initial_state, state, torch.float32), _like(h, shape, dtype),
        got["x"].data_ptr(), got["forget"].data_ptr(),
        _at(got.get("input_gate")), got["initial_state"].data_ptr(), batch,
        steps, channels, stride, grad_stride, _at(workspace), elems, _stream())
    if code:
        capi.check(code)
    return got


# ---- a linear-attention block ------------------------------------------------
# Heads are a dimension of their own: [batch, steps, heads, channels] tensors whose
# heads follow one another, and whose rows of heads may be slices of wider ones.


def _gated_plan(key, a, w_gate, w_up, grad, activation, trans_b):
    dtype = a.dtype
    m, k = a.shape
    n = w_gate.shape[0] if trans_b else w_gate.shape[1]
    stride = _row_stride(w_gate)
    assert (w_gate.shape[1] if trans_b else w_gate.shape[0]) == k
    assert w_up.shape == w_gate.shape and _row_stride(w_up) == stride
    assert w_gate.dtype == dtype and w_up.dtype == dtype
    suffix, code = _TYPES[dtype]
    out_stride = 0
    if grad is not None:
        assert grad.shape == (m, n) and grad.dtype == dtype
        out_stride = _row_stride(grad)
    p = GatedMatmulParams(
        m=m, k=k, n=n, transpose_rhs=int(trans_b), activation=activation,
        lhs_stride=_row_stride(a), rhs_stride=stride, output_stride=out_stride)
    elems = _workspace("snn_hip_gated_matmul_workspace_size", p,
                       int(grad is not None), code)
    name = "snn_hip_gated_matmul" + ("_grad" if grad is not None else "")
    return _keep(key, (_address(name + suffix), m, k, n, p.lhs_stride, stride,
                       out_stride, elems))


def gated_matmul_plan(m, k, n, dtype, product=0, activation=ACTIVATION.SILU,
                      trans_b=False, aligned=True, workspace_elems=None,
                      **strides):
    """What a gated product runs on (snn_hip_gated_matmul_planned), a dict by the
    names of capi.MATMUL_PLAN; by default with the recommended workspace."""
    p = GatedMatmulParams(m=m, k=k, n=n, transpose_rhs=int(trans_b),
                          activation=activation, **strides)
    code = _TYPES[dtype][1]
    if workspace_elems is None:
        workspace_elems = _workspace("snn_hip_gated_matmul_workspace_size", p,
                                     int(product > 0), code)
    plan = capi.MatmulBiasActPlan()
    capi.check(capi.lib().snn_hip_gated_matmul_planned(
        ctypes.byref(p), product, code, int(aligned), workspace_elems,
        ctypes.byref(plan)))
    return {name: getattr(plan, name) for name in capi.MATMUL_PLAN}


def gated_matmul(a, w_gate, w_up, bias_gate=None, bias_up=None,
                 activation=ACTIVATION.SILU, trans_b=False,
                 keep_pre_activation=False, out=None, workspace=None):
    """snn_hip_gated_matmul: act(a w_gate + bias_gate) * (a w_up + bias_up).  With
    keep_pre_activation returns (output, gate, up), of which the gradients take
    the second and third: the two factors in front of the activation."""
    dtype = a.dtype
    key = ("gated", a.shape, a.stride(), w_gate.shape, w_gate.stride(),
           w_up.shape, w_up.stride(), dtype, w_gate.dtype, w_up.dtype,
           activation, trans_b)
    plan = _plans.get(key)
    if plan is None:
        plan = _gated_plan(key, a, w_gate, w_up, None, activation, trans_b)
    fn, m, k, n, a_stride, b_stride, _, elems = plan
    if out is None:
        out = a.new_empty((m, n))
        out_stride = n
    else:
        assert out.shape == (m, n) and out.dtype == dtype
        out_stride = _row_stride(out)
    gate = up = None
    if keep_pre_activation:
        gate, up = a.new_empty((m, n)), a.new_empty((m, n))
    if workspace is None:
        if elems:
            workspace = a.new_empty(elems)
    else:
        elems = _room(workspace, a)
    code = _native.gated_matmul(
        fn, a.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
        _vector(bias_gate, n, dtype), _vector(bias_up, n, dtype),
        out.data_ptr(), _at(gate), _at(up), m, k, n, trans_b, activation,
        a_stride, b_stride, out_stride, _at(workspace), elems, _stream())
    if code:
        capi.check(code)
    return (out, gate, up) if keep_pre_activation else out


def gated_matmul_grad(grad, a, w_gate, w_up, gate, up,
                      activation=ACTIVATION.SILU, trans_b=False, bias=True,
                      need_a=True, need_b=True, workspace=None):
    """snn_hip_gated_matmul_grad: the gradients of a, w_gate, w_up, bias_gate and
    bias_up, None for those that are not wanted."""
    dtype = a.dtype
    key = ("gated", a.shape, a.stride(), w_gate.shape, w_gate.stride(),
           w_up.shape, w_up.stride(), grad.shape, grad.stride(), dtype,
           w_gate.dtype, w_up.dtype, grad.dtype, activation, trans_b)
    plan = _plans.get(key)
    if plan is None:
        plan = _gated_plan(key, a, w_gate, w_up, grad, activation, trans_b)
    fn, m, k, n, a_stride, b_stride, grad_stride, elems = plan
    grad_a = a.new_empty(a.shape) if need_a else None
    grad_gate = a.new_empty(w_gate.shape) if need_b else None
    grad_up = a.new_empty(w_gate.shape) if need_b else None
    bias_gate = a.new_empty(n) if bias else None
    bias_up = a.new_empty(n) if bias else None
    if workspace is None:
        if elems:
            workspace = a.new_empty(elems)
    else:
        elems = _room(workspace, a)
    code = _native.gated_matmul_grad(
        fn, grad.data_ptr(), a.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
        _like(gate, (m, n), dtype), _like(up, (m, n), dtype), _at(grad_a),
        _at(grad_gate), _at(grad_up), _at(bias_gate), _at(bias_up), m, k, n,
        trans_b, activation, a_stride, b_stride, grad_stride, _at(workspace),
        elems, _stream())
    if code:
        capi.check(code)
    return grad_a, grad_gate, grad_up, bias_gate, bias_up


def _head_stride(t):
    """Elements from step to step of a [batch, steps, heads, channels] tensor."""
    batch, steps, heads, channels = t.shape
    outer, step, head, unit = t.stride()
    width = heads * channels
    assert unit == 1 or channels == 1, "channels are not contiguous"
    assert head == channels or heads == 1, "heads do not follow one another"
    if steps == 1:
        step = outer if batch > 1 else width
    else:
        assert batch == 1 or outer == steps * step, \
            "sequences do not follow one another"
    assert step >= width
    return step


def rotary_frequencies(turned, base=10000.0, scaling=ROTARY_SCALING.NONE,
                       factor=1.0, context=0.0, low=1.0, high=32.0,
                       device="cuda"):
    """snn_hip_rotary_frequencies: the float64 table that `rotary` takes, turns
    from one position to the next of turned / 2 pairs, on `device`."""
    table = torch.empty(max(turned, 0) // 2, dtype=torch.float64)
    capi.check(capi.lib().snn_hip_rotary_frequencies(
        turned, base, scaling, factor, context, low, high, table.data_ptr()))
    return table.to(device)


def rotary(x, frequencies, positions=None, layout=ROTARY.HALVES, magnitude=1.0,
           inverse=False, out=None):
    """snn_hip_rotary over a [batch, steps, heads, channels] tensor, of whose
    channels the first 2 * len(frequencies) are turned.  positions: None (a token's
    step), an int32 [batch] tensor (of step 0) or [batch, steps] one.  `out` may be
    x.  The gradient is the call with `inverse` on the output's gradient."""
    batch, steps, heads, channels = shape = x.shape
    dtype = x.dtype
    assert frequencies.dtype is torch.float64 and frequencies.dim() == 1 and \
        frequencies.is_contiguous() and frequencies.is_cuda == x.is_cuda
    kind = ROTARY_POSITIONS.NONE
    if positions is not None:
        kind = ROTARY_POSITIONS.FIRST
        if positions.dim() != 1:
            kind = ROTARY_POSITIONS.EACH
        assert positions.dim() in (1, 2) and \
            positions.shape == shape[:positions.dim()]
        assert positions.dtype is torch.int32 and positions.is_contiguous() and \
            positions.is_cuda == x.is_cuda
    stride = _head_stride(x)
    if out is None:
        out = x.new_empty(shape)
        out_stride = heads * channels
    elif out is x:
        out_stride = stride
    else:
        assert out.shape == shape and out.dtype == dtype
        out_stride = _head_stride(out)
    code = _native.rotary(
        _address("snn_hip_rotary" + _TYPES[dtype][0]), x.data_ptr(),
        frequencies.data_ptr(), _at(positions), out.data_ptr(), batch, steps,
        heads, channels, 2 * frequencies.shape[0], layout, kind, inverse, stride,
        out_stride, magnitude, _stream())
    if code:
        capi.check(code)
    return out


def _attention_operands(q, k, v, decay, resets, lengths, grad):
    """Sizes, strides, the workspace's elements and the small operands'
    addresses."""
    key = ("attention", q.shape, q.stride(), k.shape, k.stride(), v.shape,
           v.stride(), q.dtype, k.dtype, v.dtype, grad)
    plan = _plans.get(key)
    if plan is None:
        batch, steps, key_heads, keys = q.shape
        heads, values = v.shape[2:]
        assert k.shape == q.shape and v.shape[:2] == q.shape[:2]
        assert k.dtype == q.dtype and v.dtype == q.dtype
        strides = _head_stride(q), _head_stride(k), _head_stride(v)
        params = LinearAttentionParams(
            batch=batch, steps=steps, heads=heads, key_heads=key_heads,
            keys=keys, values=values)
        plan = _keep(key, (
            (batch, steps, heads, key_heads, keys, values) + strides,
            _workspace("snn_hip_linear_attention_workspace_size", params,
                       int(grad), _TYPES[q.dtype][1])))
    sizes, elems = plan
    return sizes, elems, _vector(decay, sizes[2], torch.float32), \
        _like(resets, sizes[:2], torch.uint8), \
        _vector(lengths, sizes[0], torch.int32)


def linear_attention_plan(batch, steps, heads, key_heads, keys, values, dtype,
                          grad=False, aligned=True, workspace_elems=None,
                          **strides):
    """How a call goes over its sequences (snn_hip_linear_attention_planned): pieces,
    steps of a piece, and a list of launches, dicts by the names of
    capi.LINEAR_ATTENTION_LAUNCH; by default with the recommended workspace."""
    p = LinearAttentionParams(batch=batch, steps=steps, heads=heads,
                              key_heads=key_heads, keys=keys, values=values,
                              **strides)
    code = _TYPES[dtype][1]
    if workspace_elems is None:
        workspace_elems = _workspace("snn_hip_linear_attention_workspace_size", p,
                                     int(grad), code)
    plan = capi.LinearAttentionPlan()
    capi.check(capi.lib().snn_hip_linear_attention_planned(
        ctypes.byref(p), int(grad), code, int(aligned), workspace_elems,
        ctypes.byref(plan)))
    return plan.pieces, plan.piece_steps, [
        {name: getattr(l, name) for name in capi.LINEAR_ATTENTION_LAUNCH}
        for l in plan.launch[:plan.launches]]


def linear_attention(q, k, v, decay, resets=None, lengths=None,
                     initial_state=None, scale=1.0, out=None, final_state=None,
                     workspace=None):
    """snn_hip_linear_attention: q and k are [batch, steps, key_heads, keys], v is
    [batch, steps, heads, values]; decay holds the logarithms of the heads' decays
    (fp32), resets is a uint8 [batch, steps] tensor, lengths an int32 [batch] one,
    states are fp32 [batch, heads, keys, values].  Returns (output, final state);
    final_state may be initial_state, which is then updated in place."""
    sizes, elems, decay_at, resets_at, lengths_at = _attention_operands(
        q, k, v, decay, resets, lengths, False)
    batch, steps, heads, _, keys, values = sizes[:6]
    dtype = q.dtype
    if out is None:
        out = v.new_empty(v.shape)
        out_at = out.data_ptr()
    else:
        out_at = _like(out, v.shape, dtype)
    state = (batch, heads, keys, values)
    initial_at = _like(initial_state, state, torch.float32)
    if final_state is None:
        final_state = q.new_empty(state, dtype=torch.float32)
        final_at = final_state.data_ptr()
    elif final_state is initial_state:
        final_at = initial_at
    else:
        final_at = _like(final_state, state, torch.float32)
    if workspace is None:
        if elems:
            workspace = q.new_empty(elems)
    else:
        elems = _room(workspace, q)
    code = _native.linear_attention(
        _address("snn_hip_linear_attention" + _TYPES[dtype][0]), q.data_ptr(),
        k.data_ptr(), v.data_ptr(), decay_at, resets_at, lengths_at, initial_at,
        out_at, final_at, *sizes, 0, 0, 0, scale, _at(workspace), elems,
        _stream())
    if code:
        capi.check(code)
    return out, final_state


def linear_attention_grad(grad, q, k, v, decay, resets=None, lengths=None,
                          initial_state=None, grad_final_state=None, scale=1.0,
                          out=None, workspace=None):
    """snn_hip_linear_attention_grad: a dict of the gradients of q, k, v and
    initial_state.  `out` is a [batch, steps, 2 * key_heads * keys + heads * values]
    tensor, or such a slice of a wider one, that takes those of q, k and v side by
    side: the gradient of a projection that they are slices of."""
    sizes, elems, decay_at, resets_at, lengths_at = _attention_operands(
        q, k, v, decay, resets, lengths, True)
    batch, steps, heads, key_heads, keys, values = sizes[:6]
    dtype = q.dtype
    if out is None:
        got = {"q": q.new_empty(q.shape), "k": k.new_empty(k.shape),
               "v": v.new_empty(v.shape)}
        strides = 0, 0, 0
    else:
        n, m = key_heads * keys, heads * values
        assert out.shape == (batch, steps, 2 * n + m) and out.dtype == dtype
        got = {"q": out[..., :n].unflatten(2, (key_heads, keys)),
               "k": out[..., n:2 * n].unflatten(2, (key_heads, keys)),
               "v": out[..., 2 * n:].unflatten(2, (heads, values))}
        strides = (_step_stride(out),) * 3
    state = (batch, heads, keys, values)
    got["initial_state"] = q.new_empty(state, dtype=torch.float32)
    if workspace is None:
        if elems:
            workspace = q.new_empty(elems)
    else:
        elems = _room(workspace, q)
    code = _native.linear_attention_grad(
        _address("snn_hip_linear_attention_grad" + _TYPES[dtype][0]),
        _like(grad, v.shape, dtype),
        _like(grad_final_state, state, torch.float32), q.data_ptr(),
        k.data_ptr(), v.data_ptr(), decay_at, resets_at, lengths_at,
        _like(initial_state, state, torch.float32), got["q"].data_ptr(),
        got["k"].data_ptr(), got["v"].data_ptr(),
        got["initial_state"].data_ptr(), *sizes, *strides, scale,
        _at(workspace), elems, _stream())
    if code:
        capi.check(code)
    return got


__all__ = [
    "ACTIVATION", "ALGO", "BINARY_OP", "DIRECTION", "GATE", "NORM",
    "POINTWISE_OP", "POOL_OP", "ROTARY", "ROTARY_POSITIONS", "ROTARY_SCALING",
    "STATUS",
    "ConvParams", "DepthwiseParams", "PoolParams", "add_padding_to",
    "binaryop", "binaryop_raw", "calculate_padding", "conv2d",
    "conv2d_bias_act", "conv2d_prepare_filter", "conv2d_prepared",
    "conv2d_raw", "conv_flops", "conv_params", "conv_sizes",
    "default_algorithm",
    "depthwise_conv2d", "depthwise_params", "depthwise_sizes",
    "gated_matmul", "gated_matmul_grad", "gated_matmul_plan", "linear_attention",
    "linear_attention_grad", "linear_attention_plan",
    "linear_recurrence", "linear_recurrence_grad", "matmul", "matmul_bias_act",
    "matmul_bias_act_grad", "matmul_plan",
    "pointwise_forward", "pointwise_grad", "pool_params", "pooling_avg_grad",
    "pooling_forward", "pooling_max_grad", "residual_norm",
    "residual_norm_grad", "rotary", "rotary_frequencies", "workspace_size",
]


class kernel_timing:
    """Context manager around snn_hip_kernel_timing_*: times the dominant
    kernel of every convolution launched inside it with HIP events on the
    launch stream.  After exit `.total_ms` and `.kernels` hold the result."""

    def __enter__(self):
        capi.check(capi.lib().snn_hip_kernel_timing_enable(1))
        self.total_ms = 0.0
        self.kernels = 0
        return self

    def __exit__(self, *exc):
        lib = capi.lib()
        capi.check(lib.snn_hip_kernel_timing_enable(0))
        ms = ctypes.c_double(0.0)
        n = ctypes.c_int(0)
        capi.check(lib.snn_hip_kernel_timing_read(ctypes.byref(ms),
                                                  ctypes.byref(n)))
        self.total_ms = ms.value
        self.kernels = n.value
        return False
