"""ctypes binding of the libsnn_hip.so C ABI (include/snn_hip.h).

Pointers are raw device addresses (e.g. ``torch.Tensor.data_ptr()``); the
stream argument is a ``hipStream_t`` handle as an integer (0 = default).
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_HERE, "libsnn_hip.so")


class SnnHipError(RuntimeError):
    pass


class STATUS:
    OK = 0
    INVALID_ALGORITHM = 1
    INDEX_EXCEEDED = 2
    INSUFFICIENT_WORKSPACE = 3
    ALLOCATION_PROBLEM = 4
    INVALID_PARAMETER = 5
    DEVICE_ERROR = 6


class ALGO:
    NOT_SUPPORTED = 0
    DIRECT = 1
    TILED = 2
    IM2COL = 3
    WINOGRAD = 4
    WINOGRAD_LARGE = 5
    MATMUL = 6


class DIRECTION:
    FORWARD = 0
    INPUT_BACKPROP = 1
    FILTER_BACKPROP = 2


class DTYPE:
    F32 = 0
    F16 = 1
    BF16 = 2


class ACTIVATION:
    NONE = 0
    RELU = 1
    GELU = 2
    GELU_TANH = 3
    SILU = 4


class NORM:
    NONE = 0
    RMS = 1
    LAYER = 2


class GATE:
    NONE = 0
    VALUE = 1
    SIGMOID = 2
    SILU = 3


class POOL_OP:
    MAX = 0
    MAX_WITH_NAN = 1
    AVERAGE = 2


class POINTWISE_OP:
    RELU = 0
    TANH = 1
    EXP = 2
    LOG = 3
    FLOOR = 4
    SQRT = 5


class BINARY_OP:
    ADD = 0
    SUB = 1
    MUL = 2
    DIV = 3


def _struct(name, fields, defaults, types={}):
    class S(ctypes.Structure):
        _fields_ = [(f, types.get(f, ctypes.c_int)) for f in fields]

        def __init__(self, **kw):
            super().__init__()
            for f in fields:
                v = kw.pop(f, defaults.get(f, 0))
                # (ctypes cuts numbers off that a field does not hold)
                if f not in types and not -1 << 31 <= v < 1 << 31:
                    raise OverflowError("%s: %d is beyond 31 bits" % (f, v))
                setattr(self, f, v)
            if kw:
                raise TypeError("unknown fields: %s" % sorted(kw))

        def __repr__(self):
            return name + "(" + ", ".join(
                "%s=%s" % (f, getattr(self, f)) for f in fields) + ")"
    S.__name__ = name
    return S


ConvParams = _struct(
    "ConvParams",
    ["channels", "features", "batch", "in_rows", "in_cols", "window_rows",
     "window_cols", "stride_rows", "stride_cols", "out_rows", "out_cols",
     "pad_rows", "pad_cols", "dilation_rows", "dilation_cols", "groups",
     "input_format", "filter_format", "group_format"],
    {"dilation_rows": 1, "dilation_cols": 1, "groups": 1})

DepthwiseParams = _struct(
    "DepthwiseParams",
    ["channels", "channel_multiplier", "batch", "in_rows", "in_cols",
     "window_rows", "window_cols", "stride_rows", "stride_cols", "out_rows",
     "out_cols", "pad_rows", "pad_cols", "input_format", "filter_format"], {})

PoolParams = _struct(
    "PoolParams",
    ["in_rows", "in_cols", "out_rows", "out_cols", "window_rows",
     "window_cols", "stride_rows", "stride_cols", "batch", "channels",
     "pad_rows", "pad_cols", "input_format"], {})

MatmulBiasActParams = _struct(
    "MatmulBiasActParams",
    ["m", "k", "n", "transpose_lhs", "transpose_rhs", "activation",
     "lhs_stride", "rhs_stride", "residual_stride", "output_stride"], {})

MATMUL_PLAN = ["tile_rows", "tile_cols", "shared", "any_address", "pair",
               "first_inner", "second_inner", "first_copied", "second_copied",
               "shares"]
MatmulBiasActPlan = _struct("MatmulBiasActPlan", MATMUL_PLAN, {})

ResidualNormParams = _struct(
    "ResidualNormParams",
    ["rows", "channels", "post_norm", "pre_norm", "gate", "gate_rows",
     "x_stride", "gate_stride", "epsilon"],
    {"gate_rows": 1}, {"epsilon": ctypes.c_float})

_NORM_TENSORS = ["x", "residual", "gate", "scale", "post_weight", "post_bias",
                 "pre_weight", "pre_bias", "sum", "normed", "stats"]
ResidualNormTensors = _struct(
    "ResidualNormTensors", _NORM_TENSORS, {f: None for f in _NORM_TENSORS},
    {f: ctypes.c_void_p for f in _NORM_TENSORS})

_NORM_GRADIENTS = ["grad_sum", "grad_normed", "grad_x", "grad_residual",
                   "grad_gate", "grad_scale", "grad_post_weight",
                   "grad_post_bias", "grad_pre_weight", "grad_pre_bias"]
ResidualNormGradients = _struct(
    "ResidualNormGradients", _NORM_GRADIENTS,
    {f: None for f in _NORM_GRADIENTS},
    {f: ctypes.c_void_p for f in _NORM_GRADIENTS})

LinearRecurrenceParams = _struct(
    "LinearRecurrenceParams",
    ["batch", "steps", "channels", "row_stride", "grad_row_stride"], {})

_P = ctypes.c_void_p
_SZ = ctypes.c_size_t
_I = ctypes.c_int

# name -> argtypes; every symbol include/snn_hip.h declares.
SIGNATURES = {
    "snn_hip_version": [],
    "snn_hip_status_string": [_I],
    "snn_hip_last_error": [],
    "snn_hip_temporary_memory_stats": [
        ctypes.POINTER(ctypes.c_ulonglong), ctypes.POINTER(ctypes.c_ulonglong),
        _I],
    "snn_hip_kernel_timing_enable": [_I],
    "snn_hip_kernel_timing_read": [ctypes.POINTER(ctypes.c_double),
                                   ctypes.POINTER(ctypes.c_int)],
    "snn_hip_conv2d_halves_tile": [_P, _I, _I, ctypes.POINTER(_I),
                                   ctypes.POINTER(_I)],
    "snn_hip_conv2d_filter_halves_partials": [_P, _I, ctypes.POINTER(_I)],
    "snn_hip_conv2d_gather_tile": [_P, _I, _I, ctypes.POINTER(_I),
                                   ctypes.POINTER(_I), ctypes.POINTER(_I)],
    "snn_hip_conv2d_lds_form_f16": [_P, _I, ctypes.POINTER(_I)],
    "snn_hip_conv2d_forward_f32": [_P, _P, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_input_backprop_f32": [_P, _P, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_filter_backprop_f32": [_P, _P, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_forward_f16": [_P, _P, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_input_backprop_f16": [_P, _P, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_filter_backprop_f16": [_P, _P, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_forward_bias_act_f32": [_P, _P, _P, _P, _P, _I, _I, _P,
                                            _SZ, _P],
    "snn_hip_conv2d_deterministic_f32": [_I, _P, _P, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_prepare_filter_f32": [_I, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_prepared_f32": [_I, _P, _P, _P, _P, _I, _P, _SZ, _P],
    "snn_hip_conv2d_workspace_size": [_P, _I, _I, ctypes.POINTER(_SZ),
                                      ctypes.POINTER(_SZ)],
    "snn_hip_conv2d_algorithm_supports": [_P, _I, _I],
    "snn_hip_conv2d_default_algorithm": [_P, _I],
    "snn_hip_conv2d_default_algorithm_for": [_P, _I, _I],
    "snn_hip_conv2d_workspace_size_for": [_P, _I, _I, _I, ctypes.POINTER(_SZ),
                                          ctypes.POINTER(_SZ)],
    "snn_hip_depthwise_conv2d_forward_f32": [_P, _P, _P, _P, _P],
    "snn_hip_depthwise_conv2d_input_backprop_f32": [_P, _P, _P, _P, _P],
    "snn_hip_depthwise_conv2d_filter_backprop_f32": [_P, _P, _P, _P, _P],
    "snn_hip_depthwise_conv2d_filter_backprop_noalloc_f32": [_P, _P, _P, _P,
                                                             _P],
    "snn_hip_depthwise_conv2d_forward_f16": [_P, _P, _P, _P, _P],
    "snn_hip_depthwise_conv2d_input_backprop_f16": [_P, _P, _P, _P, _P],
    "snn_hip_depthwise_conv2d_filter_backprop_f16": [_P, _P, _P, _P, _P],
    "snn_hip_pooling_forward_f32": [_P, _P, _P, _I, _P],
    "snn_hip_pooling_forward_f16": [_P, _P, _P, _I, _P],
    "snn_hip_pooling_max_grad_f32": [_P, _P, _P, _P, _P, _I, _P],
    "snn_hip_pooling_avg_grad_f32": [_P, _P, _P, _P],
    "snn_hip_pooling_max_grad_f16": [_P, _P, _P, _P, _P, _I, _P],
    "snn_hip_pooling_avg_grad_f16": [_P, _P, _P, _P],
    "snn_hip_matmul_f32": [_P, _P, _P, _I, _I, _I, _I, _I, _I,
                           ctypes.c_float, _P],
    "snn_hip_matmul_f16": [_P, _P, _P, _I, _I, _I, _I, _I, _I,
                           ctypes.c_float, _P],
    "snn_hip_scale_blend_f32": [_P, _P, ctypes.c_float, ctypes.c_float, _SZ,
                                _P],
    "snn_hip_pointwise_forward_f32": [_P, _P, _SZ, _I, _P],
    "snn_hip_pointwise_forward_f16": [_P, _P, _SZ, _I, _P],
    "snn_hip_pointwise_grad_f32": [_P, _P, _P, _SZ, _I, _P],
    "snn_hip_pointwise_grad_f16": [_P, _P, _P, _SZ, _I, _P],
    "snn_hip_binaryop_f32": [_P, _P, _P, ctypes.POINTER(_I), _I,
                             ctypes.POINTER(_I), _I, _I, _P],
    "snn_hip_binaryop_f16": [_P, _P, _P, ctypes.POINTER(_I), _I,
                             ctypes.POINTER(_I), _I, _I, _P],
    "snn_hip_matmul_bias_act_workspace_size": [
        _P, _I, _I, ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)],
    "snn_hip_matmul_bias_act_planned": [_P, _I, _I, _I, _SZ, _P],
    "snn_hip_residual_norm_grad_workspace_size": [
        _P, _I, ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)],
    "snn_hip_linear_recurrence_workspace_size": [
        _P, _I, ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)],
}
for _type in ("f32", "f16", "bf16"):
    SIGNATURES["snn_hip_matmul_bias_act_" + _type] = [_P] * 8 + [_SZ, _P]
    SIGNATURES["snn_hip_matmul_bias_act_grad_" + _type] = [_P] * 9 + [_SZ, _P]
    SIGNATURES["snn_hip_residual_norm_" + _type] = [_P] * 3
    SIGNATURES["snn_hip_residual_norm_grad_" + _type] = [_P] * 4 + [_SZ, _P]
    SIGNATURES["snn_hip_linear_recurrence_" + _type] = [_P] * 10 + [_SZ, _P]
    SIGNATURES["snn_hip_linear_recurrence_grad_" + _type] = (
        [_P] * 15 + [_SZ, _P])

_lib = None


def lib_path():
    return _LIB_PATH


def lib():
    """Loads libsnn_hip.so; raises if it has not been built (no fallback)."""
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            raise SnnHipError(
                "libsnn_hip.so is missing: build it with "
                "`python -m portdnn_amd.build` (there is no CPU fallback)")
        # torch bundles its own libamdhip64; load it first so that this
        # library binds to the same HIP runtime the tensors live in (two
        # runtimes in one process do not see each other's devices).
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        L = ctypes.CDLL(_LIB_PATH)
        for name, argtypes in SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = argtypes
            fn.restype = _I
        L.snn_hip_status_string.restype = ctypes.c_char_p
        L.snn_hip_last_error.restype = ctypes.c_char_p
        _lib = L
    return _lib


def status_string(code):
    return lib().snn_hip_status_string(int(code)).decode()


def check(code):
    """Raises SnnHipError for a non-OK status."""
    if code != STATUS.OK:
        raise SnnHipError("%s (%d) %s" % (
            status_string(code), code, lib().snn_hip_last_error().decode()))
    return code
