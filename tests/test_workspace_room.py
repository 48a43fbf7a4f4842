"""What the Python calls tell an entry point about a caller's workspace: the
elements of the operands' type that its memory holds, whatever type it has.  The
calls are taken down instead of made."""
import pytest
import torch

from portdnn_amd import capi, ops
from portdnn_amd.ops import ACTIVATION, ALGO, DIRECTION, NORM

TYPES = [torch.float32, torch.float16, torch.bfloat16]


class _Taken(Exception):
    pass


@pytest.fixture
def room(monkeypatch):
    """Makes a call with a workspace and returns the count that was passed on."""
    monkeypatch.setattr(ops, "_stream", lambda: 0)

    def elements(args, workspace):
        address = workspace.data_ptr()
        at = [i for i, a in enumerate(args)
              if getattr(a, "value", a) == address]
        raise _Taken(args[at[-1] + 1])

    def run(call, workspace):
        library = capi.lib()

        class Calls:
            def __getattr__(self, name):
                return lambda *args: elements(args, workspace)

        class Library:
            def __getattr__(self, name):
                if name.endswith("workspace_size"):
                    return getattr(library, name)
                return lambda *args: elements(args, workspace)

        with monkeypatch.context() as m:
            m.setattr(ops, "_native", Calls())
            m.setattr(ops, "_address", lambda name: 0)
            m.setattr(capi, "lib", Library)
            m.setattr(ops, "_plans", {})
            with pytest.raises(_Taken) as taken:
                call(workspace)
        return taken.value.args[0]
    return run


def _sequence_calls(dtype):
    a, b = torch.zeros(4, 8, dtype=dtype), torch.zeros(8, 6, dtype=dtype)
    z = torch.zeros(4, 6, dtype=dtype)
    x = torch.zeros(2, 3, 8, dtype=dtype)
    stats = torch.zeros(4, 4)
    return {
        "matmul": lambda w: ops.matmul_bias_act(a, b, workspace=w),
        "matmul_grad": lambda w: ops.matmul_bias_act_grad(
            z, a, b, z, activation=ACTIVATION.GELU, workspace=w),
        "norm_grad": lambda w: ops.residual_norm_grad(
            a, a, stats, grad_normed=a, pre=NORM.RMS, workspace=w),
        "recurrence": lambda w: ops.linear_recurrence(x, x, workspace=w),
        "recurrence_grad": lambda w: ops.linear_recurrence_grad(
            x, x, x, x, workspace=w),
    }


def _convolution_calls(dtype):
    p = ops.conv_params(1, 8, 8, 4, 4, 3, 1, True)
    x, f, y = (torch.zeros(n, dtype=dtype)
               for n in ops.conv_sizes(p, DIRECTION.FORWARD))
    calls = {
        "conv2d_raw": lambda w: ops.conv2d_raw(
            x, f, y, p, DIRECTION.FORWARD, ALGO.TILED, w),
        "conv2d": lambda w: ops.conv2d(x, f, p, DIRECTION.FORWARD, ALGO.TILED, w),
        "conv2d_bound": lambda w: ops.conv2d_bound(
            x, f, y, p, DIRECTION.FORWARD, ALGO.TILED, w)(),
    }
    if dtype == torch.float32:
        calls.update({
            "prepared_bound": lambda w: ops.conv2d_prepared_bound(
                x, f, y, p, DIRECTION.FORWARD, ALGO.WINOGRAD, w)(),
            "prepare_filter": lambda w: ops.conv2d_prepare_filter(
                f, p, DIRECTION.FORWARD, ALGO.WINOGRAD, w),
            "prepared": lambda w: ops.conv2d_prepared(
                x, f, p, DIRECTION.FORWARD, ALGO.WINOGRAD, w),
            "deterministic": lambda w: ops.conv2d_deterministic(
                x, f, p, DIRECTION.FORWARD, ALGO.TILED, w),
            "bias_act": lambda w: ops.conv2d_bias_act(
                x, f, torch.zeros(4), p, ALGO.TILED, workspace=w),
        })
    return calls


CASES = ([(_sequence_calls, d, n) for d in TYPES
          for n in ("matmul", "matmul_grad", "norm_grad", "recurrence",
                    "recurrence_grad")] +
         [(_convolution_calls, d, n) for d in TYPES[:2]
          for n in ("conv2d_raw", "conv2d", "conv2d_bound")] +
         [(_convolution_calls, torch.float32, n)
          for n in ("prepared_bound", "prepare_filter", "prepared",
                    "deterministic", "bias_act")])


@pytest.mark.parametrize("calls,dtype,name", CASES)
def test_a_workspace_counts_by_its_bytes(room, calls, dtype, name):
    call = calls(dtype)[name]
    size = torch.zeros((), dtype=dtype).element_size()
    for kind, numel in ((dtype, 640), (torch.uint8, 1000), (torch.uint8, 1003),
                        (torch.float64, 40), (torch.int32, 100)):
        workspace = torch.zeros(numel, dtype=kind)
        assert room(call, workspace) == numel * workspace.element_size() // size


@pytest.mark.parametrize("calls,dtype,name", CASES)
def test_a_workspace_is_contiguous(monkeypatch, calls, dtype, name):
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    for workspace in (torch.zeros(1, dtype=dtype).expand(1 << 20),
                      torch.zeros(64, dtype=dtype)[::2]):
        with pytest.raises(AssertionError):
            calls(dtype)[name](workspace)
