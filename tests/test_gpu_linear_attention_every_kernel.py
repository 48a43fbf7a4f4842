"""Calls that reach every kernel of linear attention over blocks, with resets and
lengths, against 64 bits."""
import pytest
import torch

import attention_reference as plain
import sequence_reference as ref
from attention_kernel_cases import CASES
from portdnn_amd import ops
from test_attention_plans import TYPES, kernels_of
from test_gpu_linear_attention import _cuda, _make, _wide

pytestmark = pytest.mark.gpu


def _check(got, pair, operations, what):
    ref.check(got, tuple(x.cpu() for x in pair), operations, what)


@pytest.mark.parametrize("at", range(len(CASES)))
def test_case(at):
    c = CASES[at]
    lengths = None
    if c.batch > 1:  # (one of them whole)
        g = torch.Generator().manual_seed(at)
        lengths = torch.randint(c.steps + 1, (c.batch,), generator=g).tolist()
        lengths[c.batch // 2] = c.steps
    for dtype in TYPES[c.type]:
        assert kernels_of(c, dtype)
        t, (do, ds) = _make(tuple(c[2:]), dtype, resets=True, lengths=lengths,
                            seed=at)
        most, scale = max(c.keys, c.values), c.keys ** -0.5
        of_outputs = plain.operations(most, dtype)
        of_states = plain.state_operations(most, dtype)
        gpu = _cuda(t)
        # (the references' steps on the GPU as well)
        with torch.device("cuda"):
            if c.grad:
                got = ops.linear_attention_grad(
                    do.cuda(), scale=scale, grad_final_state=ds.cuda(), **gpu)
                want = plain.attention_grad(
                    do.cuda().double(), scale=scale, dtype=dtype,
                    grad_final_state=ds.cuda().double(), **_wide(gpu))
                for name, pair in want.items():
                    _check(got[name], pair, of_states if name == "initial_state"
                           else of_outputs, "%s %s d%s" % (c, dtype, name))
            else:
                o, last = ops.linear_attention(scale=scale, **gpu)
                want = plain.attention(scale=scale, dtype=dtype, **_wide(gpu))
                _check(o, want[0], of_outputs, "%s %s" % (c, dtype))
                _check(last, want[1], of_states, "%s %s state" % (c, dtype))
