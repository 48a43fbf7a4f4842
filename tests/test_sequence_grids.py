"""Work-groups that no grid holds: decided on the host.  Nothing is launched."""
import ctypes

import pytest

from portdnn_amd import capi
from portdnn_amd.capi import (DTYPE, GATE, STATUS, LinearRecurrenceParams,
                              MatmulBiasActParams, ResidualNormParams)

FAKE = 0x1000  # never dereferenced
TYPES = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("suffix", TYPES)
def test_products_of_more_tiles_than_a_grid_holds(suffix):
    p = MatmulBiasActParams(m=1 << 21, k=64, n=1 << 20)
    fn = getattr(capi.lib(), "snn_hip_matmul_bias_act_" + suffix)
    for n in (1 << 20, (1 << 20) + 1):
        p.n = n
        assert fn(FAKE, FAKE, None, None, FAKE, None, ctypes.byref(p), None, 0,
                  None) == STATUS.INDEX_EXCEEDED


@pytest.mark.parametrize("suffix", TYPES)
def test_sequences_are_divided_as_far_as_a_grid_holds_the_pieces(suffix):
    """128 steps to a piece of 1024 lanes, 144 to one of 768."""
    query = capi.lib().snn_hip_linear_recurrence_workspace_size
    required, recommended = ctypes.c_size_t(), ctypes.c_size_t()

    def elems(steps, batch=1):
        p = LinearRecurrenceParams(batch=batch, steps=steps, channels=8)
        assert query(ctypes.byref(p), getattr(DTYPE, suffix.upper()),
                     ctypes.byref(required), ctypes.byref(recommended)) == 0
        return recommended.value

    limit = (1 << 32) - 1
    assert elems(limit // 1024 * 128) > 0
    assert elems(limit // 768 * 144) > 0
    assert elems(limit // 768 * 144 + 1) == 0
    assert elems(limit // 768 // 100 * 144, batch=100) > 0
    assert elems(limit // 768 // 100 * 144 + 144, batch=100) == 0


@pytest.mark.parametrize("suffix", TYPES)
@pytest.mark.parametrize("gate_rows", [0, 2, 3, 1 << 20, (1 << 31) - 1])
def test_sums_over_as_many_rows_as_there_may_be(suffix, gate_rows):
    """Of at most 2048 work-groups, and as many of a shared gate's rows, per channel."""
    query = capi.lib().snn_hip_residual_norm_grad_workspace_size
    required, recommended = ctypes.c_size_t(), ctypes.c_size_t()
    for rows in ((1 << 30) + 1, (1 << 31) - 1):
        p = ResidualNormParams(
            rows=rows, channels=2, gate=GATE.VALUE if gate_rows else GATE.NONE,
            gate_rows=max(1, gate_rows))
        assert query(ctypes.byref(p), getattr(DTYPE, suffix.upper()),
                     ctypes.byref(required), ctypes.byref(recommended)) == 0
        size = 4 if suffix == "f32" else 2
        # (five sums, and runs of a gate's rows: no more than two for each group)
        assert 0 < required.value * size <= (5 + 2) * 2048 * 2 * 4


@pytest.mark.parametrize("suffix", TYPES)
def test_steps_and_channels_that_cannot_be_counted_on(suffix):
    """A walk counts some steps, and a work-group some channels, beyond the last."""
    query = capi.lib().snn_hip_linear_recurrence_workspace_size
    n = ctypes.c_size_t()
    most = (1 << 31) - 1
    for steps, channels, want in ((most - 64, 1, STATUS.OK),
                                  (most - 63, 1, STATUS.INDEX_EXCEEDED),
                                  (most, 1, STATUS.INDEX_EXCEEDED),
                                  (1, most - 1024, STATUS.OK),
                                  (1, most - 1023, STATUS.INDEX_EXCEEDED),
                                  (1, most, STATUS.INDEX_EXCEEDED)):
        p = LinearRecurrenceParams(batch=1, steps=steps, channels=channels)
        assert query(ctypes.byref(p), getattr(DTYPE, suffix.upper()),
                     ctypes.byref(n), ctypes.byref(n)) == want
        if want != STATUS.OK:
            name = "snn_hip_linear_recurrence"
            assert getattr(capi.lib(), "%s_%s" % (name, suffix))(
                FAKE, FAKE, None, None, None, None, FAKE, None, ctypes.byref(p),
                None, 0, None) == want
            assert getattr(capi.lib(), "%s_grad_%s" % (name, suffix))(
                FAKE, None, FAKE, FAKE, None, None, None, None, FAKE, FAKE,
                FAKE, None, None, ctypes.byref(p), None, 0, None) == want
