"""The choice among the kernels of matmul_bias_act: that the products of
matmul_kernel_cases reach all of them.  Decided on the host."""
import ctypes

import pytest
import torch

from matmul_kernel_cases import CASES
from portdnn_amd import capi, ops
from portdnn_amd.capi import ACTIVATION, DTYPE, STATUS, MatmulBiasActParams

TYPES = {"f32": [torch.float32], "16": [torch.float16, torch.bfloat16]}
NONE, FIRST, SECOND, BOTH = (0, 0), (1, 0), (0, 1), (1, 1)
ANY, ALL = {NONE}, {NONE, FIRST, SECOND, BOTH}
# kernel: copies in front of a whole reduction, and of a shared one.  (Operands by
# way of registers are not copied.  What is not here no size was found to ask for.)
REACHED = {
    ("f32", (16, 16, 1, 0, 0)): (ALL, ALL),
    ("f32", (16, 32, 1, 0, 0)): (ALL, ALL),
    ("f32", (32, 32, 1, 0, 0)): (ALL, ALL),
    ("f32", (64, 128, 0, 0, 0)): (ALL, ALL),
    ("f32", (128, 128, 0, 0, 0)): (ALL, ALL - {BOTH}),
    ("f32", (16, 16, 1, 1, 0)): (ANY, ANY),
    ("f32", (32, 32, 1, 1, 0)): (ANY, ANY),
    ("f32", (64, 32, 1, 1, 0)): (ANY, ANY),
    ("f32", (128, 128, 0, 1, 0)): (ANY, ANY),
    ("16", (16, 16, 1, 0, 0)): (ALL - {BOTH}, ALL - {BOTH}),
    ("16", (16, 32, 1, 0, 0)): (ALL, ALL - {BOTH}),
    ("16", (32, 32, 1, 0, 0)): (ALL, ALL),
    ("16", (64, 32, 1, 0, 0)): (ALL, ALL),
    ("16", (64, 128, 0, 0, 0)): (ALL, ALL),
    ("16", (128, 128, 0, 0, 0)): (ALL, set()),
    ("16", (128, 128, 0, 0, 1)): (ALL, ALL),
    ("16", (256, 256, 0, 0, 0)): (ALL, set()),
    ("16", (16, 16, 1, 1, 0)): (ANY, ANY),
    ("16", (32, 32, 1, 1, 0)): (ANY, ANY),
    ("16", (64, 32, 1, 1, 0)): (ANY, ANY),
    ("16", (128, 128, 0, 1, 0)): (ANY, ANY),
}


def planned(case, dtype):
    strides = {}
    for name, pad, trans, rows, cols in (
            ("lhs_stride", case.pad_a, case.trans_a, case.m, case.k),
            ("rhs_stride", case.pad_b, case.trans_b, case.k, case.n)):
        rows, cols = (cols, rows) if trans else (rows, cols)
        if pad and rows > 1:  # (a single row has none behind it)
            strides[name] = cols + pad
    return ops.matmul_plan(case.m, case.k, case.n, dtype, trans_a=case.trans_a,
                           trans_b=case.trans_b, aligned=case.aligned,
                           workspace_elems=None if case.workspace else 0,
                           **strides)


def test_every_case_runs_on_its_kernel():
    for case in CASES:
        for dtype in TYPES[case.type]:
            p = planned(case, dtype)
            assert (p["tile_rows"], p["tile_cols"], p["shared"],
                    p["any_address"], p["pair"]) == case.kernel, case
            assert (p["first_copied"], p["second_copied"]) == case.copies, case
            assert p["shares"] == case.shares, case
            assert p["first_inner"] == 1 - case.trans_a
            assert p["second_inner"] == case.trans_b


def test_the_cases_reach_every_kernel():
    whole, shared, orders = {}, {}, {}
    for c in CASES:
        key = (c.type, c.kernel)
        (shared if c.shares > 1 else whole).setdefault(key, set()).add(c.copies)
        orders.setdefault(key, set()).add((c.trans_a, c.trans_b))
    for key, (copies, copies_shared) in REACHED.items():
        assert whole.get(key, set()) == copies, key
        assert shared.get(key, set()) == copies_shared, key
        assert len(orders[key]) == 4, key
    assert set(orders) == set(REACHED)
    # most of them end inside a tile, and inside a chunk of 128 bytes
    ragged = [c for c in CASES if c.m % c.kernel[0] and c.n % c.kernel[1]]
    assert len(ragged) > len(CASES) // 2


def test_no_other_kernel_is_chosen():
    rng = torch.Generator().manual_seed(0)

    def size(low, high):
        v = int(low * (high / low) ** torch.rand((), generator=rng).item())
        step = (1, 1, 8, 64)[int(torch.randint(4, (), generator=rng))]
        return max(low, v // step * step)

    for _ in range(3000):
        m, k, n = size(1, 8192), size(1, 4096), size(1, 8192)
        flags = torch.randint(2, (5,), generator=rng).tolist()
        dtype = (torch.float32, torch.bfloat16)[flags[0]]
        for product in (0, 1, 2):
            p = ops.matmul_plan(
                m, k, n, dtype, product,
                ACTIVATION.SILU if flags[1] else ACTIVATION.NONE, flags[2],
                flags[3], flags[4])
            kernel = (p["tile_rows"], p["tile_cols"], p["shared"],
                      p["any_address"], p["pair"])
            copies = (p["first_copied"], p["second_copied"])
            reached = REACHED["16" if flags[0] else "f32", kernel]
            # (the gradients' products have one operand at an aligned address more)
            assert copies in reached[p["shares"] > 1] or product


def test_orders_of_the_gradients():
    """grad op(lhs) = dz op(rhs)^T, grad op(rhs) = op(lhs)^T dz, or their transposes."""
    for trans_a in (0, 1):
        for trans_b in (0, 1):
            of_lhs, of_rhs = (ops.matmul_plan(
                130, 70, 90, torch.float16, product, ACTIVATION.GELU, trans_a,
                trans_b) for product in (1, 2))
            inner = [(p["first_inner"], p["second_inner"]) for p in (of_lhs, of_rhs)]
            of_d, of_r = 1, 1 - trans_b
            assert inner[0] == ((of_r, of_d) if trans_a else (of_d, of_r))
            of_d, of_l = 0, trans_a
            assert inner[1] == ((of_d, of_l) if trans_b else (of_l, of_d))


@pytest.mark.parametrize("dtype", [DTYPE.F32, DTYPE.F16, DTYPE.BF16])
def test_refusals(dtype):
    fn = capi.lib().snn_hip_matmul_bias_act_planned
    plan = capi.MatmulBiasActPlan()
    p = MatmulBiasActParams(m=8, k=8, n=8, activation=ACTIVATION.GELU)

    def call(params=p, product=0, kind=dtype, elems=1 << 20, to=plan):
        return fn(params and ctypes.byref(params), product, kind, 1, elems,
                  to and ctypes.byref(to))

    assert call() == STATUS.OK
    for kw in (dict(params=None), dict(product=3), dict(product=-1),
               dict(kind=3), dict(kind=-1), dict(to=None),
               dict(params=MatmulBiasActParams(m=0, k=8, n=8))):
        assert call(**kw) == STATUS.INVALID_PARAMETER, kw
    for product in (1, 2):
        assert call(product=product, elems=0) == STATUS.INSUFFICIENT_WORKSPACE
    wide = MatmulBiasActParams(m=1 << 21, k=64, n=1 << 20)
    assert call(params=wide) == STATUS.INDEX_EXCEEDED
