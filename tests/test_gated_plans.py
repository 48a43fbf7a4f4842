"""The choice among the kernels of the gated product: that the products of
gated_kernel_cases reach all of them.  Decided on the host."""
import ctypes

import pytest
import torch

from gated_kernel_cases import CASES
from portdnn_amd import capi, ops
from portdnn_amd.capi import ACTIVATION, DTYPE, STATUS, GatedMatmulParams

TYPES = {"f32": [torch.float32], "16": [torch.float16, torch.bfloat16]}
FEW = [(16, 32, 1, 0, 0), (16, 64, 1, 0, 0), (32, 32, 1, 0, 0), (32, 64, 1, 0, 0)]
KERNELS = {
    "f32": FEW + [(64, 128, 0, 0, 0), (128, 128, 0, 0, 0)],
    "16": FEW + [(64, 32, 1, 0, 0), (64, 128, 0, 0, 0), (128, 128, 0, 0, 0),
                 (128, 128, 0, 0, 1), (256, 256, 0, 0, 0)]}
ANY = (16, 32, 1, 1, 0)  # operands by way of registers, which are not copied
# (type, product, kernel) that no size was found to give a shared reduction
WHOLE = {("16", 0, (128, 128, 0, 0, 0)), ("16", 0, (256, 256, 0, 0, 0)),
         ("f32", 1, (32, 64, 1, 0, 0))}


def planned(case, dtype):
    strides = {}
    if case.pad_a and case.m > 1:  # (a single row has none behind it)
        strides["lhs_stride"] = case.k + case.pad_a
    rows, cols = (case.n, case.k) if case.trans_b else (case.k, case.n)
    if case.pad_b and rows > 1:
        strides["rhs_stride"] = cols + case.pad_b
    return ops.gated_matmul_plan(
        case.m, case.k, case.n, dtype, case.product, trans_b=case.trans_b,
        aligned=case.aligned, workspace_elems=None if case.workspace else 0,
        **strides)


def kernel_of(p):
    return (p["tile_rows"], p["tile_cols"], p["shared"], p["any_address"], p["pair"])


def test_every_case_runs_on_its_kernel():
    for case in CASES:
        for dtype in TYPES[case.type]:
            p = planned(case, dtype)
            assert kernel_of(p) == case.kernel, case
            assert (p["first_copied"], p["second_copied"]) == case.copies, case
            assert p["shares"] == case.shares, case
            assert p["first_inner"] == 1
            assert p["second_inner"] == (case.trans_b if case.product == 0
                                         else 1 - case.trans_b)


def test_the_cases_reach_every_kernel():
    whole, shared, orders = {}, {}, {}
    for c in CASES:
        key = (c.type, c.product, c.kernel)
        (shared if c.shares > 1 else whole).setdefault(key, set()).add(c.copies)
        if c.shares == 1:
            orders.setdefault(key, set()).add(c.trans_b)
    for kind, kernels in KERNELS.items():
        for product in (0, 1):
            for kernel in kernels + [ANY]:
                key = (kind, product, kernel)
                copies = {(0, 0)} if kernel == ANY else {(0, 0), (0, 1), (1, 0),
                                                         (1, 1)}
                assert whole.pop(key) == copies, key
                assert ((0, 0) in shared.pop(key, set())) == (key not in WHOLE), key
                # (tiles of 16 x 32 take the input's gradient of weights by column
                # in 16 bits only in shares)
                if key != ("16", 1, (16, 32, 1, 0, 0)):
                    assert orders[key] == {0, 1}, key
    assert not whole and not shared
    # most of them end inside a tile's rows
    assert len([c for c in CASES if c.m % c.kernel[0]]) > len(CASES) // 2


def test_no_other_kernel_is_chosen():
    rng = torch.Generator().manual_seed(0)

    def size(low, high):
        v = int(low * (high / low) ** torch.rand((), generator=rng).item())
        step = (1, 1, 8, 64)[int(torch.randint(4, (), generator=rng))]
        return max(low, v // step * step)

    for _ in range(3000):
        m, k, n = size(1, 8192), size(1, 4096), size(1, 8192)
        flags = torch.randint(2, (4,), generator=rng).tolist()
        kind = "16" if flags[0] else "f32"
        for product in (0, 1, 2):
            p = ops.gated_matmul_plan(m, k, n, TYPES[kind][-1], product,
                                      trans_b=flags[1], aligned=flags[2])
            if product < 2:
                kernel = kernel_of(p)
                assert kernel in KERNELS[kind] + [ANY]
                assert p["shares"] == 1 or (kind, product, kernel) not in WHOLE


@pytest.mark.parametrize("dtype", [DTYPE.F32, DTYPE.F16, DTYPE.BF16])
def test_refusals(dtype):
    fn = capi.lib().snn_hip_gated_matmul_planned
    plan = capi.MatmulBiasActPlan()
    p = GatedMatmulParams(m=8, k=8, n=8, activation=ACTIVATION.SILU)

    def call(params=p, product=0, kind=dtype, elems=1 << 20, to=plan):
        return fn(params and ctypes.byref(params), product, kind, 1, elems,
                  to and ctypes.byref(to))

    assert call() == STATUS.OK
    for kw in (dict(params=None), dict(product=3), dict(product=-1),
               dict(kind=3), dict(kind=-1), dict(to=None),
               dict(params=GatedMatmulParams(m=0, k=8, n=8))):
        assert call(**kw) == STATUS.INVALID_PARAMETER, kw
    for product in (1, 2):
        assert call(product=product, elems=0) == STATUS.INSUFFICIENT_WORKSPACE
    wide = GatedMatmulParams(m=8, k=1 << 29, n=8)
    assert call(params=wide) == STATUS.INDEX_EXCEEDED
