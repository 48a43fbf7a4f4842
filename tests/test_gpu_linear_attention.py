"""Linear attention and its gradients against 64 bits, and against itself where
calls differ in ways that may not change a result."""
import ctypes

import pytest
import torch

import attention_reference as plain
import sequence_reference as ref
from portdnn_amd import capi, ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# batch, steps, heads, key_heads, keys, values
SIZES = [
    (2, 1, 2, 2, 16, 16), (3, 1, 6, 2, 200, 130), (2, 2, 1, 1, 1, 1),
    (2, 12, 4, 2, 24, 40), (2, 13, 4, 2, 24, 40), (2, 16, 4, 2, 24, 40),
    (2, 17, 4, 2, 24, 40), (3, 33, 3, 1, 13, 21),
    (1, 64, 2, 2, 64, 64), (2, 65, 2, 2, 64, 128), (2, 63, 4, 2, 72, 100),
    (2, 129, 2, 1, 128, 128), (1, 90, 2, 2, 255, 37), (1, 130, 1, 1, 256, 256),
    (2, 100, 2, 2, 37, 255), (3, 70, 2, 2, 8, 3), (1, 450, 2, 1, 32, 48),
    (1, 385, 1, 1, 128, 96), (2, 300, 1, 1, 160, 72),
]


def _make(size, dtype, resets=False, lengths=None, state=True, seed=0):
    batch, steps, heads, groups, keys, values = size
    g = torch.Generator().manual_seed(seed + steps + keys + values)

    def normal(*shape, kind=dtype):
        return torch.randn(shape, generator=g).to(kind)

    t = {"q": normal(batch, steps, groups, keys),
         "k": normal(batch, steps, groups, keys),
         "v": normal(batch, steps, heads, values),
         "decay": -0.3 * torch.rand(heads, generator=g)}
    t["decay"][0] = 0.0
    if resets:
        t["resets"] = (torch.rand(batch, steps, generator=g) < 0.05).to(
            torch.uint8)
    if lengths is not None:
        t["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    if state:
        t["initial_state"] = normal(batch, heads, keys, values,
                                    kind=torch.float32)
    grads = (normal(batch, steps, heads, values),
             normal(batch, heads, keys, values, kind=torch.float32))
    return t, grads


def _cuda(t):
    return {k: v.cuda() for k, v in t.items()}


def _wide(t):
    return {k: v.double() if v.is_floating_point() else v
            for k, v in t.items()}


def _check(t, grads, scale, what="", **kinds):
    dtype = t["q"].dtype
    keys, values = t["q"].shape[3], t["v"].shape[3]
    most = max(keys, values)
    gpu = _cuda(t)
    o, last = ops.linear_attention(scale=scale, **gpu, **kinds)
    want = plain.attention(scale=scale, dtype=dtype, **_wide(t))
    ref.check(o, want[0], plain.operations(most, dtype), what + " o")
    ref.check(last, want[1], plain.state_operations(most, dtype),
              what + " state")
    got = ops.linear_attention_grad(grads[0].cuda(), scale=scale,
                                    grad_final_state=grads[1].cuda(), **gpu,
                                    **kinds)
    want = plain.attention_grad(grads[0].double(), scale=scale, dtype=dtype,
                                grad_final_state=grads[1].double(), **_wide(t))
    assert set(got) == set(want)
    for name in ("q", "k", "v"):
        ref.check(got[name], want[name], plain.operations(most, dtype),
                  what + " d" + name)
    ref.check(got["initial_state"], want["initial_state"],
              plain.state_operations(most, dtype), what + " d state")


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_sizes(size, dtype):
    t, grads = _make(size, dtype)
    _check(t, grads, size[4] ** -0.5, str(size))


@pytest.mark.parametrize("size", [(3, 9, 4, 2, 24, 40), (3, 150, 4, 2, 64, 64),
                                  (4, 200, 2, 2, 40, 100),
                                  (3, 450, 1, 1, 128, 128)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("state", [True, False])
def test_resets_and_lengths(size, dtype, state):
    steps = size[1]
    lengths = [steps, 0, 1, steps - steps // 3][:size[0]]
    t, grads = _make(size, dtype, resets=True, lengths=lengths, state=state)
    t["resets"][0, 0] = 7
    # (what does not count is not read; the rest of the tensor has to be there)
    for b, n in enumerate(lengths):
        for name in ("q", "k", "v"):
            t[name][b, n:] = float("nan")
        grads[0][b, n:] = float("nan")
    sane = {k: v.nan_to_num(0.0) if v.is_floating_point() else v
            for k, v in t.items()}
    gpu, dtype = _cuda(t), t["q"].dtype
    most = max(size[4:])
    o, last = ops.linear_attention(scale=0.2, **gpu)
    want = plain.attention(scale=0.2, dtype=dtype, **_wide(sane))
    ref.check(o, want[0], plain.operations(most, dtype), "o")
    ref.check(last, want[1], plain.state_operations(most, dtype), "state")
    got = ops.linear_attention_grad(grads[0].cuda(), scale=0.2,
                                    grad_final_state=grads[1].cuda(), **gpu)
    want = plain.attention_grad(grads[0].nan_to_num(0.0).double(), scale=0.2,
                                dtype=dtype, grad_final_state=grads[1].double(),
                                **_wide(sane))
    for name, pair in want.items():
        count = plain.state_operations if name == "initial_state" else \
            plain.operations
        ref.check(got[name], pair, count(most, dtype), "d" + name)
    for b, n in enumerate(lengths):
        assert (o[b, n:] == 0).all()
        for name in ("q", "k", "v"):
            assert (got[name][b, n:] == 0).all()


@pytest.mark.parametrize("steps", [12, 150])
@pytest.mark.parametrize("dtype", TYPES)
def test_every_step_a_reset_or_none_left(steps, dtype):
    t, grads = _make((2, steps, 2, 2, 40, 24), dtype)
    t["resets"] = torch.ones(2, steps, dtype=torch.uint8)
    _check(t, grads, 1.0, "resets")
    t["decay"] = torch.tensor([3.0, -float("inf")])  # taken as 0 and -10000
    del t["resets"]
    _check(t, grads, 1.0, "decays")


@pytest.mark.parametrize("size", [(1, 450, 2, 1, 32, 48), (1, 385, 1, 1, 128, 96)])
@pytest.mark.parametrize("dtype", TYPES)
def test_without_a_workspace(size, dtype):
    """In one piece; with pieces test_sizes has them."""
    t, grads = _make(size, dtype, resets=True)
    gpu, most = _cuda(t), max(size[4:])
    room = torch.empty(0, dtype=dtype, device="cuda")
    o, last = ops.linear_attention(workspace=room, **gpu)
    want = plain.attention(dtype=dtype, **_wide(t))
    ref.check(o, want[0], plain.operations(most, dtype))
    ref.check(last, want[1], plain.state_operations(most, dtype))


def _poisoned(t, grads):
    """A value that is not finite in a column of v and, in step 60, of the
    output's gradient; the resets are in steps 40 and 90."""
    v, do = t["v"].clone(), grads[0].clone()
    v[:, 60, :, 2] = float("inf")
    v[:, 62, :, 3] = float("nan")
    do[:, 60, :, 2] = float("nan")
    return {**t, "v": v}, do


@pytest.mark.parametrize("keys,values", [(16, 16), (64, 64), (128, 128), (48, 200),
                                         (256, 256), (37, 53)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("room", [True, False])
def test_what_is_not_finite_stays_where_it_counts(keys, values, dtype, room):
    size = (1, 130, 2, 2, keys, values)
    t, grads = _make(size, dtype)
    t["resets"] = torch.zeros(1, 130, dtype=torch.uint8)
    t["resets"][:, [40, 90]] = 1
    bad, do = _poisoned(t, grads)
    kinds = {} if room else {"workspace": torch.empty(0, dtype=dtype,
                                                      device="cuda")}
    most = max(keys, values)
    o, last = ops.linear_attention(**_cuda(bad), **kinds)
    want = plain.attention(dtype=dtype, **_wide(t))
    others = [c for c in range(values) if c not in (2, 3)]

    def part(pair, f):
        return tuple(f(x) for x in pair)

    for f in (lambda x: x[:, :60], lambda x: x[:, 90:],
              lambda x: x[..., others]):
        ref.check(f(o), part(want[0], f), plain.operations(most, dtype))
    ref.check(last, want[1], plain.state_operations(most, dtype))
    assert not torch.isfinite(o[:, 60:90, :, 2].float()).any()
    # a gradient that is not finite: rows 40 to 60 of k and v, row 60 of q
    got = ops.linear_attention_grad(do.cuda(), **_cuda(t), **kinds)
    want = plain.attention_grad(grads[0].double(), dtype=dtype, **_wide(t))
    for name in ("k", "v"):
        for f in (lambda x: x[:, :40], lambda x: x[:, 61:]):
            ref.check(f(got[name]), part(want[name], f),
                      plain.operations(most, dtype), name)
    for f in (lambda x: x[:, :60], lambda x: x[:, 61:]):
        ref.check(f(got["q"]), part(want["q"], f),
                  plain.operations(most, dtype), "q")
    ref.check(got["initial_state"], want["initial_state"],
              plain.state_operations(most, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_finite_among_a_few_steps(dtype):
    t, _ = _make((2, 12, 2, 1, 40, 72), dtype)
    t["resets"] = torch.zeros(2, 12, dtype=torch.uint8)
    t["resets"][:, 8] = 1
    bad = {**t, "v": t["v"].clone(), "k": t["k"].clone(), "q": t["q"].clone()}
    bad["v"][:, 5, :, 2] = float("inf")
    bad["q"][:, 2] = float("nan")
    bad["k"][1, 7] = float("nan")
    o, last = ops.linear_attention(**_cuda(bad))
    want = plain.attention(dtype=dtype, **_wide(t))
    others = [c for c in range(72) if c != 2]
    count = plain.operations(72, dtype)

    def part(pair, f):
        return tuple(f(x) for x in pair)

    for f in (lambda x: x[:, :2], lambda x: x[:, 3:5], lambda x: x[:, 8:],
              lambda x: x[:1, 3:][..., others]):
        ref.check(f(o), part(want[0], f), count)
    assert torch.isnan(o[:, 2].float()).all()
    assert torch.isnan(o[1, 7].float()).all()
    assert not torch.isfinite(o[:, 5:8, :, 2].float()).any()
    ref.check(last, want[1], plain.state_operations(72, dtype))


@pytest.mark.parametrize("steps", [12, 150])
def test_lengths_beyond_the_sequence(steps):
    """They are taken as 0 and as all steps."""
    t, grads = _make((3, steps, 2, 1, 24, 40), torch.bfloat16,
                     lengths=[-5, steps + 1, 2 ** 31 - 1])
    _check(t, grads, 0.3)


@pytest.mark.parametrize("steps", [5, 200])
@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_states_end_at_a_reset(steps, dtype):
    t, _ = _make((1, steps, 2, 2, 24, 40), dtype)
    t["resets"] = torch.zeros(1, steps, dtype=torch.uint8)
    t["resets"][:, 3] = 1
    bad = {**t, "initial_state": t["initial_state"].clone()}
    bad["initial_state"][:, :, 7, 11] = float("inf")
    bad["initial_state"][:, :, 2, 30] = float("nan")
    o, last = ops.linear_attention(**_cuda(bad))
    want = plain.attention(dtype=dtype, **_wide(t))
    others = [c for c in range(40) if c not in (11, 30)]
    for f in (lambda x: x[:, 3:], lambda x: x[..., others]):
        ref.check(f(o), tuple(f(x) for x in want[0]), plain.operations(40, dtype))
    assert not torch.isfinite(o[:, :3, :, [11, 30]].float()).any()
    ref.check(last, want[1], plain.state_operations(40, dtype))


@pytest.mark.parametrize("steps", [5, 200])
def test_differences(steps):
    """Outputs are linear in q, k, v and the state: <gradient, e> is half the
    difference between the calls with +e and -e, but for what each of the 2
    steps * channels terms is off by."""
    size = (2, steps, 4, 2, 24, 40)
    t, (do, ds) = _make(size, torch.float32, resets=True,
                        lengths=[steps, steps - 2])
    gpu = _cuda(t)
    got = ops.linear_attention_grad(do.cuda(), grad_final_state=ds.cuda(), **gpu)

    def loss(**changed):
        o, last = ops.linear_attention(**{**gpu, **changed})
        return ((o.double().cpu() * do).sum() +
                (last.double().cpu() * ds).sum()).item()

    want = plain.attention(**_wide(t))
    size = ((want[0][1] * do.abs()).sum() + (want[1][1] * ds.abs()).sum()).item()
    g = torch.Generator().manual_seed(1)
    for name in ("q", "k", "v", "initial_state"):
        e = torch.randn(t[name].shape, generator=g)
        up, down = t[name] + e, t[name] - e
        by = 0.5 * (loss(**{name: up.cuda()}) - loss(**{name: down.cuda()}))
        of = (got[name].cpu().double() * (up - down).double() * 0.5).sum().item()
        # (the operand is at most some 6 times as large as before)
        bound = 8 * plain.operations(40, torch.float32) * ref.F32 * size
        assert abs(by - of) <= bound, (name, by, of, bound)


@pytest.mark.parametrize("steps", [1, 40, 200])
@pytest.mark.parametrize("dtype", TYPES)
def test_slices_of_a_projection(steps, dtype):
    """The same as for tensors of their own, also at addresses that are a multiple
    of nothing; gradients side by side, and what is around them stays."""
    size = batch, _, heads, groups, keys, values = 2, steps, 4, 2, 24, 32
    t, (do, _) = _make(size, dtype)
    gpu, do = _cuda(t), do.cuda()
    want = ops.linear_attention(**gpu)
    want_d = ops.linear_attention_grad(do, **gpu)
    n, m = groups * keys, heads * values
    for first in (0, 8, 3):
        p = torch.full((batch, steps, 2 * n + m + 16), 9.0, dtype=dtype,
                       device="cuda")
        rows = p[..., first:first + 2 * n + m]
        q = rows[..., :n].unflatten(2, (groups, keys))
        k = rows[..., n:2 * n].unflatten(2, (groups, keys))
        v = rows[..., 2 * n:].unflatten(2, (heads, values))
        for name, x in (("q", q), ("k", k), ("v", v)):
            x.copy_(gpu[name])
        these = {**gpu, "q": q, "k": k, "v": v}
        out = torch.empty(batch, steps, heads, values, dtype=dtype, device="cuda")
        got = ops.linear_attention(out=out, **these)
        assert got[0] is out
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        d = torch.full_like(p, 5.0)
        got = ops.linear_attention_grad(
            do, out=d[..., first:first + 2 * n + m], **these)
        for name, x in want_d.items():
            assert torch.equal(got[name], x), name
        assert (d[..., :first] == 5.0).all()
        assert (d[..., first + 2 * n + m:] == 5.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_token_by_token_in_place(dtype):
    """A prompt and then single tokens that update the state in place, against the
    whole sequence."""
    size = (2, 100, 4, 2, 64, 64)
    t, _ = _make(size, dtype)
    gpu = _cuda(t)
    want = plain.attention(dtype=dtype, **_wide(t))
    state = gpu.pop("initial_state").clone()

    def some(first, last):
        part = {n: gpu[n][:, first:last].contiguous() for n in ("q", "k", "v")}
        o, s = ops.linear_attention(decay=gpu["decay"], initial_state=state,
                                    final_state=state, **part)
        assert s is state
        return o

    rows = [some(0, 81), some(81, 90)] + [some(i, i + 1) for i in range(90, 100)]
    # (twelve calls: the state is rounded to fp32 in between, no more)
    count = plain.operations(64, dtype) + 12 + plain.state_operations(64, dtype)
    ref.check(torch.cat(rows, 1), want[0], count)
    ref.check(state, want[1], count)


def test_rows_far_apart():
    """A projection of more than 2^31 elements: offsets that pass 31 bits."""
    batch, steps, heads, n = 1, 32768, 2, 64
    wide = 66048
    p = torch.empty(steps, wide, dtype=torch.bfloat16, device="cuda")
    rows = p[None, :, wide - 6 * n:]
    g = torch.Generator().manual_seed(0)
    parts = []
    for i in range(3):
        part = torch.randn(batch, steps, heads, n, generator=g).to(torch.bfloat16)
        rows[..., i * 2 * n:(i + 1) * 2 * n].copy_(part.cuda().flatten(2))
        parts.append(part.cuda())
    decay = torch.tensor([-0.01, -0.3]).cuda()
    slices = [rows[..., i * 2 * n:(i + 1) * 2 * n].unflatten(2, (heads, n))
              for i in range(3)]
    want = ops.linear_attention(*parts, decay)
    got = ops.linear_attention(*slices, decay)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    do = torch.randn(batch, steps, heads, n, generator=g).to(torch.bfloat16).cuda()
    want = ops.linear_attention_grad(do, *parts, decay)
    d = p[None, :, :6 * n]
    # (the gradients of a projection, beside it)
    got = ops.linear_attention_grad(do, *slices, decay, out=d)
    for name, x in want.items():
        assert torch.equal(got[name], x), name
    # the last steps by themselves, from the state in front of them
    tail = 300
    _, s = ops.linear_attention(*[x[:, :-tail].contiguous() for x in parts], decay)
    end = [x[:, -tail:].contiguous().cpu().double() for x in parts]
    o, _ = ops.linear_attention(*parts, decay)
    want = plain.attention(*end, decay.cpu().double(), dtype=torch.bfloat16,
                           initial_state=s.cpu().double())
    ref.check(o[:, -tail:], want[0], 2 * plain.operations(n, torch.bfloat16))


@pytest.mark.parametrize("steps", [7, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_streams_and_graphs(steps, dtype):
    """On a stream of the caller's, twice at once, and as a graph that is replayed
    with other values in between; all the same to the bit."""
    size = (2, steps, 4, 2, 40, 72)
    a, (do, _) = _make(size, dtype, resets=True, lengths=[steps, steps // 2])
    b, _ = _make(size, dtype, resets=True, lengths=[steps - 1, steps], seed=5)
    do = do.cuda()
    both = [_cuda(a), _cuda(b)]

    def run(t):
        o, last = ops.linear_attention(**t)
        d = ops.linear_attention_grad(do, **t)
        return [o, last] + [d[n] for n in ("q", "k", "v", "initial_state")]

    want = [[x.clone() for x in run(t)] for t in both]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s, t in zip(streams, both):
        with torch.cuda.stream(s):
            got.append(run(t))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g, w))
    t = {k: v.clone() for k, v in both[0].items()}
    with torch.cuda.stream(streams[0]):
        run(t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(t)
    for turn in (0, 1, 0, 1):
        for k, v in both[turn].items():
            t[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want[turn]))
        run(both[1 - turn])  # eager work in between


@pytest.mark.parametrize("groups", [4, 2])
@pytest.mark.parametrize("steps", [9, 200])
def test_parts_that_are_not_wanted(groups, steps):
    """Each gradient alone is what it is among the others."""
    t, (do, ds) = _make((2, steps, 4, groups, 40, 40), torch.float32)
    gpu, do, ds = _cuda(t), do.cuda(), ds.cuda()
    want = ops.linear_attention_grad(do, grad_final_state=ds, **gpu)
    p = capi.LinearAttentionParams(batch=2, steps=steps, heads=4,
                                   key_heads=groups, keys=40, values=40,
                                   scale=1.0)
    room = torch.empty(1 << 20, device="cuda")
    for name, w in want.items():
        got = torch.empty_like(w)
        at = {n: got.data_ptr() if n == name else None for n in want}
        capi.check(capi.lib().snn_hip_linear_attention_grad_f32(
            do.data_ptr(), ds.data_ptr(), gpu["q"].data_ptr(),
            gpu["k"].data_ptr(), gpu["v"].data_ptr(), gpu["decay"].data_ptr(),
            None, None, gpu["initial_state"].data_ptr(), at["q"], at["k"],
            at["v"], at["initial_state"], ctypes.byref(p), room.data_ptr(),
            room.numel(), None))
        torch.cuda.synchronize()
        assert torch.equal(got, w), name


@pytest.mark.parametrize("steps", [3, 100])
@pytest.mark.parametrize("values", [24, 13])
def test_states_at_any_address(steps, values):
    """States that begin four bytes behind a multiple of sixteen."""
    size = (2, steps, 2, 2, 40, values)
    t, (do, ds) = _make(size, torch.bfloat16)
    gpu, do, ds = _cuda(t), do.cuda(), ds.cuda()
    want = ops.linear_attention(**gpu)
    want_d = ops.linear_attention_grad(do, grad_final_state=ds, **gpu)

    def moved(x):
        y = torch.empty(x.numel() + 1, device="cuda")[1:].view(x.shape)
        return y.copy_(x)

    gpu["initial_state"] = moved(gpu["initial_state"])
    got = ops.linear_attention(final_state=moved(ds), **gpu)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = ops.linear_attention_grad(do, grad_final_state=moved(ds), **gpu)
    assert all(torch.equal(got[n], w) for n, w in want_d.items())
