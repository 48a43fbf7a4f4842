"""The gated linear recurrence and its gradients against 64 bits.  A step's
gates, whose exponentials are off by a few units times the logit, and its sums
stay below 64 operations."""
import pytest
import torch

import sequence_reference as ref
from portdnn_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
OPERATIONS = 64


def _make(batch, steps, channels, dtype, gated, resets=False, lengths=None,
          state=True, seed=0):
    g = torch.Generator().manual_seed(seed + steps + channels)

    def normal(*shape, mean=0.0, kind=dtype):
        return (torch.randn(shape, generator=g) + mean).to(kind)

    t = {"x": normal(batch, steps, channels),
         "forget": normal(batch, steps, channels, mean=2.0)}
    if gated:
        t["input_gate"] = normal(batch, steps, channels)
    if resets:
        t["resets"] = (torch.rand(batch, steps, generator=g) < 0.1).to(
            torch.uint8)
    if lengths is not None:
        t["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    if state:
        t["initial_state"] = normal(batch, channels, kind=torch.float32)
    return g, t


def _reference(t):
    names = {"x": "x", "forget": "f", "input_gate": "i", "resets": "resets",
             "lengths": "lengths", "initial_state": "h0"}
    return {names[k]: v.double() if v.is_floating_point() else v
            for k, v in t.items()}


def _check(t, dtype, g, workspace=None):
    what = "%s %s" % (tuple(t["x"].shape), sorted(t))
    gpu = {k: v.cuda() for k, v in t.items()}
    h, last = ops.linear_recurrence(**gpu, workspace=workspace)
    want_h, want_last = ref.recurrence(**_reference(t))
    ref.check(h, want_h, OPERATIONS, what + " h")
    ref.check(last, want_last, OPERATIONS, what + " last")
    dh = torch.randn(t["x"].shape, generator=g).to(dtype)
    d_last = torch.randn(last.shape, generator=g)
    got = ops.linear_recurrence_grad(dh.cuda(), h=h, grad_final_state=d_last.cuda(),
                                     workspace=workspace, **gpu)
    want = ref.recurrence_grad(dh.double(), h=h.cpu().double(),
                               d_last=d_last.double(), **_reference(t))
    assert set(got) == set(want)
    for name, v in got.items():
        ref.check(v, want[name], OPERATIONS, what + " " + name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_sizes(dtype, gated, masked):
    for batch, steps, channels in (
            (1, 1, 1), (2, 1, 64), (5, 1, 333), (1, 7, 256), (3, 8, 100),
            (2, 9, 130), (1, 64, 260), (2, 65, 64), (3, 130, 77), (1, 500, 36),
            (1, 1203, 8)):
        lengths = None
        if masked:
            lengths = [steps, 0, steps // 2, 1, max(0, steps - 1)][:batch]
        g, t = _make(batch, steps, channels, dtype, gated, resets=masked,
                     lengths=lengths)
        _check(t, dtype, g)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_workspace_and_without_a_state(dtype):
    none = torch.empty(0, dtype=dtype, device="cuda")
    for steps in (1, 40, 333):
        g, t = _make(2, steps, 72, dtype, True, state=False)
        _check(t, dtype, g)
        _check(t, dtype, g, workspace=none)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_slices_of_a_projection(dtype, gated, shift):
    parts = 3 if gated else 2
    names = ["x", "forget", "input_gate"][:parts]
    for batch, steps, channels in ((3, 1, 64), (2, 100, 68), (1, 77, 33)):
        g, t = _make(batch, steps, channels, dtype, gated, resets=True)
        plain = {k: v.cuda() for k, v in t.items()}
        both = torch.full((batch, steps, parts * channels + 8), float("nan"),
                          dtype=dtype, device="cuda")
        views = dict(plain)
        for i, name in enumerate(names):
            at = shift + i * channels
            views[name] = both[..., at:at + channels]
            views[name].copy_(plain[name])
        h, last = ops.linear_recurrence(**views)
        want_h, want_last = ref.recurrence(**_reference(t))
        ref.check(h, want_h, OPERATIONS)
        ref.check(last, want_last, OPERATIONS)
        dh = torch.randn(h.shape, generator=g).to(dtype).cuda()
        out = torch.full((batch, steps, parts * channels), float("nan"),
                         dtype=dtype, device="cuda")
        got = ops.linear_recurrence_grad(dh, h=h, out=out, **views)
        want = ref.recurrence_grad(dh.cpu().double(), h=h.cpu().double(),
                                   **_reference(t))
        for i, name in enumerate(names):
            ref.check(out[..., i * channels:(i + 1) * channels], want[name],
                      OPERATIONS, name)
        ref.check(got["initial_state"], want["initial_state"], OPERATIONS)


@pytest.mark.parametrize("dtype", TYPES)
def test_single_tokens_in_place_are_the_sequence(dtype):
    batch, steps, channels = 3, 20, 72
    g, t = _make(batch, steps, channels, dtype, True)
    gpu = {k: v.cuda() for k, v in t.items()}
    state = gpu.pop("initial_state").clone()
    rows = []
    for n in range(steps):
        one = {k: v[:, n:n + 1].contiguous() for k, v in gpu.items()}
        h, after = ops.linear_recurrence(**one, initial_state=state,
                                         final_state=state)
        assert after is state
        rows.append(h)
    want_h, want_last = ref.recurrence(**_reference(t))
    ref.check(torch.cat(rows, 1), want_h, OPERATIONS)
    ref.check(state, want_last, OPERATIONS)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_sequences_in_place_and_in_parts(dtype):
    """The state of the first half is the second half's; the buffer is one."""
    batch, steps, channels = 1, 2000, 48
    g, t = _make(batch, steps, channels, dtype, False, resets=True)
    gpu = {k: v.cuda() for k, v in t.items()}
    state = gpu.pop("initial_state").clone()
    cut = 1111
    halves = []
    for part in (slice(0, cut), slice(cut, steps)):
        one = {k: v[:, part].contiguous() for k, v in gpu.items()}
        halves.append(ops.linear_recurrence(**one, initial_state=state,
                                            final_state=state)[0])
    want_h, want_last = ref.recurrence(**_reference(t))
    ref.check(torch.cat(halves, 1), want_h, OPERATIONS)
    ref.check(state, want_last, OPERATIONS)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("steps", [12, 700])
def test_what_lies_behind_a_reset_or_the_end_does_not_matter(dtype, steps):
    batch, channels = 4, 40
    lengths = [0, 5, steps - 3, steps]
    g, t = _make(batch, steps, channels, dtype, True, lengths=lengths)
    resets = torch.zeros(batch, steps, dtype=torch.uint8)
    resets[2, 4] = 200
    resets[3, 0] = 1
    t["resets"] = resets
    _check(t, dtype, g)
    gpu = {k: v.cuda() for k, v in t.items()}
    clean_h, clean_last = ops.linear_recurrence(**gpu)
    dh = torch.randn(batch, steps, channels, generator=g).to(dtype).cuda()
    clean = ops.linear_recurrence_grad(dh, h=clean_h, **gpu)
    for name in ("x", "forget", "input_gate"):
        gpu[name] = gpu[name].clone()
        for b, n in enumerate(lengths):
            gpu[name][b, n:] = float("nan")
    spoilt = clean_h.clone()
    for b, n in enumerate(lengths):
        dh[b, n:] = float("nan")
        spoilt[b, n:] = float("nan")
    # an infinite state in front of a reset
    gpu["initial_state"] = gpu["initial_state"].clone()
    gpu["initial_state"][3] = float("inf")
    h, last = ops.linear_recurrence(**gpu)
    assert torch.equal(h, clean_h) and torch.equal(last, clean_last)
    got = ops.linear_recurrence_grad(dh, h=spoilt, **gpu)
    for name, v in got.items():
        assert torch.equal(v, clean[name]), name
    assert not got["x"][1, 5:].any() and not h[0].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_gates_that_are_shut_and_open(dtype):
    """Logits far out: no overflow, no NaN, and the exact limits."""
    steps = 50
    x = torch.randn(1, steps, 64, device="cuda").to(dtype)
    state = torch.randn(1, 64, device="cuda")
    far = torch.full_like(x, 60000.0 if dtype == torch.float16 else 1e30)
    h, last = ops.linear_recurrence(x, far, initial_state=state)
    assert torch.equal(last, state)
    h, last = ops.linear_recurrence(x, -far, initial_state=state)
    assert torch.equal(h, x)
    h, last = ops.linear_recurrence(x, -far, input_gate=far)
    assert torch.equal(h, x)
    got = ops.linear_recurrence_grad(x, x, far, h, input_gate=-far)
    assert all(v.isfinite().all() for v in got.values())
    assert not got["forget"].any() and not got["x"].any()


def test_lengths_out_of_range_are_clamped():
    g, t = _make(3, 30, 64, torch.float32, False, lengths=[-5, 99, 30])
    gpu = {k: v.cuda() for k, v in t.items()}
    h, last = ops.linear_recurrence(**gpu)
    gpu["lengths"] = torch.tensor([0, 30, 30], dtype=torch.int32).cuda()
    again = ops.linear_recurrence(**gpu)
    assert torch.equal(h, again[0]) and torch.equal(last, again[1])


def test_sequences_beyond_two_gigabytes():
    steps, channels = (1 << 20) + 100, 2056
    dtype = torch.float16
    x = torch.zeros((1, steps, channels), dtype=dtype, device="cuda")
    f = torch.full_like(x, 3.0)
    g = torch.Generator().manual_seed(1)
    tail = torch.randn(1, 400, channels, generator=g).to(dtype)
    x[:, -400:] = tail.cuda()
    h, last = ops.linear_recurrence(x, f)
    want_h, want_last = ref.recurrence(tail.double(),
                                       torch.full_like(tail, 3.0).double())
    ref.check(h[:, -400:], want_h, OPERATIONS)
    ref.check(last, want_last, OPERATIONS)
    del f
    dh = torch.zeros_like(x)
    dh[:, :300] = tail[:, :300].cuda()
    f = torch.full_like(x, 3.0)
    got = ops.linear_recurrence_grad(dh, x, f, h)
    want = ref.recurrence_grad(
        tail[:, :300].double(), x[:, :300].cpu().double(),
        f[:, :300].cpu().double(), h[:, :300].cpu().double())
    ref.check(got["x"][:, :300], want["x"], OPERATIONS)
    ref.check(got["initial_state"], want["initial_state"], OPERATIONS)


def test_another_stream_a_graph_and_the_same_bits_again():
    _, t = _make(2, 900, 264, torch.bfloat16, True, resets=True)
    gpu = {k: v.cuda() for k, v in t.items()}
    dh = torch.randn(2, 900, 264, device="cuda").bfloat16()

    def run():
        h, last = ops.linear_recurrence(**gpu)
        return [h, last, *ops.linear_recurrence_grad(
            dh, h=h, grad_final_state=last, **gpu).values()]

    eager = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = run()
    stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(3):
        for v in captured:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = run()
        assert all(torch.equal(x, y) for x, y in zip(captured, again))
