"""The recurrent block of the examples, which runs the operators for sequences
together, against the same formulas in 64 bits with automatic differentiation.

Every operator rounds its output once and is off by at most some 64 fp32
operations on terms that are up to ten times the result; norm by norm a stream
through eight operators is then off by 8 (2^-24 640 + rounding), and a gradient,
which has been through twice as many, by twice that."""
import pytest
import torch

import sequence_reference as ref
from portdnn_amd.examples import recurrent_block as example

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# batch, steps, width, inner, hidden
SIZES = [(2, 70, 40, 36, 56), (1, 1, 64, 64, 64), (3, 150, 72, 100, 33)]


def _bound(dtype, operators):
    return operators * (640 * ref.F32 + ref.ROUND[dtype])


def _close(got, want, bound, what):
    off = (got.detach().cpu().double() - want).norm().item()
    assert off <= bound * want.norm().item() + 1e-30, \
        "%s: off by %g of %g" % (what, off, want.norm().item())


def _rms(v, weight):
    return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight


def _plain(s, w, batch, steps, state=None, resets=None, lengths=None):
    """The block in the type of its operands: the stream and the state."""
    n = w["norm_inner"].numel()
    p = _rms(s, w["norm_in"]) @ w["w_in"] + w["b_in"]
    x, f, i, g = p.view(batch, steps, 4, n).unbind(2)
    a, b = torch.sigmoid(f), torch.sigmoid(i) * x
    h = torch.zeros(batch, n, dtype=s.dtype) if state is None else state
    rows = []
    for t in range(steps):
        keep = torch.ones(batch, 1, dtype=s.dtype)
        if resets is not None:
            keep = (resets[:, t:t + 1] == 0).to(s.dtype)
        now = a[:, t] * h * keep + b[:, t]
        if lengths is None:
            h = now
            rows.append(now)
        else:
            counts = (t < lengths)[:, None]
            h = torch.where(counts, now, h)
            rows.append(torch.where(counts, now, torch.zeros_like(now)))
    r = torch.stack(rows, 1).view(batch * steps, n)
    g = g.reshape(batch * steps, n)
    y = _rms(r, w["norm_inner"]) * g * torch.sigmoid(g)
    s2 = s + w["scale"] * (y @ w["w_out"])
    z = _rms(s2, w["norm_hidden"]) @ w["w_up"] + w["b_up"]
    return s2 + ref.activation(z, "GELU_TANH") @ w["w_down"], h


def _make(size, dtype, seed):
    batch, steps, width, inner, hidden = size
    rng = torch.Generator().manual_seed(seed)
    block = example.RecurrentBlock(width, inner, hidden, dtype, generator=rng)
    s = torch.randn(batch * steps, width, generator=rng).to(dtype)
    weights = {k: v.cpu().double().requires_grad_()
               for k, v in block.weights.items()}
    return rng, block, s, weights


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_block_and_its_gradients(size, dtype, ragged):
    batch, steps, width = size[:3]
    rng, block, s, weights = _make(size, dtype, 7)
    resets = lengths = None
    if ragged:
        resets = (torch.rand(batch, steps, generator=rng) < 0.1).to(torch.uint8)
        lengths = torch.randint(0, steps + 1, (batch,), generator=rng,
                                dtype=torch.int32)
        lengths[0] = steps
    on_gpu = [None if v is None else v.cuda() for v in (resets, lengths)]
    got, kept = block.forward(s.cuda(), batch, steps, resets=on_gpu[0],
                              lengths=on_gpu[1], keep=True)
    first = s.double().requires_grad_()
    want, _ = _plain(first, weights, batch, steps, resets=resets,
                     lengths=lengths)
    _close(got, want.detach(), _bound(dtype, 8), "stream")
    grad = torch.randn(s.shape, generator=rng).to(dtype)
    d_first, d_weights = block.backward(grad.cuda(), kept)
    want.backward(grad.double())
    _close(d_first, first.grad, _bound(dtype, 16), "gradient")
    assert set(d_weights) == set(weights)
    for name, d in d_weights.items():
        assert d.dtype == dtype
        _close(d, weights[name].grad, _bound(dtype, 16), name)


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_go_on_where_the_prompt_ended(dtype):
    size = batch, steps, width = 3, 90, 64
    prompt = 81
    _, block, s, weights = _make(size + (48, 80), dtype, 3)
    want, last = _plain(s.double(), {k: v.detach() for k, v in weights.items()},
                        batch, steps)
    rows = s.view(batch, steps, width).cuda()
    state = block.state(batch)
    out = [block.forward(rows[:, :prompt].reshape(-1, width), batch, prompt,
                         state=state).view(batch, prompt, width)]
    for t in range(prompt, steps):
        token = rows[:, t].contiguous()
        out.append(example.answer([block], [state], token)[:, None])
    _close(torch.cat(out, 1).view(-1, width), want, _bound(dtype, 8), "stream")
    _close(state, last, _bound(dtype, 8), "state")


def test_program_learns_and_answers():
    errors, apart = example.main(width=64, inner=96, hidden=128, depth=2,
                                 batch=4, steps=100, updates=12)
    assert all(e == e for e in errors)
    assert errors[-1] < errors[0]
    # values of the stream stay below ten or so
    assert apart < 2 * 10 * 2 * _bound(torch.float32, 8)
