"""The linear-attention block of the examples, which runs the operators together,
against the same formulas in 64 bits with automatic differentiation.

Every operator rounds its output once and is off by at most some 64 fp32
operations on terms that are up to ten times the result; norm by norm a stream
through ten operators is then off by 10 (2^-24 640 + rounding), and a gradient,
which has been through twice as many, by twice that.  The attention rounds its
products of queries and keys besides: one operator more."""
import math

import pytest
import torch

import sequence_reference as ref
from portdnn_amd.examples import linear_attention_block as example

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# batch, steps, width, heads, key_heads, channels, hidden
SIZES = [(2, 70, 40, 4, 2, 16, 56), (1, 1, 64, 2, 2, 32, 64),
         (3, 150, 72, 3, 1, 20, 33)]


def _bound(dtype, operators):
    return operators * (640 * ref.F32 + ref.ROUND[dtype])


def _close(got, want, bound, what):
    off = (got.detach().cpu().double() - want).norm().item()
    assert off <= bound * want.norm().item() + 1e-30, \
        "%s: off by %g of %g" % (what, off, want.norm().item())


def _rms(v, weight):
    return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight


def _turned(x, first):
    """Positions by rotation of [batch, steps, heads, channels]."""
    n = x.shape[3] // 2
    at = first.double()[:, None] + torch.arange(x.shape[1]).double()
    w = at[..., None] * 10000.0 ** (-torch.arange(n).double() / n)
    c, s = w.cos()[:, :, None], w.sin()[:, :, None]
    a, b = x[..., :n], x[..., n:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain(s, block, w, batch, steps, first=None, resets=None, lengths=None):
    """The block in the type of its operands: the stream and the state."""
    heads, groups, n = block.heads, block.key_heads, block.channels
    p = (_rms(s, w["norm_in"]) @ w["w_in"]).view(batch, steps, -1)
    first = torch.zeros(batch) if first is None else first
    q = _turned(p[..., :groups * n].unflatten(2, (groups, n)), first)
    k = _turned(p[..., groups * n:2 * groups * n].unflatten(2, (groups, n)), first)
    q, k = (t.repeat_interleave(heads // groups, 2) for t in (q, k))
    v, g = p[..., 2 * groups * n:].unflatten(2, (2, heads, n)).unbind(2)
    a = block.decay.cpu().double().exp()
    state = torch.zeros(batch, heads, n, n, dtype=s.dtype)
    rows = []
    for t in range(steps):
        keep = a.expand(batch, heads)
        if resets is not None:
            keep = keep * (resets[:, t:t + 1] == 0)
        now = (keep[..., None, None] * state +
               k[:, t, :, :, None] * v[:, t, :, None, :])
        row = n ** -0.5 * (q[:, t, :, :, None] * now).sum(2)
        if lengths is not None:
            counts = (t < lengths)[:, None, None]
            now = torch.where(counts[..., None], now, state)
            row = torch.where(counts, row, torch.zeros_like(row))
        state = now
        rows.append(row)
    h = torch.stack(rows, 1).reshape(batch * steps, -1)
    g = g.reshape(batch * steps, -1)
    y = _rms(h, w["norm_inner"]) * g * torch.sigmoid(g)
    s2 = s + y @ w["w_out"]
    z = _rms(s2, w["norm_hidden"])
    m = ref.activation(z @ w["w_gate"], "SILU") * (z @ w["w_up"])
    return s2 + m @ w["w_down"], state


def _make(size, dtype, seed):
    batch, steps, width = size[:3]
    rng = torch.Generator().manual_seed(seed)
    block = example.LinearAttentionBlock(width, *size[3:], dtype, generator=rng)
    s = torch.randn(batch * steps, width, generator=rng).to(dtype)
    weights = {k: v.cpu().double().requires_grad_()
               for k, v in block.weights.items()}
    return rng, block, s, weights


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_block_and_its_gradients(size, dtype, ragged):
    batch, steps = size[:2]
    rng, block, s, weights = _make(size, dtype, 7)
    resets = lengths = first = None
    if ragged:
        resets = (torch.rand(batch, steps, generator=rng) < 0.1).to(torch.uint8)
        lengths = torch.randint(0, steps + 1, (batch,), generator=rng,
                                dtype=torch.int32)
        lengths[0] = steps
        first = torch.randint(0, 1000, (batch,), generator=rng,
                              dtype=torch.int32)
    on_gpu = [None if v is None else v.cuda() for v in (resets, lengths, first)]
    got, kept = block.forward(s.cuda(), batch, steps, resets=on_gpu[0],
                              lengths=on_gpu[1], positions=on_gpu[2], keep=True)
    stream = s.double().requires_grad_()
    want, _ = _plain(stream, block, weights, batch, steps, first, resets, lengths)
    _close(got, want.detach(), _bound(dtype, 11), "stream")
    grad = torch.randn(s.shape, generator=rng).to(dtype)
    d_stream, d_weights = block.backward(grad.cuda(), kept)
    want.backward(grad.double())
    _close(d_stream, stream.grad, _bound(dtype, 22), "gradient")
    assert set(d_weights) == set(weights)
    for name, d in d_weights.items():
        assert d.dtype == dtype
        _close(d, weights[name].grad, _bound(dtype, 22), name)


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_go_on_where_the_prompt_ended(dtype):
    batch, steps, width, prompt = 3, 90, 64, 81
    _, block, s, weights = _make((batch, steps, width, 4, 2, 16, 80), dtype, 3)
    want, last = _plain(s.double(), block,
                        {k: v.detach() for k, v in weights.items()}, batch, steps)
    rows = s.view(batch, steps, width).cuda()
    state = block.state(batch)
    out = [block.forward(rows[:, :prompt].reshape(-1, width), batch, prompt,
                         state=state).view(batch, prompt, width)]
    for t in range(prompt, steps):
        at = torch.full((batch,), t, dtype=torch.int32, device="cuda")
        out.append(example.answer([block], [state], rows[:, t].contiguous(),
                                  at)[:, None])
    _close(torch.cat(out, 1).view(-1, width), want, _bound(dtype, 11), "stream")
    _close(state, last, _bound(dtype, 11), "state")


def test_program_runs():
    errors, apart = example.main(width=64, heads=4, key_heads=2, channels=24,
                                 hidden=128, depth=2, batch=4, steps=100,
                                 updates=12)
    assert all(math.isfinite(e) for e in errors)
    # values of the stream stay below ten or so
    assert apart < 2 * 10 * 2 * _bound(torch.float32, 11)
