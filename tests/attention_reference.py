"""Plain 64-bit implementations of the operators of a linear-attention block, each
with the magnitude that bounds the error of an implementation in fp32 as in
sequence_reference: what the value would be if all its terms had one sign.
"""
import math

import torch

import sequence_reference as ref

F32, ROUND = ref.F32, ref.ROUND


def per_rounding(dtype):
    """fp32 operations that are off by as much as one rounding to `dtype`."""
    return ROUND[dtype] / F32


# ---- the gated product ----------------------------------------------------------


def slope(z, kind):
    """The derivative of ref.activation."""
    if kind == "RELU":
        return (z > 0).double()
    if kind == "GELU":
        return (0.5 * torch.special.erfc(-z / math.sqrt(2.0)) +
                z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi))
    if kind == "GELU_TANH":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return (0.5 * (1.0 + t) +
                0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z))
    if kind == "SILU":
        s = ref.sigma(z)
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def gated(x, gate, up, bias_gate=None, bias_up=None, kind="SILU"):
    """(output, gate's factor, up's factor), each with its magnitude.  No slope is
    above 1.2, and |act(z)| is at most |z|."""
    z, u = x @ gate, x @ up
    mz, mu = x.abs() @ gate.abs(), x.abs() @ up.abs()
    if bias_gate is not None:
        z, mz = z + bias_gate, mz + bias_gate.abs()
    if bias_up is not None:
        u, mu = u + bias_up, mu + bias_up.abs()
    out = ref.activation(z, kind) * u
    return ((out, 1.2 * mz * u.abs() + z.abs() * mu), (z, mz), (u, mu))


def gated_grad(dy, x, gate, up, z, u, kind="SILU"):
    """Gradients of x, gate, up and of the two biases."""
    dz = dy * u * slope(z, kind)
    du = dy * ref.activation(z, kind)
    # (of slopes and activations the terms: at most 3 |z| + 1.2 and |z|)
    mz, mu = dy.abs() * u.abs() * (1.2 + 3.0 * z.abs()), dy.abs() * z.abs()
    return {
        "x": (dz @ gate.T + du @ up.T,
              mz @ gate.abs().T + mu @ up.abs().T),
        "gate": (x.T @ dz, x.abs().T @ mz), "up": (x.T @ du, x.abs().T @ mu),
        "bias_gate": (dz.sum(0), mz.sum(0)), "bias_up": (du.sum(0), mu.sum(0))}


# ---- positions by rotation ------------------------------------------------------


def rotary(x, frequencies, positions, halves=True, magnitude=1.0, inverse=False):
    """positions: [batch, steps] integers, frequencies: float64 turns."""
    n = frequencies.numel()
    turns = positions.double()[..., None] * frequencies
    angle = 2.0 * math.pi * (turns - turns.round())
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    if inverse:
        s = -s
    y, m = x.clone(), x.abs()
    first = slice(0, n) if halves else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if halves else slice(1, 2 * n, 2)
    a, b = x[..., first], x[..., second]
    y[..., first] = magnitude * (a * c - b * s)
    y[..., second] = magnitude * (a * s + b * c)
    m[..., first] = m[..., second] = abs(magnitude) * (a.abs() + b.abs())
    # (the other channels are copies: their rounding is none, and this bounds it)
    return y, m


def frequencies(turned, base=10000.0, scaling="NONE", factor=1.0, context=0.0,
                low=1.0, high=32.0):
    i = torch.arange(turned // 2, dtype=torch.float64)
    if scaling == "BASE" and turned > 2:
        base = base * factor ** (turned / (turned - 2))
    f = base ** (-2.0 * i / turned) / (2.0 * math.pi)
    if scaling == "POSITIONS":
        f = f / factor
    if scaling == "BANDS":
        keep = ((context * f - low) / (high - low)).clamp(0.0, 1.0)
        f = keep * f + (1.0 - keep) * f / factor
    return f


# ---- linear attention -----------------------------------------------------------


def walk(q, k, v, keep, state, counts, from_end=False, first_decays=True):
    """o_t = q_t S_t with S_t = keep_t S_{t-1} + k_t^T v_t from `state` on, over
    [batch, steps, heads, ...]; keep: [batch, steps, heads]; rows that do not
    count are skipped.  From the end keep_t belongs to the step from t on to
    t - 1, and the first step takes `state` as it is where not first_decays."""
    batch, steps, heads = v.shape[:3]
    o = torch.zeros(batch, steps, heads, v.shape[3], dtype=v.dtype)
    rows = []
    states = state
    fresh = torch.ones(batch, dtype=torch.bool)
    before = torch.ones(batch, heads, dtype=v.dtype)  # the weight of the state
    order = range(steps - 1, -1, -1) if from_end else range(steps)
    for t in order:
        on = counts[:, t]
        weight = before if from_end else keep[:, t]
        if not first_decays:
            weight = torch.where(fresh[:, None], torch.ones_like(weight), weight)
        now = (torch.where(weight[..., None, None] == 0,
                           torch.zeros_like(states),
                           weight[..., None, None] * states) +
               k[:, t, :, :, None] * v[:, t, :, None, :])
        states = torch.where(on[:, None, None, None], now, states)
        got = (q[:, t, :, :, None] * states).sum(2)
        rows.append(torch.where(on[:, None, None], got, torch.zeros_like(got)))
        before = torch.where(on[:, None], keep[:, t], before)
        fresh = fresh & ~on
    if from_end:
        rows.reverse()
        # (to the state in front of the first step)
        states = torch.where(before[..., None, None] == 0,
                             torch.zeros_like(states),
                             before[..., None, None] * states)
    return (torch.stack(rows, 1) if steps else o), states


def _weights(shape, decay, resets, lengths):
    batch, steps, heads = shape[:3]
    a = torch.exp(decay.double().clamp(-10000.0, 0.0))
    keep = a.expand(batch, steps, heads).clone()
    full = torch.ones_like(keep)  # without decays
    if resets is not None:
        keep[resets != 0] = 0.0
        full[resets != 0] = 0.0
    counts = torch.ones(batch, steps, dtype=torch.bool)
    if lengths is not None:
        counts = (torch.arange(steps)[None] <
                  lengths.clamp(0, steps)[:, None])
    return keep, full, counts


def _shared(t, heads):
    return t.repeat_interleave(heads // t.shape[2], 2)


def _all(dtype, q, k, v, keep, full, state, counts, **kinds):
    """(outputs, state), each a value and a magnitude that also holds what values
    too small for binary16 lose: half of 2^-24 for each weighted value, each state
    and each q_t k_s that is rounded to it, as many as there are, whatever decays
    take from them.  Powers of a decay have 2^-126 added to them, so that they are
    above zero: as much of what has not decayed."""
    value = walk(q, k, v, keep, state, counts, **kinds)
    size = walk(q.abs(), k.abs(), v.abs(), keep, state.abs(), counts, **kinds)
    if keep.min() < 0.1:
        whole = walk(q.abs(), k.abs(), v.abs(), full, state.abs(), counts, **kinds)
        size = tuple(a + 2.0 ** -126 / F32 * b for a, b in zip(size, whole))
    if dtype is torch.float16:
        ones = torch.ones_like
        kept = ones(keep)
        lost = 2.0 ** -25 / F32
        of_v = walk(q.abs(), k.abs(), lost * ones(v), kept,
                    lost * ones(state), counts, **kinds)
        of_p = walk(lost * ones(q[..., :1]), ones(q[..., :1]), v.abs(), kept,
                    torch.zeros_like(state[:, :, :1]), counts, **kinds)
        size = (size[0] + of_v[0] + of_p[0], size[1] + of_v[1])
    return list(zip(value, size))


def attention(q, k, v, decay, resets=None, lengths=None, initial_state=None,
              scale=1.0, dtype=torch.float32):
    """((output, magnitude), (final state, magnitude)); operands as the operator
    takes them, in 64 bits; dtype: the operator's."""
    heads = v.shape[2]
    q, k = scale * _shared(q, heads), _shared(k, heads)
    keep, full, counts = _weights(v.shape, decay, resets, lengths)
    if initial_state is None:
        initial_state = torch.zeros(v.shape[0], heads, q.shape[3], v.shape[3],
                                    dtype=v.dtype)
    return _all(dtype, q, k, v, keep, full, initial_state, counts)


def attention_grad(do, q, k, v, decay, resets=None, lengths=None,
                   initial_state=None, grad_final_state=None, scale=1.0,
                   dtype=torch.float32):
    """A dict of pairs: the gradients of q, k, v and initial_state."""
    heads, groups = v.shape[2], q.shape[2]
    Q, K = scale * _shared(q, heads), _shared(k, heads)
    keep, full, counts = _weights(v.shape, decay, resets, lengths)
    state = torch.zeros(v.shape[0], heads, q.shape[3], v.shape[3], dtype=v.dtype)
    s0 = state if initial_state is None else initial_state
    ds = state if grad_final_state is None else grad_final_state
    end = dict(from_end=True, first_decays=False)
    dq, _ = _all(dtype, do, v, K, keep, full, s0.transpose(2, 3), counts)
    dq = tuple(abs(scale) * t if i else scale * t for i, t in enumerate(dq))
    dk, _ = _all(dtype, v, do, Q, keep, full, ds.transpose(2, 3), counts,
                 **end)
    dv, d0 = _all(dtype, K, Q, do, keep, full, ds, counts, **end)

    def sums(pair):
        return tuple(t.unflatten(2, (groups, heads // groups)).sum(3)
                     for t in pair)

    return {"q": sums(dq), "k": sums(dk), "v": dv, "initial_state": d0}


def operations(channels, dtype):
    """fp32 operations that bound what a linear attention's outputs are off by:
    sums over the channels and over 64 steps of a block, decays whose exponent is
    at most 88 and that come block by block; in 16 bits the rounding of q_t k_s and
    half a step of the second of the two values of a state, and the states' own."""
    least = channels + 320
    if dtype is torch.float32:
        return least
    return (state_operations(channels, dtype) +
            per_rounding(dtype) * (1.01 + ROUND[dtype]))


def state_operations(channels, dtype):
    """... and its states: of weighted values as sums of three values of bfloat16 or
    two of binary16, half a step of the last."""
    least = channels + 320
    if dtype is torch.float32:
        return least
    parts = 2 if dtype is torch.float16 else 3
    return least + 2 * per_rounding(dtype) * ROUND[dtype] ** (parts - 1)
