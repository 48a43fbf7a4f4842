"""Plain 64-bit implementations of the operators of a residual block over
sequences, each with a bound on the error of an implementation that holds its
sums, statistics and states in fp32 and rounds an output once.

Every function returns (value, magnitude) pairs: `magnitude` is what the value
would be if all its terms had one sign, so that a result of about `c` fp32
operations in a row is off by at most c * 2^-24 * magnitude, and by half a unit
in the last place of its type for the final rounding.
"""
import math

import torch

F32 = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
         torch.bfloat16: 2.0 ** -8}
# (half the distance of the smallest binary16 values)
LEAST = {torch.float32: 1e-37, torch.float16: 2.0 ** -25,
         torch.bfloat16: 1e-37}


def check(got, pair, operations, what=""):
    """got against (value, magnitude) of `operations` fp32 operations."""
    value, magnitude = pair
    dtype = got.dtype
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    bound = (ROUND[dtype] * value.abs() + LEAST[dtype] +
             (1.0 + ROUND[dtype]) * operations * F32 * magnitude)
    off = (got - value).abs()
    bad = ~(off <= bound)
    if bad.any():
        at = int(torch.argmax(torch.where(bad, off / bound, 0.0).nan_to_num(
            nan=1e30)))
        raise AssertionError("%s: %d of %d values, the worst at %d: %r for %r, "
                             "bound %g" % (what, int(bad.sum()), bad.numel(),
                                           at, got.flatten()[at].item(),
                                           value.flatten()[at].item(),
                                           bound.flatten()[at].item()))


def sigma(v):
    return 1.0 / (1.0 + torch.exp(-v))


# ---- act(L R + bias) + residual ----------------------------------------------

ACTIVATIONS = ["NONE", "RELU", "GELU", "GELU_TANH", "SILU"]


def activation(z, kind):
    if kind == "RELU":
        return torch.clamp(z, min=0.0)
    if kind == "GELU":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
    if kind == "GELU_TANH":
        return 0.5 * z * (1.0 + torch.tanh(
            math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
    if kind == "SILU":
        return z * sigma(z)
    return z


def slope(z, kind):
    z = z.detach().clone().requires_grad_()
    if kind == "NONE":
        return torch.ones_like(z)
    if kind == "RELU":
        return (z > 0).double()
    return torch.autograd.grad(activation(z, kind).sum(), z)[0]


def matmul(a, b, bias=None, residual=None, kind="NONE"):
    """(output, pre-activation) of double matrices."""
    z, mz = a @ b, a.abs() @ b.abs()
    if bias is not None:
        z, mz = z + bias, mz + bias.abs()
    # (the activations' slopes are below 1.13 and their values below |z|)
    y, my = activation(z, kind), 1.13 * mz + z.abs()
    if residual is not None:
        y, my = y + residual, my + residual.abs()
    return (y, my), (z, mz)


def matmul_grad(dy, a, b, z, kind, dtype):
    """Gradients of a, b and the bias; `dtype` is what the gradient of z is
    rounded to between, where there is an activation."""
    dz = dy * slope(z, kind)
    # (a slope's terms are below 1.5 (1 + |z|), whatever it comes to)
    mz = dy.abs() * (1.0 if kind in ("NONE", "RELU") else 1.5 * (1.0 + z.abs()))
    between = 0.0 if kind == "NONE" else ROUND[dtype] / F32
    extra = between * dz.abs() + 16.0 * mz  # in units of 2^-24

    def terms(x, y):  # magnitude in units of one operation
        return x @ y

    da = (dz @ b.t(), mz @ b.t().abs(), terms(extra, b.t().abs()))
    db = (a.t() @ dz, a.t().abs() @ mz, terms(a.t().abs(), extra))
    return da, db, (dz.sum(0), mz.sum(0))


# ---- norms around a block ------------------------------------------------------


def moments(v, kind, eps):
    rows = v.shape[0]
    if kind == "NONE":
        return torch.zeros(rows, 1).double(), torch.zeros(rows, 1).double()
    mean = v.mean(1, keepdim=True) if kind == "LAYER" else torch.zeros(
        rows, 1).double()
    return mean, ((v - mean).square().mean(1, keepdim=True) + eps).rsqrt()


def apply_norm(v, mv, kind, eps, weight, bias):
    """The norm of v (magnitude mv), its magnitude, mean and deviation."""
    mean, r = moments(v, kind, eps)
    if kind == "NONE":
        return v, mv, mean, r
    h = (v - mean) * r
    # an error e of v moves the mean by mean(e) and the deviation's logarithm by
    # mean(h e) r
    me = mv + mv.mean(1, keepdim=True) if kind == "LAYER" else mv
    mh = r * me + h.abs() * (1.0 + (h.abs() * me).mean(1, keepdim=True) * r)
    n, mn = h, mh
    if weight is not None:
        n, mn = n * weight, mn * weight.abs()
    if bias is not None:
        n, mn = n + bias, mn + bias.abs()
    return n, mn, mean, r


def gate_of(gate, kind, rows, gate_rows):
    """Value, slope and magnitude of the slope of the gate for every row."""
    if gate is None:
        one = torch.ones((), dtype=torch.float64)
        return one, one, one
    v = gate[torch.arange(rows) // gate_rows]
    s, rest = sigma(v), sigma(-v)
    if kind == "VALUE":
        return v, torch.ones_like(v), torch.ones_like(v)
    if kind == "SIGMOID":
        return s, s * rest, s * rest
    return v * s, s + v * s * rest, s + v.abs() * s * rest


def residual_norm(x, residual=None, gate=None, scale=None, post="NONE",
                  post_weight=None, post_bias=None, pre="NONE",
                  pre_weight=None, pre_bias=None, gate_op="VALUE", gate_rows=1,
                  eps=1e-6):
    """sum, normed (None without pre) and the four statistics."""
    n, mn, m0, r0 = apply_norm(x, x.abs(), post, eps, post_weight, post_bias)
    g = gate_of(gate, gate_op, x.shape[0], gate_rows)[0]
    s = torch.ones((), dtype=torch.float64) if scale is None else scale
    y, my = n * g * s, mn * (g * s).abs()
    if residual is not None:
        y, my = y + residual, my + residual.abs()
    u, mu, m1, r1 = apply_norm(y, my, pre, eps, pre_weight, pre_bias)
    stats = torch.cat([m0, r0, m1, r1], 1)
    return (y, my), (u, mu), stats


def residual_norm_grad(x, y, stats, dy=None, du=None, gate=None, scale=None,
                       post="NONE", post_weight=None, post_bias=None,
                       pre="NONE", pre_weight=None, pre_bias=None,
                       gate_op="VALUE", gate_rows=1, eps=1e-6):
    """A dict of (value, magnitude)."""
    rows = x.shape[0]
    one = torch.ones((), dtype=torch.float64)
    m0, r0, m1, r1 = stats.split(1, 1)
    w0 = one if post_weight is None else post_weight
    w1 = one if pre_weight is None else pre_weight
    s = one if scale is None else scale
    g, dg, mdg = gate_of(gate, gate_op, rows, gate_rows)

    def unit(v, mean, r, kind):
        if kind == "NONE":
            return v, v.abs()
        return (v - mean) * r, (v.abs() + mean.abs()) * r

    def through(v, mv, h, mh, r, kind):
        if kind == "NONE":
            return v, mv
        along, m_along = ((v * h).mean(1, keepdim=True),
                          (mv * mh).mean(1, keepdim=True))
        out, mag = v - h * along, mv + mh * m_along
        if kind == "LAYER":
            out = out - v.mean(1, keepdim=True)
            mag = mag + mv.mean(1, keepdim=True)
        return out * r, mag * r

    out = {}
    total = torch.zeros_like(x) if dy is None else dy
    m_total = total.abs()
    if du is not None:
        yh, myh = unit(y, m1, r1, pre)
        t, mt = through(du * w1, (du * w1).abs(), yh, myh, r1, pre)
        total, m_total = total + t, m_total + mt
        out["pre_weight"] = ((du * yh).sum(0), (du.abs() * myh).sum(0))
        out["pre_bias"] = (du.sum(0), du.abs().sum(0))
    out["residual"] = (total, m_total)
    xh, mxh = unit(x, m0, r0, post)
    n, mn = xh * w0, mxh * w0.abs()
    if post_bias is not None:
        n, mn = n + post_bias, mn + post_bias.abs()
    if gate is not None:
        each, m_each = total * s * n * dg, m_total * s.abs() * mn * mdg
        groups = gate.shape[0]
        index = torch.arange(rows) // gate_rows
        zero = torch.zeros(groups, x.shape[1], dtype=torch.float64)
        out["gate"] = (zero.index_add(0, index, each),
                       zero.index_add(0, index, m_each))
    dn, mdn = total * g, m_total * g.abs()
    out["scale"] = ((dn * n).sum(0), (mdn * mn).sum(0))
    dn, mdn = dn * s, mdn * s.abs()
    out["post_weight"] = ((dn * xh).sum(0), (mdn * mxh).sum(0))
    out["post_bias"] = (dn.sum(0), mdn.sum(0))
    out["x"] = through(dn * w0, mdn * w0.abs(), xh, mxh, r0, post)
    return out


# ---- the gated linear recurrence -------------------------------------------------


def _gates(f, i):
    a, rest = sigma(f), sigma(-f)
    if i is None:
        return a, rest, rest, None
    return a, rest, sigma(i), sigma(-i)


def recurrence(x, f, i=None, resets=None, lengths=None, h0=None):
    """((h, magnitude), (last state, magnitude)): a step adds an error of a few
    roundings of its terms to a times the error of the one before, so that the
    magnitude is a recurrence of its own."""
    batch, steps, channels = x.shape
    a, _, w, _ = _gates(f, i)
    state = torch.zeros(batch, channels).double() if h0 is None else h0
    size, error = state.abs(), state.abs()
    h, mh = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(steps):
        inside = torch.ones(batch, 1, dtype=torch.bool)
        if lengths is not None:
            inside = (t < lengths)[:, None]
        keep = a[:, t]
        if resets is not None:
            keep = torch.where(resets[:, t, None] != 0, 0.0, keep)
        kept = torch.where(keep == 0, 0.0, keep * state)
        add = torch.where(inside, w[:, t] * x[:, t], 0.0)
        new = kept + add
        new_size = torch.where(keep == 0, 0.0, keep * size) + add.abs()
        new_error = torch.where(keep == 0, 0.0, keep * error) + new_size
        state = torch.where(inside, new, state)
        size = torch.where(inside, new_size, size)
        error = torch.where(inside, new_error, error)
        h[:, t] = torch.where(inside, new, 0.0)
        mh[:, t] = torch.where(inside, new_error, 0.0)
    return (h, mh), (state, error)


def recurrence_grad(dh, x, f, h, i=None, resets=None, lengths=None, h0=None,
                    d_last=None):
    batch, steps, channels = x.shape
    a, rest, w, w_rest = _gates(f, i)
    zero = torch.zeros(batch, channels).double()
    D = zero if d_last is None else d_last
    size, error = D.abs(), D.abs()
    names = ["x", "forget"] + (["input_gate"] if i is not None else [])
    out = {n: (torch.zeros_like(x), torch.zeros_like(x)) for n in names}
    for t in range(steps - 1, -1, -1):
        inside = torch.ones(batch, 1, dtype=torch.bool)
        if lengths is not None:
            inside = (t < lengths)[:, None]
        fresh = torch.zeros(batch, 1, dtype=torch.bool)
        if resets is not None:
            fresh = resets[:, t, None] != 0
        G = dh[:, t] + D
        m = dh[:, t].abs() + size + error
        before = h[:, t - 1] if t else (zero if h0 is None else h0)
        before = torch.where(fresh, 0.0, before)
        other = 0.0 if i is not None else x[:, t]
        parts = {"x": (G * w[:, t], m * w[:, t]),
                 "forget": (G * (before - other) * a[:, t] * rest[:, t],
                            m * (before.abs() + abs(other)) * a[:, t] *
                            rest[:, t])}
        if i is not None:
            parts["input_gate"] = (G * x[:, t] * w[:, t] * w_rest[:, t],
                                   m * x[:, t].abs() * w[:, t] * w_rest[:, t])
        for n, (v, mv) in parts.items():
            out[n][0][:, t] = torch.where(inside, v, 0.0)
            out[n][1][:, t] = torch.where(inside, mv, 0.0)
        keep = torch.where(fresh, 0.0, a[:, t])
        new = keep * G
        new_size = keep * (dh[:, t].abs() + size)
        new_error = keep * error + new_size
        D = torch.where(inside, new, D)
        size = torch.where(inside, new_size, size)
        error = torch.where(inside, new_error, error)
    out["initial_state"] = (D, error)
    return out
