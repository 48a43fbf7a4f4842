"""The references of a linear-attention block against automatic differentiation
and against differences."""
import pytest
import torch

import attention_reference as plain
import sequence_reference as ref


def _normal(g, *shape):
    return torch.randn(shape, generator=g, dtype=torch.float64)


def _simple(q, k, v, decay, resets, lengths, s0, scale):
    """Step by step, each sequence and head by itself."""
    batch, steps, heads, _ = v.shape
    share = heads // q.shape[2]
    out = torch.zeros_like(v)
    last = torch.empty_like(s0)
    outs, lasts = [], []
    for b in range(batch):
        for h in range(heads):
            s, rows = s0[b, h], []
            for t in range(steps):
                if t >= int(lengths[b]):
                    rows.append(out[b, t, h])
                    continue
                s = 0 * s if resets[b, t] else decay[h].exp() * s
                s = s + torch.outer(k[b, t, h // share], v[b, t, h])
                rows.append(scale * q[b, t, h // share] @ s)
            outs.append(torch.stack(rows))
            lasts.append(s)
    return (torch.stack(outs).view(batch, heads, steps, -1).transpose(1, 2),
            torch.stack(lasts).view(last.shape))


@pytest.mark.parametrize("heads,groups", [(2, 2), (4, 2)])
def test_attention(heads, groups):
    g = torch.Generator().manual_seed(heads)
    batch, steps, keys, values = 3, 9, 3, 2
    t = [_normal(g, batch, steps, groups, keys),
         _normal(g, batch, steps, groups, keys),
         _normal(g, batch, steps, heads, values),
         _normal(g, batch, heads, keys, values)]
    decay = -_normal(g, heads).abs()
    resets = (torch.rand(batch, steps, generator=g) < 0.2).to(torch.uint8)
    resets[0, 0] = 1
    lengths = torch.tensor([9, 0, 5])
    do, ds = _normal(g, batch, steps, heads, values), _normal(
        g, batch, heads, keys, values)

    def loss(q, k, v, s0):
        o, last = _simple(q, k, v, decay, resets, lengths, s0, 0.7)
        return (o * do).sum() + (last * ds).sum()

    for x in t:
        x.requires_grad_()
    o, last = _simple(*t[:3], decay, resets, lengths, t[3], 0.7)
    got = plain.attention(*[x.detach() for x in t[:3]], decay, resets, lengths,
                          t[3].detach(), 0.7)
    torch.testing.assert_close(got[0][0], o.detach())
    torch.testing.assert_close(got[1][0], last.detach())
    assert (got[0][1] >= got[0][0].abs() - 1e-12).all()
    want = torch.autograd.grad(loss(*t), t)
    d = plain.attention_grad(do, *[x.detach() for x in t[:3]], decay, resets,
                             lengths, t[3].detach(), ds, 0.7)
    for name, w in zip(("q", "k", "v", "initial_state"), want):
        torch.testing.assert_close(d[name][0], w)
        assert (d[name][1] >= w.abs() - 1e-12).all()
    # linear in each operand: differences are exact
    with torch.no_grad():
        for i, name in enumerate(("q", "k", "v", "initial_state")):
            e = _normal(g, *t[i].shape)
            up, down = list(t), list(t)
            up[i], down[i] = t[i] + e, t[i] - e
            torch.testing.assert_close(
                0.5 * (loss(*up) - loss(*down)), (d[name][0] * e).sum())


@pytest.mark.parametrize("kind", ref.ACTIVATIONS)
def test_gated(kind):
    g = torch.Generator().manual_seed(1)
    t = [_normal(g, *s).requires_grad_()
         for s in ((4, 3), (3, 5), (3, 5), (5,), (5,))]
    dy = _normal(g, 4, 5)

    def f(x, a, b, c, d):
        return (ref.activation(x @ a + c, kind) * (x @ b + d) * dy).sum()

    assert torch.autograd.gradcheck(f, t)
    want = torch.autograd.grad(f(*t), t)
    (out, size), (z, _), (u, _) = plain.gated(*[x.detach() for x in t], kind)
    torch.testing.assert_close((out * dy).sum(), f(*t).detach())
    got = plain.gated_grad(dy, *[x.detach() for x in t[:3]], z, u, kind)
    for w, (value, magnitude) in zip(want, got.values()):
        torch.testing.assert_close(value, w)
        assert (magnitude >= w.abs() - 1e-12).all()


@pytest.mark.parametrize("halves", [True, False])
def test_rotary(halves):
    g = torch.Generator().manual_seed(2)
    x = _normal(g, 2, 5, 3, 10).requires_grad_()
    f = plain.frequencies(6)
    at = torch.tensor([[0, 1, 2, 3, 4], [-7, 100, 0, 9, 2 ** 30]])
    dy = _normal(g, 2, 5, 3, 10)
    y, size = plain.rotary(x.detach(), f, at, halves, 1.3)
    # (differences in one direction, which a linear map has exactly)
    e = _normal(g, *x.shape)
    up, _ = plain.rotary(x.detach() + e, f, at, halves, 1.3)
    dx, _ = plain.rotary(dy, f, at, halves, 1.3, inverse=True)
    turned = dx[..., :6] * e[..., :6]
    torch.testing.assert_close(turned.sum(),
                               ((up - y) * dy)[..., :6].sum())
    back, _ = plain.rotary(y, f, at, halves, 1 / 1.3, inverse=True)
    torch.testing.assert_close(back, x.detach())
    assert (size >= y.abs() - 1e-12).all()
