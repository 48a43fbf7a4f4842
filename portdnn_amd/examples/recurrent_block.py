"""A recurrent language-model block of the operators for sequences: training on
whole sequences and answering token by token with a state of fixed size.

With the residual stream s, [batch * steps, width]:

  u = rms(s)                                 residual_norm (its pre_norm)
  x, f, i, g = u W_in + b_in                 matmul_bias_act
  h_t = sig(f_t) h_{t-1} + sig(i_t) x_t      linear_recurrence, on slices
  y = silu(g) rms(h)                         residual_norm (post_norm and gate)
  o = y W_out                                matmul_bias_act
  s2 = s + scale o,  v = rms(s2)             residual_norm
  s' = s2 + gelu(v W_up + b_up) W_down       matmul_bias_act twice

A token is a call with one step, which updates the state in place; a prompt is a
call with its steps, which leaves the state behind the last of them.

    python -m portdnn_amd.examples.recurrent_block
"""
import torch

from portdnn_amd import ops
from portdnn_amd.ops import ACTIVATION, GATE, NORM


class RecurrentBlock:
    """The block's weights by name (`weights`), its forward pass and gradients.

    width: channels of the residual stream; inner: of the recurrence; hidden: of
    the layers behind it."""

    def __init__(self, width, inner, hidden, dtype=torch.bfloat16,
                 device="cuda", generator=None):
        def normal(rows, cols):
            w = torch.randn(rows, cols, generator=generator) * rows ** -0.5
            return w.to(device, dtype)

        def constant(n, value):
            return torch.full((n,), value, dtype=dtype, device=device)

        self.width, self.inner, self.dtype = width, inner, dtype
        bias = torch.zeros(4 * inner)
        bias[inner:2 * inner] = 2.0  # states that last some steps
        self.weights = {
            "norm_in": constant(width, 1.0),
            "w_in": normal(width, 4 * inner),
            "b_in": bias.to(device, dtype),
            "norm_inner": constant(inner, 1.0),
            "w_out": normal(inner, width),
            "scale": constant(width, 0.5),
            "norm_hidden": constant(width, 1.0),
            "w_up": normal(width, hidden),
            "b_up": constant(hidden, 0.0),
            "w_down": normal(hidden, width),
        }

    def state(self, batch):
        """The state in front of a sequence."""
        return torch.zeros(batch, self.inner,
                           device=self.weights["w_in"].device)

    def _slices(self, p, batch, steps):
        """x, forget and input gate as sequences, and the gate's rows."""
        n = self.inner
        rows = p.view(batch, steps, 4 * n)
        return ([rows[..., k * n:(k + 1) * n] for k in range(3)],
                p[:, 3 * n:])

    def forward(self, s, batch, steps, state=None, resets=None, lengths=None,
                keep=False):
        """The stream behind the block.  `state` is updated in place; with
        `keep` returns (stream, what `backward` takes)."""
        w = self.weights
        _, u, stats_in = ops.residual_norm(
            s, pre=NORM.RMS, pre_weight=w["norm_in"], keep_sum=False,
            keep_stats=keep)
        p = ops.matmul_bias_act(u, w["w_in"], bias=w["b_in"])
        (x, f, i), g = self._slices(p, batch, steps)
        # (the gradients read the state in front, which this call overwrites)
        initial = state.clone() if keep and state is not None else state
        h, _ = ops.linear_recurrence(x, f, i, resets=resets, lengths=lengths,
                                     initial_state=state, final_state=state)
        rows = h.view(batch * steps, self.inner)
        y, _, stats_inner = ops.residual_norm(
            rows, gate=g, gate_op=GATE.SILU, post=NORM.RMS,
            post_weight=w["norm_inner"], keep_stats=keep)
        o = ops.matmul_bias_act(y, w["w_out"])
        s2, v, stats_hidden = ops.residual_norm(
            o, residual=s, scale=w["scale"], pre=NORM.RMS,
            pre_weight=w["norm_hidden"], keep_stats=keep)
        m = ops.matmul_bias_act(v, w["w_up"], bias=w["b_up"],
                                activation=ACTIVATION.GELU_TANH,
                                keep_pre_activation=keep)
        m, z = m if keep else (m, None)
        out = ops.matmul_bias_act(m, w["w_down"], residual=s2)
        if not keep:
            return out
        return out, dict(s=s, u=u, p=p, h=h, y=y, o=o, s2=s2, v=v, m=m, z=z,
                         stats_in=stats_in, stats_inner=stats_inner,
                         stats_hidden=stats_hidden, initial=initial,
                         resets=resets, lengths=lengths, batch=batch,
                         steps=steps)

    def backward(self, grad, kept):
        """The gradients of the stream in front of the block and, by name, of
        the weights."""
        w, n, got = self.weights, self.inner, {}
        batch, steps = kept["batch"], kept["steps"]
        dm, got["w_down"], _ = ops.matmul_bias_act_grad(
            grad, kept["m"], w["w_down"], bias=False)
        dv, got["w_up"], got["b_up"] = ops.matmul_bias_act_grad(
            dm, kept["v"], w["w_up"], pre_activation=kept["z"],
            activation=ACTIVATION.GELU_TANH)
        d = ops.residual_norm_grad(
            kept["o"], kept["s2"], kept["stats_hidden"], grad_sum=grad,
            grad_normed=dv, scale=w["scale"], pre=NORM.RMS,
            pre_weight=w["norm_hidden"])
        got["scale"], got["norm_hidden"] = d["scale"], d["pre_weight"]
        ds = d["residual"]
        dy, got["w_out"], _ = ops.matmul_bias_act_grad(
            d["x"], kept["y"], w["w_out"], bias=False)
        (x, f, i), g = self._slices(kept["p"], batch, steps)
        d = ops.residual_norm_grad(
            kept["h"].view(batch * steps, n), kept["y"], kept["stats_inner"],
            grad_sum=dy, gate=g, gate_op=GATE.SILU, post=NORM.RMS,
            post_weight=w["norm_inner"])
        got["norm_inner"] = d["post_weight"]
        # the projection's gradient: three slices by the recurrence, the gate's
        dp = torch.empty_like(kept["p"])
        dp[:, 3 * n:] = d["gate"]
        ops.linear_recurrence_grad(
            d["x"].view(batch, steps, n), x, f, kept["h"], input_gate=i,
            resets=kept["resets"], lengths=kept["lengths"],
            initial_state=kept["initial"],
            out=dp.view(batch, steps, 4 * n)[..., :3 * n])
        du, got["w_in"], got["b_in"] = ops.matmul_bias_act_grad(
            dp, kept["u"], w["w_in"])
        d = ops.residual_norm_grad(
            kept["s"], kept["s"], kept["stats_in"], grad_sum=ds, grad_normed=du,
            pre=NORM.RMS, pre_weight=w["norm_in"])
        got["norm_in"] = d["pre_weight"]
        return d["x"], got


def train(blocks, inputs, targets, batch, steps, rate, resets=None):
    """One step of gradient descent on the mean square error between the
    stream behind the blocks and `targets`; the error before the step."""
    s, kept = inputs, []
    for block in blocks:
        s, k = block.forward(s, batch, steps, resets=resets, keep=True)
        kept.append(k)
    error = s.float() - targets.float()
    grad = (error * (2.0 / error.numel())).to(s.dtype)
    for block, k in zip(reversed(blocks), reversed(kept)):
        grad, got = block.backward(grad, k)
        for name, g in got.items():
            block.weights[name].sub_(g, alpha=rate)
    return error.square().mean()


def answer(blocks, states, token):
    """One token of every sequence through the blocks."""
    for block, state in zip(blocks, states):
        token = block.forward(token, token.shape[0], 1, state=state)
    return token


def main(width=512, inner=768, hidden=1024, depth=2, batch=8, steps=256,
         updates=20, rate=1.0, seed=0):
    rng = torch.Generator().manual_seed(seed)
    blocks = [RecurrentBlock(width, inner, hidden, torch.float32,
                             generator=rng) for _ in range(depth)]
    # a stream to be delayed by one step
    signal = torch.randn(batch, steps + 1, width, generator=rng).cuda()
    inputs = signal[:, 1:].reshape(-1, width).contiguous()
    targets = signal[:, :-1].reshape(-1, width).contiguous()
    errors = [train(blocks, inputs, targets, batch, steps, rate).item()
              for _ in range(updates)]
    print("error %.4f -> %.4f in %d steps" % (errors[0], errors[-1], updates))
    whole = inputs
    for block in blocks:
        whole = block.forward(whole, batch, steps)
    whole = whole.view(batch, steps, width)
    states = [block.state(batch) for block in blocks]
    tokens = inputs.view(batch, steps, width)
    got = torch.stack([answer(blocks, states, tokens[:, t].contiguous())
                       for t in range(steps)], 1)
    apart = (got - whole).abs().max().item()
    print("token by token, apart by at most %.2e" % apart)
    return errors, apart


if __name__ == "__main__":
    main()
