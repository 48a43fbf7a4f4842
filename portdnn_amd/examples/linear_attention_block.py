"""A language-model block of linear attention and a gated feed-forward part:
training on whole sequences and answering token by token with a state of fixed
size.

With the residual stream s, [batch * steps, width]:

  u = rms(s)                                   residual_norm (its pre_norm)
  q, k, v, g = u W_in                          matmul_bias_act
  q, k = rotated(q), rotated(k)                rotary, in place on slices
  h = linear_attention(q, k, v)                linear_attention, on slices
  y = silu(g) rms(h)                           residual_norm (post_norm and gate)
  s2 = s + y W_out                             matmul_bias_act
  z = rms(s2)                                  residual_norm
  m = silu(z W_gate) * (z W_up)                gated_matmul
  s' = s2 + m W_down                           matmul_bias_act

A token is a call with one step, which updates the state in place; a prompt is a
call with its steps, which leaves the state behind the last of them.

    python -m portdnn_amd.examples.linear_attention_block
"""
import torch

from portdnn_amd import ops
from portdnn_amd.ops import GATE, NORM


class LinearAttentionBlock:
    """The block's weights by name (`weights`), its forward pass and gradients.

    width: channels of the residual stream; heads of `channels` queries, keys and
    values, key_heads of queries and keys; hidden: of the gated part."""

    def __init__(self, width, heads, key_heads, channels, hidden,
                 dtype=torch.bfloat16, device="cuda", generator=None):
        def normal(rows, cols):
            w = torch.randn(rows, cols, generator=generator) * rows ** -0.5
            return w.to(device, dtype)

        def ones(n):
            return torch.ones(n, dtype=dtype, device=device)

        self.width, self.dtype = width, dtype
        self.heads, self.key_heads, self.channels = heads, key_heads, channels
        self.scale = channels ** -0.5
        # heads that forget within some steps to heads that last for hundreds
        self.decay = torch.log1p(
            -(2.0 ** -torch.linspace(2.0, 8.0, heads))).to(device)
        self.frequencies = ops.rotary_frequencies(
            channels // 2 * 2, device=device)
        inner, shared = heads * channels, key_heads * channels
        self.weights = {
            "norm_in": ones(width),
            "w_in": normal(width, 2 * shared + 2 * inner),
            "norm_inner": ones(inner),
            "w_out": normal(inner, width),
            "norm_hidden": ones(width),
            "w_gate": normal(width, hidden),
            "w_up": normal(width, hidden),
            "w_down": normal(hidden, width),
        }

    def state(self, batch):
        """The state in front of a sequence."""
        return torch.zeros(batch, self.heads, self.channels, self.channels,
                           device=self.decay.device)

    def _slices(self, p, batch, steps):
        """q, k and v as sequences of heads, and the gate's rows."""
        n, m = self.key_heads * self.channels, self.heads * self.channels
        rows = p.view(batch, steps, -1)
        return (rows[..., :n].unflatten(2, (self.key_heads, -1)),
                rows[..., n:2 * n].unflatten(2, (self.key_heads, -1)),
                rows[..., 2 * n:2 * n + m].unflatten(2, (self.heads, -1)),
                p[:, 2 * n + m:])

    def _rotate(self, t, positions, inverse=False):
        ops.rotary(t, self.frequencies, positions=positions, inverse=inverse,
                   out=t)

    def forward(self, s, batch, steps, state=None, positions=None, resets=None,
                lengths=None, keep=False):
        """The stream behind the block.  `state` is updated in place; positions:
        those of the sequences' first steps, an int32 [batch] tensor (zero); with
        `keep` returns (stream, what `backward` takes)."""
        w = self.weights
        _, u, stats_in = ops.residual_norm(
            s, pre=NORM.RMS, pre_weight=w["norm_in"], keep_sum=False,
            keep_stats=keep)
        p = ops.matmul_bias_act(u, w["w_in"])
        q, k, v, g = self._slices(p, batch, steps)
        self._rotate(q, positions)
        self._rotate(k, positions)
        # (the gradients read the state in front, which this call overwrites)
        initial = state.clone() if keep and state is not None else state
        h, _ = ops.linear_attention(
            q, k, v, self.decay, resets=resets, lengths=lengths,
            initial_state=state, final_state=state, scale=self.scale)
        rows = h.view(batch * steps, -1)
        y, _, stats_inner = ops.residual_norm(
            rows, gate=g, gate_op=GATE.SILU, post=NORM.RMS,
            post_weight=w["norm_inner"], keep_stats=keep)
        s2 = ops.matmul_bias_act(y, w["w_out"], residual=s)
        _, z, stats_hidden = ops.residual_norm(
            s2, pre=NORM.RMS, pre_weight=w["norm_hidden"], keep_sum=False,
            keep_stats=keep)
        m = ops.gated_matmul(z, w["w_gate"], w["w_up"], keep_pre_activation=keep)
        m, gate, up = m if keep else (m, None, None)
        out = ops.matmul_bias_act(m, w["w_down"], residual=s2)
        if not keep:
            return out
        return out, dict(s=s, u=u, p=p, h=h, y=y, s2=s2, z=z, m=m, gate=gate,
                         up=up, stats_in=stats_in, stats_inner=stats_inner,
                         stats_hidden=stats_hidden, initial=initial,
                         positions=positions, resets=resets, lengths=lengths,
                         batch=batch, steps=steps)

    def backward(self, grad, kept):
        """The gradients of the stream in front of the block and, by name, of
        the weights."""
        w, got = self.weights, {}
        batch, steps = kept["batch"], kept["steps"]
        dm, got["w_down"], _ = ops.matmul_bias_act_grad(
            grad, kept["m"], w["w_down"], bias=False)
        dz, got["w_gate"], got["w_up"], _, _ = ops.gated_matmul_grad(
            dm, kept["z"], w["w_gate"], w["w_up"], kept["gate"], kept["up"],
            bias=False)
        d = ops.residual_norm_grad(
            kept["s2"], kept["s2"], kept["stats_hidden"], grad_sum=grad,
            grad_normed=dz, pre=NORM.RMS, pre_weight=w["norm_hidden"])
        got["norm_hidden"] = d["pre_weight"]
        ds = d["x"]
        dy, got["w_out"], _ = ops.matmul_bias_act_grad(
            ds, kept["y"], w["w_out"], bias=False)
        q, k, v, g = self._slices(kept["p"], batch, steps)
        d = ops.residual_norm_grad(
            kept["h"].view(batch * steps, -1), kept["y"], kept["stats_inner"],
            grad_sum=dy, gate=g, gate_op=GATE.SILU, post=NORM.RMS,
            post_weight=w["norm_inner"])
        got["norm_inner"] = d["post_weight"]
        # the projection's gradient: three slices by the attention, the gate's
        dp = torch.empty_like(kept["p"])
        dq, dk, _, dg = self._slices(dp, batch, steps)
        dg.copy_(d["gate"])
        ops.linear_attention_grad(
            d["x"].view(v.shape), q, k, v, self.decay, resets=kept["resets"],
            lengths=kept["lengths"], initial_state=kept["initial"],
            scale=self.scale,
            out=dp.view(batch, steps, -1)[..., :dp.shape[1] - dg.shape[1]])
        self._rotate(dq, kept["positions"], inverse=True)
        self._rotate(dk, kept["positions"], inverse=True)
        du, got["w_in"], _ = ops.matmul_bias_act_grad(
            dp, kept["u"], w["w_in"], bias=False)
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


def answer(blocks, states, token, positions):
    """One token of every sequence through the blocks."""
    for block, state in zip(blocks, states):
        token = block.forward(token, token.shape[0], 1, state=state,
                              positions=positions)
    return token


def main(width=512, heads=8, key_heads=4, channels=64, hidden=1024, depth=2,
         batch=8, steps=256, updates=20, rate=1.0, seed=0):
    rng = torch.Generator().manual_seed(seed)
    blocks = [LinearAttentionBlock(width, heads, key_heads, channels, hidden,
                                   torch.float32, generator=rng)
              for _ in range(depth)]
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
    at = torch.zeros(batch, dtype=torch.int32, device="cuda")
    got = []
    for t in range(steps):
        got.append(answer(blocks, states, tokens[:, t].contiguous(), at))
        at += 1
    apart = (torch.stack(got, 1) - whole).abs().max().item()
    print("token by token, apart by at most %.2e" % apart)
    return errors, apart


if __name__ == "__main__":
    main()
