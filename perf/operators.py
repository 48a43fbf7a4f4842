"""Performance cases of the operators of a residual block over sequences.

  op = "matmul"      y = act(L R + bias) + residual and its gradients
                     (ops.matmul_bias_act, ops.matmul_bias_act_grad)
  op = "norm"        y = residual + scale * gate * norm(x), u = norm(y) and
                     their gradients (ops.residual_norm, ops.residual_norm_grad)
  op = "recurrence"  h_t = a_t h_{t-1} + b_t with gates from logits, and its
                     gradients (ops.linear_recurrence, ops.linear_recurrence_grad)

The ranges: products of 1 to 8192 rows, 64 to 4096 deep, 64 to 8192 columns;
norms of 1 to 32768 rows of 64 to 8192 channels; recurrences of 1 to 64
sequences, 1 to 32768 steps, 64 to 4096 channels; fp32, binary16 and bfloat16;
sizes that are no multiple of anything.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6


def _matmul(name, mode, dtype, m, k, n, activation, trans_b=False, bias=True,
            residual=False):
    return {"name": name, "op": "matmul", "mode": mode, "dtype": dtype, "m": m,
            "k": k, "n": n, "activation": activation, "trans_b": trans_b,
            "bias": bias, "residual": residual}


def _norm(name, mode, dtype, rows, channels, post, pre, gate, gate_rows=1,
          scale=True):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype,
            "rows": rows, "channels": channels, "post": post, "pre": pre,
            "gate": gate, "gate_rows": gate_rows, "scale": scale}


def _recurrence(name, mode, dtype, batch, steps, channels, input_gate,
                resets=False, ragged=False):
    return {"name": name, "op": "recurrence", "mode": mode, "dtype": dtype,
            "batch": batch, "steps": steps, "channels": channels,
            "input_gate": input_gate, "resets": resets, "ragged": ragged}


def listed():
    return [
        # One token through the widening layer of a feed-forward part: the
        # latency of serving, all of it the weights' way from memory.
        _matmul("matmul_token_bf16", "infer", "bf16", 1, 2048, 8192, "SILU"),
        # A serving batch through an output projection whose weights are
        # stored by feature, with the residual stream added.
        _matmul("matmul_batch_f16", "infer", "f16", 24, 4096, 4096, "NONE",
                trans_b=True, residual=True),
        # A product with no size that is a multiple of anything.
        _matmul("matmul_odd_f16", "infer", "f16", 4095, 1023, 1001, "GELU"),
        # An fp32 layer of the matmul sizes of the test-suite.
        _matmul("matmul_f32", "infer", "f32", 4096, 1024, 1024, "RELU"),
        # A training step's forward pass of a wide layer, which also keeps the
        # values in front of the activation.
        _matmul("matmul_train_bf16", "train", "bf16", 8192, 4096, 8192,
                "GELU_TANH"),
        # The gradients of such a layer.
        _matmul("matmul_grad_bf16", "grad", "bf16", 8192, 2048, 8192, "GELU"),
        # The norms between two blocks while a batch of eight decodes.
        _norm("norm_token_f32", "infer", "f32", 8, 4096, "RMS", "RMS", "NONE"),
        # The same in training, on eight sequences with a gate of their own.
        _norm("norm_train_bf16", "train", "bf16", 32768, 4096, "RMS", "RMS",
              "VALUE", 4096),
        # The gradients, with a gate for every token.
        _norm("norm_grad_bf16", "grad", "bf16", 16384, 2048, "RMS", "LAYER",
              "SILU", 1),
        # One token of 64 sequences that decode together.
        _recurrence("recurrence_token_f32", "infer", "f32", 64, 1, 4096, True),
        # A long document.
        _recurrence("recurrence_long_bf16", "infer", "bf16", 1, 32768, 2048,
                    False),
        # The gradients of a training batch of packed documents.
        _recurrence("recurrence_grad_f16", "grad", "f16", 4, 4096, 2048, True,
                    resets=True),
    ]


def _spread(rng, low, high):
    """A size between the two, even over its logarithm; half of them odd ones,
    the others multiples of the largest power of two up to 64 that fits."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    v = min(high, max(low, v))
    if rng.random() < 0.5:
        return min(high - 1, v | 1) if high > low + 1 else v
    step = 64
    while step > 1 and v < step:
        step //= 2
    return max(low, v // step * step)


def draw(rng):
    op = rng.choice(["matmul", "norm", "recurrence"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    mode = rng.choice(["infer", "train", "grad"] if op != "recurrence" else
                      ["infer", "grad"])
    if op == "matmul":
        c = _matmul(None, mode, dtype, _spread(rng, 1, 8192),
                    _spread(rng, 64, 4096), _spread(rng, 64, 8192),
                    rng.choice(["NONE", "RELU", "GELU", "GELU_TANH", "SILU"]),
                    rng.random() < 0.5, rng.random() < 0.75,
                    rng.random() < 0.5)
        # (two products each as large as the one of the largest listed case)
        if mode == "grad":
            c["m"] = max(1, c["m"] // 2)
    elif op == "norm":
        channels = _spread(rng, 64, 8192)
        rows = _spread(rng, 1, min(32768, (1 << 26) // channels))
        gate = rng.choice(["NONE", "VALUE", "SIGMOID", "SILU"])
        shared = rng.choice([1, rows]) if gate != "NONE" else 1
        c = _norm(None, mode, dtype, rows, channels,
                  rng.choice(["NONE", "RMS", "LAYER"]),
                  rng.choice(["RMS", "LAYER"]), gate, shared,
                  rng.random() < 0.5)
    else:
        channels = _spread(rng, 64, 4096)
        batch = _spread(rng, 1, 64)
        steps = _spread(rng, 1, min(32768, (1 << 25) // (channels * batch)))
        c = _recurrence(None, mode, dtype, batch, steps, channels,
                        rng.random() < 0.5, rng.random() < 0.5,
                        rng.random() < 0.5)
    del c["name"]
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, kind=dtype):
        x = torch.randn(shape, generator=g, device="cuda")
        return x.mul_(std).add_(mean).to(kind)

    s = dict(case)
    if case["op"] == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        s["lhs"] = normal(m, k)
        # (weights of variance 1 / k keep the activations' size)
        s["rhs"] = normal(*((n, k) if case["trans_b"] else (k, n)),
                          std=k ** -0.5)
        s["b"] = normal(n, std=0.1) if case["bias"] else None
        s["add"] = normal(m, n) if case["residual"] else None
        if case["mode"] == "grad":
            s["dy"] = normal(m, n)
            s["z"] = normal(m, n)
    elif case["op"] == "norm":
        rows, channels = case["rows"], case["channels"]
        groups = -(-rows // case["gate_rows"])
        s["x"] = normal(rows, channels)
        s["residual"] = normal(rows, channels, std=2.0)
        s["g"] = (normal(groups, channels, mean=0.5)
                  if case["gate"] != "NONE" else None)
        s["s"] = (normal(channels, mean=0.5, std=0.1)
                  if case["scale"] else None)
        s["post_w"] = (normal(channels, mean=1.0, std=0.1)
                       if case["post"] != "NONE" else None)
        s["post_b"] = (normal(channels, std=0.1)
                       if case["post"] == "LAYER" else None)
        s["pre_w"] = normal(channels, mean=1.0, std=0.1)
        s["pre_b"] = (normal(channels, std=0.1)
                      if case["pre"] == "LAYER" else None)
        if case["mode"] == "grad":
            s["dy"] = normal(rows, channels)
            s["du"] = normal(rows, channels)
            # (what the forward pass of the layer has left)
            s["y"], _, s["stats"] = _norm_forward(s)
            s["y"] = s["y"].to(dtype)
    else:
        batch, steps, channels = (case[v] for v in
                                  ("batch", "steps", "channels"))
        parts = 3 if case["input_gate"] else 2
        # (the gates and x are slices of what one projection has written)
        both = normal(batch, steps, parts * channels)
        both[..., channels:2 * channels] += 2.0
        s["x"], s["f"] = both[..., :channels], both[..., channels:2 * channels]
        s["i"] = both[..., 2 * channels:] if parts == 3 else None
        s["h0"] = normal(batch, channels, kind=torch.float32)
        s["reset"] = s["length"] = None
        if case["resets"]:
            # (documents of about 500 tokens)
            s["reset"] = (torch.rand(batch, steps, generator=g, device="cuda")
                          < 0.002).to(torch.uint8)
        if case["ragged"]:
            s["length"] = torch.randint(0, steps + 1, (batch,), generator=g,
                                        device="cuda", dtype=torch.int32)
        if case["mode"] == "grad":
            s["dh"] = normal(batch, steps, channels)
            s["dlast"] = normal(batch, channels, kind=torch.float32)
            s["h"] = _recurrence_forward(s)[0].to(dtype)
    return s


# ---- the plain forms ---------------------------------------------------------


def _act(z, kind):
    if kind == "RELU":
        return torch.clamp(z, min=0.0)
    if kind == "GELU":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if kind == "GELU_TANH":
        return 0.5 * z * (1.0 + torch.tanh(
            math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if kind == "SILU":
        return z * torch.sigmoid(z)
    return z


def _act_slope(z, kind):
    if kind == "RELU":
        return (z > 0).to(z.dtype)
    if kind == "GELU":
        return (0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) +
                z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi))
    if kind == "GELU_TANH":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return (0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c *
                (1.0 + 3.0 * 0.044715 * z * z))
    if kind == "SILU":
        sg = torch.sigmoid(z)
        return sg * (1.0 + z * (1.0 - sg))
    return torch.ones_like(z)


def _plain_matmul(s):
    dtype = s["lhs"].dtype
    lhs, rhs = s["lhs"].float(), s["rhs"].float()
    if s["trans_b"]:
        rhs = rhs.t()
    if s["mode"] == "grad":
        dz = s["dy"].float() * _act_slope(s["z"].float(), s["activation"])
        drhs = lhs.t() @ dz
        out = {"lhs": (dz @ rhs.t()).to(dtype),
               "rhs": (drhs.t() if s["trans_b"] else drhs).to(dtype)}
        if s["b"] is not None:
            out["bias"] = dz.sum(0).to(dtype)
        return out
    z = lhs @ rhs
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["activation"])
    if s["add"] is not None:
        y = y + s["add"].float()
    out = {"y": y.to(dtype)}
    if s["mode"] == "train":
        out["z"] = z.to(dtype)
    return out


def _statistics(v, kind):
    if kind == "NONE":
        return torch.zeros_like(v[:, :1]), torch.zeros_like(v[:, :1])
    if kind == "RMS":
        return (torch.zeros_like(v[:, :1]),
                torch.rsqrt((v * v).mean(1, keepdim=True) + _EPS))
    mean = v.mean(1, keepdim=True)
    c = v - mean
    return mean, torch.rsqrt((c * c).mean(1, keepdim=True) + _EPS)


def _normalised(v, mean, rstd, kind):
    return v if kind == "NONE" else (v - mean) * rstd


def _affine(v, w, b):
    if w is not None:
        v = v * w.float()
    return v if b is None else v + b.float()


def _gate(s):
    """The gate's factor and its slope, one row for each row of x."""
    if s["g"] is None:
        return None, None
    g = s["g"].float()
    if s["gate"] == "VALUE":
        v, d = g, torch.ones_like(g)
    else:
        sg = torch.sigmoid(g)
        if s["gate"] == "SIGMOID":
            v, d = sg, sg * (1.0 - sg)
        else:
            v, d = g * sg, sg * (1.0 + g * (1.0 - sg))
    if s["gate_rows"] > 1:
        rows = s["rows"]
        v = v.repeat_interleave(s["gate_rows"], 0)[:rows]
        d = d.repeat_interleave(s["gate_rows"], 0)[:rows]
    return v, d


def _norm_forward(s):
    x = s["x"].float()
    m0, r0 = _statistics(x, s["post"])
    y = _affine(_normalised(x, m0, r0, s["post"]), s["post_w"], s["post_b"])
    gate, _ = _gate(s)
    if gate is not None:
        y = y * gate
    if s["s"] is not None:
        y = y * s["s"].float()
    y = s["residual"].float() + y
    m1, r1 = _statistics(y, s["pre"])
    u = _affine(_normalised(y, m1, r1, s["pre"]), s["pre_w"], s["pre_b"])
    return y, u, torch.cat([m0, r0, m1, r1], 1)


def _through_norm(d, normalised, rstd, kind):
    """The gradient in front of a normalisation from the one behind it."""
    if kind == "NONE":
        return d
    d = d - normalised * (d * normalised).mean(1, keepdim=True) - (
        d.mean(1, keepdim=True) if kind == "LAYER" else 0.0)
    return d * rstd


def _plain_norm(s):
    dtype = s["x"].dtype
    if s["mode"] != "grad":
        y, u, stats = _norm_forward(s)
        out = {"y": y.to(dtype), "u": u.to(dtype)}
        if s["mode"] == "train":
            out["stats"] = stats
        return out
    m0, r0, m1, r1 = s["stats"].split(1, 1)
    du = s["du"].float()
    yn = _normalised(s["y"].float(), m1, r1, s["pre"])
    dy = s["dy"].float() + _through_norm(_affine(du, s["pre_w"], None), yn, r1,
                                         s["pre"])
    xn = _normalised(s["x"].float(), m0, r0, s["post"])
    n = _affine(xn, s["post_w"], s["post_b"])
    gate, slope = _gate(s)
    out = {"residual": dy.to(dtype), "pre_w": (du * yn).sum(0).to(dtype)}
    if s["pre_b"] is not None:
        out["pre_b"] = du.sum(0).to(dtype)
    dn = dy if gate is None else dy * gate
    if s["s"] is not None:
        out["s"] = (dn * n).sum(0).to(dtype)
        dn = dn * s["s"].float()
    if gate is not None:
        dg = _affine(dy * n * slope, s["s"], None)
        if s["gate_rows"] > 1:
            groups, each = s["g"].shape[0], s["gate_rows"]
            wide = dg.new_zeros(groups * each, dg.shape[1])
            wide[:dg.shape[0]] = dg
            dg = wide.view(groups, each, -1).sum(1)
        out["g"] = dg.to(dtype)
    if s["post_w"] is not None:
        out["post_w"] = (dn * xn).sum(0).to(dtype)
    if s["post_b"] is not None:
        out["post_b"] = dn.sum(0).to(dtype)
    out["x"] = _through_norm(_affine(dn, s["post_w"], None), xn, r0,
                             s["post"]).to(dtype)
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 by doubling: after the step of
    distance d, (a, b) of t stand for the steps t - 2 d + 1 ... t."""
    d = 1
    while d < a.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def _recurrence_gates(s):
    """Decay (zero at a reset, one behind a sequence's end), its slope, the
    input's factor and its slope, and the steps that count (None: all)."""
    a = torch.sigmoid(s["f"].float())
    da = a * (1.0 - a)
    if s["i"] is None:
        w, dw = torch.sigmoid(-s["f"].float()), None
    else:
        w = torch.sigmoid(s["i"].float())
        dw = w * (1.0 - w)
    keep = None
    if s["reset"] is not None:
        a = a.masked_fill(s["reset"].bool()[..., None], 0.0)
    if s["length"] is not None:
        steps = torch.arange(a.shape[1], device=a.device)
        keep = (steps[None] < s["length"][:, None])[..., None]
        a = a.masked_fill(~keep, 1.0)
    return a, da, w, dw, keep


def _recurrence_forward(s):
    a, _, w, _, keep = _recurrence_gates(s)
    b = w * s["x"].float()
    if keep is not None:
        b = b.masked_fill(~keep, 0.0)
    b[:, 0] += a[:, 0] * s["h0"]
    h = _scan(a, b)
    last = h[:, -1].clone()
    return (h if keep is None else h.masked_fill(~keep, 0.0)), last


def _plain_recurrence(s):
    dtype = s["x"].dtype
    if s["mode"] != "grad":
        h, last = _recurrence_forward(s)
        return {"h": h.to(dtype), "last": last}
    a, da, w, dw, keep = _recurrence_gates(s)
    dh = s["dh"].float()
    if keep is not None:
        dh = dh.masked_fill(~keep, 0.0)
    # G_t = dh_t + a_{t+1} G_{t+1}, the last state's gradient behind the end
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dlast"][:, None]], 1)
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    total = _scan(after.flip(1), dh.flip(1)).flip(1)
    out = {"h0": a[:, 0] * total[:, 0]}
    x = s["x"].float()
    before = torch.cat([s["h0"][:, None], s["h"].float()[:, :-1]], 1)
    if s["reset"] is not None:
        before = before.masked_fill(s["reset"].bool()[..., None], 0.0)
    if s["i"] is None:
        df = total * (before - x) * da
    else:
        df = total * before * da
    grads = {"x": total * w, "f": df}
    if s["i"] is not None:
        grads["i"] = total * x * dw
    for name, v in grads.items():
        out[name] = (v if keep is None else v.masked_fill(~keep, 0.0)).to(dtype)
    return out


# ---- the framework's operators -----------------------------------------------


def _own_matmul(s):
    from portdnn_amd import ops
    act = getattr(ops.ACTIVATION, s["activation"])
    if s["mode"] == "grad":
        got = ops.matmul_bias_act_grad(
            s["dy"], s["lhs"], s["rhs"], s["z"], activation=act,
            trans_b=s["trans_b"], bias=s["b"] is not None)
        out = {"lhs": got[0], "rhs": got[1]}
        if s["b"] is not None:
            out["bias"] = got[2]
        return out
    if s["mode"] == "train":
        y, z = ops.matmul_bias_act(
            s["lhs"], s["rhs"], bias=s["b"], residual=s["add"], activation=act,
            trans_b=s["trans_b"], keep_pre_activation=True)
        return {"y": y, "z": z}
    return {"y": ops.matmul_bias_act(
        s["lhs"], s["rhs"], bias=s["b"], residual=s["add"], activation=act,
        trans_b=s["trans_b"])}


def _own_norm(s):
    from portdnn_amd import ops
    kinds = {"post": getattr(ops.NORM, s["post"]),
             "pre": getattr(ops.NORM, s["pre"]),
             "gate_op": getattr(ops.GATE, s["gate"]),
             "gate_rows": s["gate_rows"], "eps": _EPS}
    if s["mode"] == "grad":
        got = ops.residual_norm_grad(
            s["x"], s["y"], s["stats"], grad_sum=s["dy"], grad_normed=s["du"],
            gate=s["g"], scale=s["s"], post_weight=s["post_w"],
            post_bias=s["post_b"], pre_weight=s["pre_w"], pre_bias=s["pre_b"],
            **kinds)
        names = {"x": "x", "residual": "residual", "gate": "g", "scale": "s",
                 "post_weight": "post_w", "post_bias": "post_b",
                 "pre_weight": "pre_w", "pre_bias": "pre_b"}
        return {names[k]: v for k, v in got.items()}
    y, u, stats = ops.residual_norm(
        s["x"], s["residual"], gate=s["g"], scale=s["s"],
        post_weight=s["post_w"], post_bias=s["post_b"], pre_weight=s["pre_w"],
        pre_bias=s["pre_b"], keep_stats=s["mode"] == "train", **kinds)
    out = {"y": y, "u": u}
    if stats is not None:
        out["stats"] = stats
    return out


def _own_recurrence(s):
    from portdnn_amd import ops
    if s["mode"] == "grad":
        got = ops.linear_recurrence_grad(
            s["dh"], s["x"], s["f"], s["h"], input_gate=s["i"],
            resets=s["reset"], lengths=s["length"], initial_state=s["h0"],
            grad_final_state=s["dlast"])
        names = {"x": "x", "forget": "f", "input_gate": "i",
                 "initial_state": "h0"}
        return {names[k]: v for k, v in got.items()}
    h, last = ops.linear_recurrence(
        s["x"], s["f"], input_gate=s["i"], resets=s["reset"],
        lengths=s["length"], initial_state=s["h0"])
    return {"h": h, "last": last}


def run(state):
    if own:
        return {"matmul": _own_matmul, "norm": _own_norm,
                "recurrence": _own_recurrence}[state["op"]](state)
    return {"matmul": _plain_matmul, "norm": _plain_norm,
            "recurrence": _plain_recurrence}[state["op"]](state)


def work(case):
    e = _SIZE[case["dtype"]]
    grad = case["mode"] == "grad"
    if case["op"] == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        matrices = m * k + k * n
        if grad:
            return {"bytes": e * (2 * matrices + 2 * m * n +
                                  n * case["bias"]),
                    "flops": 4 * m * k * n}
        outputs = m * n * (1 + case["residual"] + (case["mode"] == "train"))
        return {"bytes": e * (matrices + outputs + n * case["bias"]),
                "flops": 2 * m * k * n}
    if case["op"] == "norm":
        rows, channels = case["rows"], case["channels"]
        size = rows * channels
        gates = (-(-rows // case["gate_rows"]) * channels
                 if case["gate"] != "NONE" else 0)
        vectors = channels * (case["scale"] + (case["post"] != "NONE") +
                              (case["post"] == "LAYER") + 1 +
                              (case["pre"] == "LAYER"))
        if grad:
            return {"bytes": e * (6 * size + 2 * gates + 2 * vectors) +
                    16 * rows, "flops": 30 * size}
        return {"bytes": e * (4 * size + gates + vectors) +
                16 * rows * (case["mode"] == "train"), "flops": 12 * size}
    batch, steps, channels = (case[v] for v in ("batch", "steps", "channels"))
    size = batch * steps * channels
    gates = 1 + case["input_gate"]
    states = 4 * batch * channels
    if grad:
        # dh, x, h and the gates in, the gradients of x and the gates out
        return {"bytes": e * size * (4 + 2 * gates) + 3 * states,
                "flops": 14 * size}
    return {"bytes": e * size * (2 + gates) + 2 * states, "flops": 8 * size}


# ---- the definitions in 64 bits ------------------------------------------------


def _sigma(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _exact_matmul(s):
    lhs, dt = s["lhs"].double(), torch.float64
    rhs = (s["rhs"].mT if s["trans_b"] else s["rhs"]).to(dt)

    def both(z):
        """act(z) and act'(z) with respect to z."""
        kind = s["activation"]
        if kind == "NONE":
            return z, torch.ones_like(z)
        if kind == "RELU":
            on = z > 0
            return torch.where(on, z, 0.0), on.to(dt)
        if kind == "GELU":
            phi = 0.5 * torch.special.erfc(-z / 2.0 ** 0.5)
            return z * phi, phi + z * torch.exp(-z * z / 2.0) / (
                2.0 * math.pi) ** 0.5
        if kind == "SILU":
            g = _sigma(z)
            return z * g, g + z * g * _sigma(-z)
        # (1 + tanh(v)) / 2 = sigma(2 v)
        c = (8.0 / math.pi) ** 0.5
        g = _sigma(c * (z + 0.044715 * z ** 3))
        return z * g, g + z * g * (1.0 - g) * c * (1.0 + 0.134145 * z * z)

    if s["mode"] == "grad":
        dz = s["dy"].double() * both(s["z"].double())[1]
        drhs = torch.matmul(dz.mT, lhs) if s["trans_b"] else torch.matmul(
            lhs.mT, dz)
        out = {"lhs": torch.matmul(dz, rhs.mT), "rhs": drhs}
        if s["b"] is not None:
            out["bias"] = torch.sum(dz, 0)
        return out
    z = torch.matmul(lhs, rhs)
    if s["b"] is not None:
        z += s["b"].double()
    y = both(z)[0]
    out = {"y": y if s["add"] is None else y + s["add"].double()}
    if s["mode"] == "train":
        out["z"] = z
    return out


def _exact_norm(s):
    d = {k: v.double() if isinstance(v, torch.Tensor) else v
         for k, v in s.items()}
    rows, channels = s["rows"], s["channels"]
    one = torch.ones((), dtype=torch.float64, device=d["x"].device)
    gate = slope = one
    if d["g"] is not None:
        index = torch.arange(rows, device=one.device) // s["gate_rows"]
        v = d["g"][index]
        sg = _sigma(v)
        gate, slope = {"VALUE": (v, one), "SIGMOID": (sg, sg * _sigma(-v)),
                       "SILU": (v * sg, sg + v * sg * _sigma(-v))}[s["gate"]]
    scale = one if d["s"] is None else d["s"]
    post_w = one if d["post_w"] is None else d["post_w"]
    pre_w = d["pre_w"]

    def centred(v, mean, rstd, kind):
        return v if kind == "NONE" else (v - mean[:, None]) * rstd[:, None]

    def moments(v, kind):
        zero = torch.zeros(rows, dtype=torch.float64, device=v.device)
        if kind == "NONE":
            return zero, zero
        mean = v.sum(1) / channels if kind == "LAYER" else zero
        square = ((v - mean[:, None]) ** 2).sum(1) / channels
        return mean, (square + _EPS) ** -0.5

    if s["mode"] != "grad":
        m0, r0 = moments(d["x"], s["post"])
        n = centred(d["x"], m0, r0, s["post"]) * post_w
        if d["post_b"] is not None:
            n = n + d["post_b"]
        y = d["residual"] + scale * gate * n
        m1, r1 = moments(y, s["pre"])
        u = centred(y, m1, r1, s["pre"]) * pre_w
        out = {"y": y, "u": u if d["pre_b"] is None else u + d["pre_b"]}
        if s["mode"] == "train":
            out["stats"] = torch.stack([m0, r0, m1, r1], 1)
        return out

    def back(v, unit, rstd, kind):
        if kind == "NONE":
            return v
        along = (v * unit).sum(1, keepdim=True) / channels
        level = v.sum(1, keepdim=True) / channels if kind == "LAYER" else 0.0
        return rstd[:, None] * (v - level - along * unit)

    m0, r0, m1, r1 = d["stats"].unbind(1)
    yn = centred(d["y"], m1, r1, s["pre"])
    xn = centred(d["x"], m0, r0, s["post"])
    n = xn * post_w if d["post_b"] is None else xn * post_w + d["post_b"]
    dy = d["dy"] + back(d["du"] * pre_w, yn, r1, s["pre"])
    dn = dy * scale * gate
    out = {"residual": dy, "x": back(dn * post_w, xn, r0, s["post"]),
           "pre_w": (d["du"] * yn).sum(0)}
    if d["pre_b"] is not None:
        out["pre_b"] = d["du"].sum(0)
    if d["post_w"] is not None:
        out["post_w"] = (dn * xn).sum(0)
    if d["post_b"] is not None:
        out["post_b"] = dn.sum(0)
    if d["s"] is not None:
        out["s"] = (dy * gate * n).sum(0)
    if d["g"] is not None:
        out["g"] = torch.zeros_like(d["g"]).index_add_(
            0, index, dy * scale * n * slope)
    return out


def _exact_recurrence(s):
    """Step by step."""
    batch, steps = s["batch"], s["steps"]
    f, x = s["f"].double(), s["x"].double()
    keep, into = _sigma(f), _sigma(-f)
    dkeep, dinto = keep * into, None
    if s["i"] is not None:
        into = _sigma(s["i"].double())
        dinto = into * _sigma(-s["i"].double())
    fresh = (torch.zeros(batch, steps, 1, dtype=torch.bool, device=x.device)
             if s["reset"] is None else s["reset"][..., None] != 0)
    length = (torch.full((batch, 1), steps, device=x.device)
              if s["length"] is None else s["length"][:, None])
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    if s["mode"] != "grad":
        state, h = s["h0"].double(), torch.zeros_like(x)
        for t in range(steps):
            new = (torch.where(fresh[:, t], zero, keep[:, t] * state) +
                   into[:, t] * x[:, t])
            inside = length > t
            state = torch.where(inside, new, state)
            h[:, t] = torch.where(inside, new, zero)
        return {"h": h, "last": state}
    dh, h, total = s["dh"].double(), s["h"].double(), s["dlast"].double()
    out = {"x": torch.zeros_like(x), "f": torch.zeros_like(x)}
    if dinto is not None:
        out["i"] = torch.zeros_like(x)
    for t in range(steps - 1, -1, -1):
        inside = length > t
        g = total + dh[:, t]
        before = h[:, t - 1] if t else s["h0"].double()
        before = torch.where(fresh[:, t], zero, before)
        if dinto is None:
            df = g * (before - x[:, t]) * dkeep[:, t]
        else:
            df = g * before * dkeep[:, t]
            out["i"][:, t] = torch.where(inside, g * x[:, t] * dinto[:, t],
                                         zero)
        out["x"][:, t] = torch.where(inside, g * into[:, t], zero)
        out["f"][:, t] = torch.where(inside, df, zero)
        back = torch.where(fresh[:, t], zero, keep[:, t] * g)
        total = torch.where(inside, back, total)
    out["h0"] = total
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"matmul": _exact_matmul, "norm": _exact_norm,
            "recurrence": _exact_recurrence}[case["op"]](s)
