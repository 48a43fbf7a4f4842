"""Performance cases of a linear-attention block's operators.

  op = "gated"     h = act(x W_gate + b_gate) * (x W_up + b_up) and its gradients
                   (ops.gated_matmul, ops.gated_matmul_grad)
  op = "rotary"    pairs of a head's channels turned by an angle that grows with
                   the position (ops.rotary)
  op = "attention" S_t = a S_{t-1} + k_t^T v_t, o_t = scale q_t S_t with a decay
                   a for each head, and its gradients (ops.linear_attention,
                   ops.linear_attention_grad)

The ranges: products of 1 to 8192 rows, 64 to 4096 deep, 64 to 8192 columns;
heads of 16 to 256 channels, 1 to 64 of them; 1 to 64 sequences of 1 to 32768
steps; fp32, binary16 and bfloat16; sizes that are no multiple of anything.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _gated(name, mode, dtype, m, k, n, activation, trans_b=False, bias=False):
    return {"name": name, "op": "gated", "mode": mode, "dtype": dtype, "m": m,
            "k": k, "n": n, "activation": activation, "trans_b": trans_b,
            "bias": bias}


def _rotary(name, mode, dtype, batch, steps, heads, channels, turned, layout,
            positions, scaling="NONE"):
    return {"name": name, "op": "rotary", "mode": mode, "dtype": dtype,
            "batch": batch, "steps": steps, "heads": heads,
            "channels": channels, "turned": turned, "layout": layout,
            "positions": positions, "scaling": scaling}


def _attention(name, mode, dtype, batch, steps, heads, key_heads, keys, values,
               resets=False, ragged=False):
    return {"name": name, "op": "attention", "mode": mode, "dtype": dtype,
            "batch": batch, "steps": steps, "heads": heads,
            "key_heads": key_heads, "keys": keys, "values": values,
            "resets": resets, "ragged": ragged}


def listed():
    return [
        # One token through a feed-forward part: the latency of serving, all of
        # it the two weights' way from memory.
        _gated("gated_token_bf16", "infer", "bf16", 1, 2048, 8192, "SILU"),
        # A serving batch, with weights that are stored by feature.
        _gated("gated_batch_f16", "infer", "f16", 32, 4096, 8192, "SILU",
               trans_b=True),
        # A product with no size that is a multiple of anything.
        _gated("gated_odd_f32", "infer", "f32", 1001, 1023, 515, "GELU",
               bias=True),
        # A training step's forward pass, which keeps both projections.
        _gated("gated_train_bf16", "train", "bf16", 8192, 2048, 8192, "SILU"),
        # The gradients of such a layer, with biases.
        _gated("gated_grad_bf16", "grad", "bf16", 4096, 2048, 8192, "GELU_TANH",
               bias=True),
        # Queries and keys of a token of sixteen sequences, each at a place of
        # its own.
        _rotary("rotary_token_bf16", "infer", "bf16", 16, 1, 40, 128, 128,
                "HALVES", "FIRST"),
        # A training batch.
        _rotary("rotary_train_bf16", "infer", "bf16", 4, 4096, 32, 128, 128,
                "HALVES", "NONE"),
        # The gradients of packed long documents: neighbouring channels, a part
        # of the head, positions of their own, frequencies for long contexts.
        _rotary("rotary_grad_f32", "grad", "f32", 2, 5001, 12, 100, 64,
                "PAIRS", "EACH", "BANDS"),
        # One token of 64 sequences that decode together.
        _attention("attention_token_bf16", "infer", "bf16", 64, 1, 16, 16, 128,
                   128),
        # A long prompt.
        _attention("attention_long_bf16", "infer", "bf16", 1, 32768, 16, 16,
                   128, 128),
        # Prompts of many lengths, keys shared by three heads, odd sizes.
        _attention("attention_odd_f16", "infer", "f16", 3, 1000, 6, 2, 72, 100,
                   resets=True, ragged=True),
        # The gradients of a training batch of packed documents.
        _attention("attention_grad_bf16", "grad", "bf16", 4, 4096, 16, 16, 128,
                   128, resets=True),
    ]


def _spread(rng, low, high, step=64):
    """A size between the two, even over its logarithm; half of them odd ones,
    the others multiples of the largest power of two up to `step` that fits."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    v = min(high, max(low, v))
    if rng.random() < 0.5:
        return min(high - 1, v | 1) if high > low + 1 else v
    while step > 1 and v < step:
        step //= 2
    return max(low, v // step * step)


def draw(rng):
    op = rng.choice(["gated", "rotary", "attention"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "gated":
        mode = rng.choice(["infer", "train", "grad"])
        c = _gated(None, mode, dtype, _spread(rng, 1, 8192),
                   _spread(rng, 64, 4096), _spread(rng, 64, 8192),
                   rng.choice(["NONE", "RELU", "GELU", "GELU_TANH", "SILU"]),
                   rng.random() < 0.5, rng.random() < 0.5)
        # (no more than the largest listed case; gradients are two forward passes)
        most = (1 << 36) if mode == "grad" else (1 << 37)
        c["m"] = max(1, min(c["m"], most // (c["k"] * c["n"])))
    elif op == "rotary":
        channels = _spread(rng, 16, 256, 8)
        heads = _spread(rng, 1, 64, 8)
        batch = _spread(rng, 1, 64, 8)
        steps = _spread(rng, 1, max(1, min(
            32768, (1 << 26) // (channels * heads * batch))))
        turned = rng.choice([channels, max(2, channels // 2)]) // 2 * 2
        c = _rotary(None, rng.choice(["infer", "grad"]), dtype, batch, steps,
                    heads, channels, turned, rng.choice(["HALVES", "PAIRS"]),
                    rng.choice(["NONE", "FIRST", "EACH"]),
                    rng.choice(["NONE", "POSITIONS", "BASE", "BANDS"]))
    else:
        keys = _spread(rng, 16, 256, 16)
        values = rng.choice([keys, _spread(rng, 16, 256, 16)])
        key_heads = _spread(rng, 1, 16, 8)
        heads = key_heads * rng.choice([1, 1, 2, 3])
        size = heads * max(keys, values)
        batch = _spread(rng, 1, max(1, min(64, (1 << 24) // (
            heads * keys * values))), 8)
        steps = _spread(rng, 1, max(1, min(32768, (1 << 25) // (size * batch))))
        c = _attention(None, rng.choice(["infer", "grad"]), dtype, batch, steps,
                       heads, key_heads, keys, values, rng.random() < 0.5,
                       rng.random() < 0.5)
    del c["name"]
    return c


_BASE = 10000.0
_FACTOR = 8.0
_CONTEXT = 4096


def _frequencies(s):
    """Radians from one position to the next of each pair, in 64 bits."""
    n = s["turned"]
    i = torch.arange(0, n, 2, dtype=torch.float64, device="cuda")
    base = _BASE
    if s["scaling"] == "BASE" and n > 2:
        base *= _FACTOR ** (n / (n - 2))
    f = base ** (-i / n)
    if s["scaling"] == "POSITIONS":
        f = f / _FACTOR
    elif s["scaling"] == "BANDS":
        # (pairs that turn more than 32 times within the trained context stay,
        # those that turn less than once are slowed down)
        turns = f * (_CONTEXT / (2.0 * math.pi))
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / _FACTOR)
    return f


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, kind=dtype):
        x = torch.randn(shape, generator=g, device="cuda")
        return x.mul_(std).add_(mean).to(kind)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda",
                             dtype=torch.int32)

    s = dict(case)
    if case["op"] == "gated":
        m, k, n = case["m"], case["k"], case["n"]
        weight = (n, k) if case["trans_b"] else (k, n)
        s["x"] = normal(m, k)
        # (weights of variance 1 / k keep the activations' size)
        s["wg"] = normal(*weight, std=k ** -0.5)
        s["wu"] = normal(*weight, std=k ** -0.5)
        s["bg"] = normal(n, std=0.1) if case["bias"] else None
        s["bu"] = normal(n, std=0.1) if case["bias"] else None
        if case["mode"] == "grad":
            s["dh"] = normal(m, n)
            # (what the layer's forward pass keeps)
            s["g"] = normal(m, n)
            s["u"] = normal(m, n)
    elif case["op"] == "rotary":
        batch, steps = case["batch"], case["steps"]
        heads, channels = case["heads"], case["channels"]
        # (a slice of a projection that holds values as well)
        rows = normal(batch, steps, heads + heads // 4, channels)
        s["x"] = rows[:, :, :heads]
        s["at"] = None
        if case["positions"] == "FIRST":
            # (caches of different lengths)
            s["at"] = whole(0, 131072, batch)
        elif case["positions"] == "EACH":
            # (documents of about 500 tokens and some that are very long)
            s["at"] = whole(0, 500, batch, steps)
            s["at"] += whole(0, 2, batch, steps) * whole(0, 1000000, batch,
                                                         steps)
        if own:
            from portdnn_amd import ops
            kind = getattr(ops.ROTARY_SCALING, case["scaling"])
            s["table"] = ops.rotary_frequencies(
                case["turned"], base=_BASE, scaling=kind, factor=_FACTOR,
                context=_CONTEXT)
        else:
            s["table"] = _frequencies(case)
    else:
        batch, steps = case["batch"], case["steps"]
        heads, shared = case["heads"], case["key_heads"]
        keys, values = case["keys"], case["values"]
        # (slices of what one projection has written)
        both = normal(batch, steps, 2 * shared * keys + heads * values)
        n = shared * keys
        s["q"] = both[..., :n].unflatten(2, (shared, keys))
        s["k"] = both[..., n:2 * n].unflatten(2, (shared, keys))
        s["v"] = both[..., 2 * n:].unflatten(2, (heads, values))
        s["scale"] = keys ** -0.5
        # (from a memory of some steps to one of some thousands)
        rate = torch.linspace(3.0, 11.0, heads, device="cuda")
        s["decay"] = torch.log1p(-torch.exp2(-rate))
        s["s0"] = normal(batch, heads, keys, values, kind=torch.float32)
        s["reset"] = s["length"] = None
        if case["resets"]:
            # (documents of about 500 tokens)
            s["reset"] = (torch.rand(batch, steps, generator=g, device="cuda")
                          < 0.002).to(torch.uint8)
        if case["ragged"]:
            s["length"] = whole(0, steps + 1, batch)
        if case["mode"] == "grad":
            s["do"] = normal(batch, steps, heads, values)
            s["ds"] = normal(batch, heads, keys, values, kind=torch.float32)
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


def _plain_gated(s):
    dtype = s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    if s["trans_b"]:
        wg, wu = wg.t(), wu.t()
    if s["mode"] == "grad":
        dh, g, u = s["dh"].float(), s["g"].float(), s["u"].float()
        dg = dh * u * _act_slope(g, s["activation"])
        du = dh * _act(g, s["activation"])
        dwg, dwu = x.t() @ dg, x.t() @ du
        if s["trans_b"]:
            dwg, dwu = dwg.t(), dwu.t()
        out = {"x": (dg @ wg.t() + du @ wu.t()).to(dtype), "wg": dwg.to(dtype),
               "wu": dwu.to(dtype)}
        if s["bg"] is not None:
            out["bg"] = dg.sum(0).to(dtype)
            out["bu"] = du.sum(0).to(dtype)
        return out
    g, u = x @ wg, x @ wu
    if s["bg"] is not None:
        g = g + s["bg"].float()
        u = u + s["bu"].float()
    out = {"h": (_act(g, s["activation"]) * u).to(dtype)}
    if s["mode"] == "train":
        out["g"], out["u"] = g.to(dtype), u.to(dtype)
    return out


def _angles(s):
    """[batch or 1, steps, pairs], in 64 bits."""
    steps = torch.arange(s["steps"], device="cuda", dtype=torch.float64)
    if s["at"] is None:
        at = steps[None]
    elif s["at"].dim() == 1:
        at = s["at"].double()[:, None] + steps[None]
    else:
        at = s["at"].double()
    return at[..., None] * s["table"]


def _plain_rotary(s):
    x = s["x"].float()
    n = s["turned"]
    angle = _angles(s)
    if s["mode"] == "grad":
        angle = -angle
    c = torch.cos(angle).float()[:, :, None]
    d = torch.sin(angle).float()[:, :, None]
    out = x.clone()
    if s["layout"] == "HALVES":
        first, second = slice(0, n // 2), slice(n // 2, n)
    else:
        first, second = slice(0, n, 2), slice(1, n, 2)
    a, b = x[..., first], x[..., second]
    out[..., first] = a * c - b * d
    out[..., second] = a * d + b * c
    return {"y": out.to(s["x"].dtype)}


_CHUNK = 64


def _chunks(x):
    """[batch, heads, steps, ...] -> [batch, heads, chunks, _CHUNK, ...]."""
    batch, heads, steps = x.shape[:3]
    count = -(-steps // _CHUNK)
    wide = x.new_zeros(batch, heads, count * _CHUNK, *x.shape[3:])
    wide[:, :, :steps] = x
    return wide.view(batch, heads, count, _CHUNK, *x.shape[3:])


def _attend(q, k, v, log, part, first_part, state):
    """o_t = sum over s <= t of one part: exp(log_t - log_s) (q_t k_s) v_s, and
    what the state in front of the sequence adds where the part is its part;
    with the state behind.  Tensors [batch, heads, steps, ...]."""
    steps = q.shape[2]
    pad = -steps % _CHUNK
    if pad:  # (the last step's, so that the state behind stays as it is)
        log = torch.cat([log, log[..., -1:].expand(*log.shape[:-1], pad)], -1)
        part = torch.cat([part, part[..., -1:].expand(*part.shape[:-1], pad)],
                         -1)
    log, part = _chunks(log), _chunks(part)
    q, k, v = _chunks(q), _chunks(k), _chunks(v)
    count = q.shape[2]
    apart = log[..., :, None] - log[..., None, :]
    order = torch.arange(_CHUNK, device=q.device)
    on = (order[:, None] >= order[None]) & (part[..., :, None] ==
                                            part[..., None, :])
    weight = torch.where(on, torch.exp(torch.where(on, apart, 0.0)), 0.0)
    weight = weight.float() * torch.matmul(q, k.mT.contiguous())
    out = torch.matmul(weight, v)
    del weight, apart, on
    end_log, end_part = log[..., -1:], part[..., -1:]
    before_log = torch.cat([torch.zeros_like(end_log[:, :, :1]),
                            end_log[:, :, :-1]], 2)
    before_part = torch.cat([first_part[..., None, None].expand_as(
        end_part[:, :, :1]), end_part[:, :, :-1]], 2)
    into = torch.where(part == end_part, torch.exp(end_log - log), 0.0).float()
    local = torch.matmul((k * into[..., None]).mT.contiguous(), v)
    carry = torch.where(end_part == before_part,
                        torch.exp(end_log - before_log), 0.0).float()
    states = []
    for n in range(count):
        states.append(state)
        state = carry[:, :, n, :, None] * state + local[:, :, n]
    reach = torch.where(part == before_part, torch.exp(log - before_log),
                        0.0).float()
    out += reach[..., None] * torch.matmul(q, torch.stack(states, 2))
    out = out.flatten(2, 3)[:, :, :steps]
    return out, state


def _plain_attention(s):
    dtype = s["q"].dtype
    batch, steps = s["batch"], s["steps"]
    heads, each = s["heads"], s["heads"] // s["key_heads"]

    def wide(x):
        return x.float().repeat_interleave(each, 2).transpose(1, 2)

    q, k, v = wide(s["q"]), wide(s["k"]), s["v"].float().transpose(1, 2)
    keep = torch.ones(batch, steps, dtype=torch.bool, device=q.device)
    if s["length"] is not None:
        order = torch.arange(steps, device=q.device)
        keep = order[None] < s["length"][:, None]
    fresh = torch.zeros_like(keep)
    if s["reset"] is not None:
        fresh = s["reset"].bool() & keep
    inside = keep[:, None, :, None]
    q, k, v = q * inside, k * inside, v * inside
    # (logarithms of decays from the first step on, documents counted)
    log = torch.cumsum(s["decay"].double()[None, :, None] * keep[:, None], 2)
    part = torch.cumsum(fresh.double(), 1)[:, None].expand(-1, heads, -1)
    zero = part.new_zeros(batch, heads)
    if s["mode"] != "grad":
        o, last = _attend(q * s["scale"], k, v, log, part, zero, s["s0"])
        return {"o": (o * inside).transpose(1, 2).to(dtype), "last": last}
    do = s["do"].float().transpose(1, 2) * inside * s["scale"]
    dq, _ = _attend(do, v, k, log, part, zero, s["s0"].mT.contiguous())
    # the sequence from its end: what a state hands to those behind it
    back = log[..., -1:] - log.flip(2)
    parts, end_part = part.flip(2), part[..., -1]
    ds = s["ds"]
    dk, _ = _attend(v.flip(2), do.flip(2), q.flip(2), back, parts, end_part,
                    ds.mT.contiguous())
    dv, first = _attend(k.flip(2), q.flip(2), do.flip(2), back, parts, end_part,
                        ds)
    reach = torch.where(part[..., 0] == 0, torch.exp(log[..., 0]), 0.0).float()

    def narrow(x):
        x = (x * inside).transpose(1, 2)
        return x.unflatten(2, (heads // each, each)).sum(3).to(dtype)

    return {"q": narrow(dq), "k": narrow(dk.flip(2)),
            "v": (dv.flip(2) * inside).transpose(1, 2).to(dtype),
            "s0": first * reach[..., None, None]}


# ---- the framework's operators -----------------------------------------------


def _own_gated(s):
    from portdnn_amd import ops
    act = getattr(ops.ACTIVATION, s["activation"])
    if s["mode"] == "grad":
        got = ops.gated_matmul_grad(
            s["dh"], s["x"], s["wg"], s["wu"], s["g"], s["u"], activation=act,
            trans_b=s["trans_b"], bias=s["bg"] is not None)
        names = ["x", "wg", "wu"] + (["bg", "bu"] if s["bg"] is not None else [])
        return dict(zip(names, got))
    if s["mode"] == "train":
        h, g, u = ops.gated_matmul(
            s["x"], s["wg"], s["wu"], bias_gate=s["bg"], bias_up=s["bu"],
            activation=act, trans_b=s["trans_b"], keep_pre_activation=True)
        return {"h": h, "g": g, "u": u}
    return {"h": ops.gated_matmul(
        s["x"], s["wg"], s["wu"], bias_gate=s["bg"], bias_up=s["bu"],
        activation=act, trans_b=s["trans_b"])}


def _own_rotary(s):
    from portdnn_amd import ops
    return {"y": ops.rotary(s["x"], s["table"], positions=s["at"],
                            layout=getattr(ops.ROTARY, s["layout"]),
                            inverse=s["mode"] == "grad")}


def _own_attention(s):
    from portdnn_amd import ops
    kinds = {"resets": s["reset"], "lengths": s["length"],
             "initial_state": s["s0"], "scale": s["scale"]}
    if s["mode"] == "grad":
        got = ops.linear_attention_grad(
            s["do"], s["q"], s["k"], s["v"], s["decay"],
            grad_final_state=s["ds"], **kinds)
        return {"q": got["q"], "k": got["k"], "v": got["v"],
                "s0": got["initial_state"]}
    o, last = ops.linear_attention(s["q"], s["k"], s["v"], s["decay"], **kinds)
    return {"o": o, "last": last}


def run(state):
    if own:
        return {"gated": _own_gated, "rotary": _own_rotary,
                "attention": _own_attention}[state["op"]](state)
    return {"gated": _plain_gated, "rotary": _plain_rotary,
            "attention": _plain_attention}[state["op"]](state)


def work(case):
    e = _SIZE[case["dtype"]]
    grad = case["mode"] == "grad"
    if case["op"] == "gated":
        m, k, n = case["m"], case["k"], case["n"]
        weights = 2 * k * n + 2 * n * case["bias"]
        if grad:
            return {"bytes": e * (2 * m * k + 2 * weights + 3 * m * n),
                    "flops": 8 * m * k * n}
        outputs = m * n * (3 if case["mode"] == "train" else 1)
        return {"bytes": e * (m * k + weights + outputs), "flops": 4 * m * k * n}
    batch, steps, heads = case["batch"], case["steps"], case["heads"]
    if case["op"] == "rotary":
        size = batch * steps * heads * case["channels"]
        at = {"NONE": 0, "FIRST": batch, "EACH": batch * steps}
        return {"bytes": 2 * e * size + 4 * at[case["positions"]] +
                4 * case["turned"], "flops": 3 * size}
    keys, values = case["keys"], case["values"]
    of_keys = batch * steps * case["key_heads"] * keys
    of_values = batch * steps * heads * values
    states = batch * heads * keys * values
    # a state's product and its update at every step: four operations
    flops = 4 * batch * steps * heads * keys * values
    flags = batch * steps * case["resets"]
    if grad:
        # q, k, v, do in, the gradients of q, k and v out, three states; the
        # products of do with the states, of the states' gradients with k and v,
        # and two updates
        return {"bytes": e * (4 * of_keys + 3 * of_values) + 12 * states +
                flags, "flops": 5 * flops // 2}
    return {"bytes": e * (2 * of_keys + 2 * of_values) + 8 * states + flags,
            "flops": flops}


# ---- the definitions in 64 bits ------------------------------------------------


def _sigma(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _exact_gated(s):
    dt = torch.float64
    x = s["x"].to(dt)
    wg, wu = ((w.mT if s["trans_b"] else w).to(dt) for w in (s["wg"], s["wu"]))

    def both(z):
        """act(z) and act'(z)."""
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
        value, slope = both(s["g"].to(dt))
        du = s["dh"].to(dt) * value
        dg = s["dh"].to(dt) * slope * s["u"].to(dt)
        out = {"x": torch.matmul(dg, wg.mT) + torch.matmul(du, wu.mT)}
        for name, d in (("wg", dg), ("wu", du)):
            out[name] = (torch.matmul(d.mT, x) if s["trans_b"] else
                         torch.matmul(x.mT, d))
        if s["bg"] is not None:
            out["bg"], out["bu"] = torch.sum(dg, 0), torch.sum(du, 0)
        return out
    g, u = torch.matmul(x, wg), torch.matmul(x, wu)
    if s["bg"] is not None:
        g += s["bg"].to(dt)
        u += s["bu"].to(dt)
    out = {"h": both(g)[0] * u}
    if s["mode"] == "train":
        out["g"], out["u"] = g, u
    return out


def _exact_rotary(s):
    """Pairs as complex numbers times exp(i angle)."""
    batch, steps, n = s["batch"], s["steps"], s["turned"]
    at = torch.arange(steps, device="cuda").expand(batch, steps)
    if s["positions"] == "FIRST":
        at = at + s["at"][:, None]
    elif s["positions"] == "EACH":
        at = s["at"]
    angle = at.to(torch.float64)[..., None] * _frequencies(s)
    sign = -1.0 if s["mode"] == "grad" else 1.0
    turn = torch.complex(torch.cos(angle), sign * torch.sin(angle))[:, :, None]
    y = s["x"].to(torch.float64)
    head = y[..., :n]
    if s["layout"] == "HALVES":
        z = torch.complex(head[..., :n // 2], head[..., n // 2:]) * turn
        head = torch.cat([z.real, z.imag], -1)
    else:
        z = head.unflatten(-1, (n // 2, 2))
        z = torch.complex(z[..., 0], z[..., 1]) * turn
        head = torch.stack([z.real, z.imag], -1).flatten(-2)
    return {"y": torch.cat([head, y[..., n:]], -1)}


def _exact_attention(s):
    """Step by step."""
    batch, steps, heads = s["batch"], s["steps"], s["heads"]
    dt = torch.float64
    group = torch.arange(heads, device="cuda") // (heads // s["key_heads"])
    q, k, v = s["q"].to(dt)[:, :, group], s["k"].to(dt)[:, :, group], s["v"].to(dt)
    a = torch.exp(s["decay"].to(dt))[None, :, None, None]
    one = torch.ones(batch, 1, 1, 1, dtype=dt, device="cuda")
    # 0 where a document begins, 1 elsewhere; whether a step counts
    stays = (one.expand(batch, steps, 1, 1) if s["reset"] is None else
             (s["reset"] == 0).to(dt)[..., None, None])
    length = (torch.full((batch,), steps, device="cuda") if s["length"] is None
              else s["length"]).view(batch, 1, 1, 1)
    state = s["s0"].to(dt)
    if s["mode"] != "grad":
        o = torch.zeros_like(v)
        for t in range(steps):
            new = a * stays[:, t, None] * state + k[:, t, :, :, None] * v[:, t, :, None]
            state = torch.where(length > t, new, state)
            row = torch.matmul(q[:, t, :, None], state)[:, :, 0] * s["scale"]
            o[:, t] = torch.where(length[..., 0] > t, row, 0.0)
        return {"o": o, "last": state}
    do = s["do"].to(dt) * s["scale"]
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(steps):
        new = a * stays[:, t, None] * state + k[:, t, :, :, None] * v[:, t, :, None]
        state = torch.where(length > t, new, state)
        row = torch.matmul(state, do[:, t, :, :, None])[..., 0]
        dq[:, t] = torch.where(length[..., 0] > t, row, 0.0)
    total = s["ds"].to(dt)
    for t in range(steps - 1, -1, -1):
        inside = length > t
        new = total + q[:, t, :, :, None] * do[:, t, :, None]
        row = torch.matmul(new, v[:, t, :, :, None])[..., 0]
        dk[:, t] = torch.where(inside[..., 0], row, 0.0)
        row = torch.matmul(k[:, t, :, None], new)[:, :, 0]
        dv[:, t] = torch.where(inside[..., 0], row, 0.0)
        total = torch.where(inside, a * stays[:, t, None] * new, total)

    def shared(x):
        out = torch.zeros(batch, steps, s["key_heads"], s["keys"], dtype=dt,
                          device="cuda")
        return out.index_add_(2, group, x)

    return {"q": shared(dq), "k": shared(dk), "v": dv, "s0": total}


def exact(case, seed):
    s = prepare(case, seed)
    return {"gated": _exact_gated, "rotary": _exact_rotary,
            "attention": _exact_attention}[case["op"]](s)
