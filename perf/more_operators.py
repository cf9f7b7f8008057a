"""Timed cases of a layer's projections in 8-bit integers: what makes the rows, the product, and a feed-forward of them.

A row of activations and a channel of weights are held as integers of -127 .. 127 with one 32-bit scale each, ``value = scale * q``:

    rows of x:         m = max |x|,  q = rint(x * (127 / m)),  scale = m / 127                      (m = 0: q = 0, scale 0)
    normed rows:       x += add,  v = x * weight,  q and m from v as above,  scale = m / 127 / sqrt(mean(x^2) + eps)
    activated rows:    h = act(g) * u rounded to bfloat16,  q and scale from h as above
    product:           out[t, n] (+)= scale_a[t] * scale_w[n] * sum over k of a[t, k] * w[n, k]

Rows lie in buffers whose width is the next multiple of 16, with zeros behind. Every operator has a plain form here, of elementary torch
operations in 32 bits. What comes out in 8 bits is returned as the values it stands for.
"""
import math

import torch

own = False          # False: the plain forms; True: this repository's kernels

DEV = "cuda:0"
EPS = 1e-5
ACTIVATIONS = ("silu", "relu", "gelu_tanh", "capped_swish")
LIMIT = 7.0          # of capped_swish


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    norm = {"op": "norm", "add": "float32"}
    gated = {"op": "gated", "activation": "silu", "dtype": "float32", "bias": False}
    product = {"op": "product", "rows": "int8", "out": "float32", "accumulate": False}
    block = {"op": "feed_forward", "activation": "silu"}
    return [
        # one user's token at the 1B shape, behind the attention's output projection: latency
        dict(norm, name="norm_one_token", T=1, D=2048),
        # a prompt of 2,048 tokens, the projection's output in 16 bits
        dict(norm, name="norm_prompt", T=2048, D=2048, add="bfloat16"),
        # a large step at the 8B width
        dict(norm, name="norm_large", T=8192, D=4096),
        # eight single tokens between the feed-forward's products at the 1B shape
        dict(gated, name="gated_few", T=8, I=8192),
        # a large step at the 8B shape, another activation with a bias, from 16 bits
        dict(gated, name="gated_large", T=4096, I=14336, activation="capped_swish", dtype="bfloat16", bias=True),
        # one token through the down projection of the 1B shape, added to the residual stream: bound by the weights' bytes
        dict(product, name="product_one_token", T=1, K=8192, N=2048, accumulate=True),
        # 64 tokens through gate and up of the 8B shape
        dict(product, name="product_batch", T=64, K=4096, N=28672),
        # a portion of a prompt, an odd number of rows, the attention's output in 16 bits into the 8B shape's output projection
        dict(product, name="product_portion", T=333, K=4096, N=4096, rows="bfloat16", out="bfloat16"),
        # a large step through the 8B shape's down projection
        dict(product, name="product_large", T=8192, K=14336, N=4096, out="bfloat16"),
        # a decode step's feed-forward at the 1B shape: norm, gate and up, activation, down
        dict(block, name="feed_forward_decode", T=8, H=2048, I=8192),
        # a prompt's
        dict(block, name="feed_forward_prompt", T=2048, H=2048, I=8192),
        # odd sizes throughout
        dict(block, name="feed_forward_odd", T=501, H=1533, I=4099, activation="gelu_tanh"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["norm", "gated", "product", "product", "feed_forward"])
    if op == "norm":
        D = _log(rng, 16, 16384)
        return {"op": op, "T": _log(rng, 1, min(8192, 33_000_000 // D)), "D": D, "add": rng.choice(["none", "float32", "bfloat16"])}
    if op == "gated":
        I = _log(rng, 16, 28672)
        return {"op": op, "T": _log(rng, 1, min(4096, 58_000_000 // I)), "I": I, "activation": rng.choice(ACTIVATIONS),
                "dtype": rng.choice(["float32", "bfloat16"]), "bias": rng.random() < 0.3}
    if op == "product":
        K, N = rng.choice([(2048, 2048), (2048, 16384), (8192, 2048), (4096, 4096), (4096, 6144), (4096, 28672), (14336, 4096),
                           (_log(rng, 16, 14336), _log(rng, 1, 8192)), (_log(rng, 16, 14336), _log(rng, 1, 8192))])
        rows = rng.choice(["int8", "int8", "bfloat16", "float32"])
        # (rows made in the pass: values next to a border of two integers may fall to either, so the output has 16 bits)
        accumulate = rows == "int8" and rng.random() < 0.5
        return {"op": op, "T": _log(rng, 1, min(8192, 480_000_000_000 // (K * N), 58_000_000 // N)), "K": K, "N": N, "rows": rows,
                "out": "float32" if accumulate else rng.choice(["float32", "bfloat16"]) if rows == "int8" else "bfloat16",
                "accumulate": accumulate}
    H, I = _log(rng, 64, 4096), _log(rng, 64, 14336)
    return {"op": op, "T": _log(rng, 1, min(4096, 100_000_000_000 // (H * I))), "H": H, "I": I, "activation": rng.choice(ACTIVATIONS)}


# ---------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"norm": _prepare_norm, "gated": _prepare_gated, "product": _prepare_product, "feed_forward": _prepare_block}[case["op"]](case, g)


def _dtype(name):
    return {"float32": torch.float32, "bfloat16": torch.bfloat16}[name]


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _width(n):
    return (n + 15) // 16 * 16


def _ints(rows, width):
    return torch.empty(rows, width, dtype=torch.int8, device=DEV)


def _stream(g, T, D):
    """Rows of a residual stream: a few of the channels are ten times as large as the others."""
    return _normal(g, T, D) * torch.where(torch.rand(D, generator=g, device=DEV) < 0.01, 10.0, 1.0) * (0.5 + torch.rand(T, 1, generator=g, device=DEV))


def _in_8_bits(v):
    """q and scale of every row of v; q in 32 bits."""
    m = v.abs().amax(1, keepdim=True)
    q = torch.round(v * torch.where(m > 0, torch.full_like(m, 127.0) / m, 0.0))      # (one quotient: 127.0 / m takes a reciprocal and a product)
    return q, m / 127.0


def _padded(q):
    out = torch.zeros(q.shape[0], _width(q.shape[1]), dtype=torch.int8, device=DEV)
    out[:, :q.shape[1]] = q
    return out


def _weight(g, N, K):
    q, scale = _in_8_bits(_normal(g, N, K) / math.sqrt(K))
    return q.to(torch.int8), scale[:, 0].contiguous()


def _laid_out(w, gated=False):
    """The weight as the product reads it: a program lays it out once, when it loads the model."""
    if own:
        from geneinfer_b200.ops import kernels
        return kernels.int8_weight(w[0], w[1], gated=gated)
    return None


def _prepare_norm(case, g):
    T, D = case["T"], case["D"]
    return {"op": "norm", "x": _stream(g, T, D), "add": None if case["add"] == "none" else (0.3 * _normal(g, T, D)).to(_dtype(case["add"])),
            "weight": 0.5 + torch.rand(D, generator=g, device=DEV), "q": _ints(T, _width(D)), "scales": torch.empty(T, device=DEV),
            "values": torch.empty(T, D, dtype=torch.bfloat16, device=DEV)}


def _prepare_gated(case, g):
    T, I = case["T"], case["I"]
    return {"op": "gated", "gate_up": (1.5 * _stream(g, T, 2 * I)).to(_dtype(case["dtype"])), "activation": case["activation"],
            "bias": 0.2 * _normal(g, 2 * I) if case["bias"] else None, "q": _ints(T, _width(I)), "scales": torch.empty(T, device=DEV),
            "values": torch.empty(T, I, dtype=torch.bfloat16, device=DEV)}


def _prepare_product(case, g):
    T, K, N = case["T"], case["K"], case["N"]
    w = _weight(g, N, K)
    x = _stream(g, T, K)
    s = {"op": "product", "K": K, "w": w, "laid_out": _laid_out(w), "accumulate": case["accumulate"],
         "out": _normal(g, T, N).to(_dtype(case["out"]))}
    if case["rows"] == "int8":
        q, scale = _in_8_bits(x)
        return dict(s, x=None, a=_padded(q), a_scales=scale[:, 0].contiguous())
    return dict(s, x=x.to(_dtype(case["rows"])), a=_ints(T, _width(K)), a_scales=torch.empty(T, device=DEV))


def _prepare_block(case, g):
    T, H, I = case["T"], case["H"], case["I"]
    up, down = _weight(g, 2 * I, H), _weight(g, H, I)
    s = {"op": "feed_forward", "x": _stream(g, T, H), "add": 0.3 * _normal(g, T, H), "weight": 0.5 + torch.rand(H, generator=g, device=DEV),
         "up": up, "down": down, "laid_out": (_laid_out(up, gated=True), _laid_out(down)), "activation": case["activation"],
         "q": _ints(T, _width(H)), "scales": torch.empty(T, device=DEV), "h": _ints(T, _width(I)), "h_scales": torch.empty(T, device=DEV),
         "work": torch.empty(T * 2 * I, device=DEV), "out": torch.empty(T, H, dtype=torch.bfloat16, device=DEV)}
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "gated": _plain_gated, "product": _plain_product, "feed_forward": _plain_block}[state["op"]](state)


def _values(q, scales, out):
    """The values that q stands for, in bfloat16."""
    return torch.mul(q[:, :out.shape[1]], scales[:, None], out=out)


def _own(s):
    from geneinfer_b200.ops import kernels
    if s["op"] == "norm":
        kernels.rmsnorm_int8(s["x"], s["weight"], s["q"], s["scales"], EPS, add=s["add"])
        return {"values": _values(s["q"], s["scales"], s["values"]), "x": s["x"]}
    if s["op"] == "gated":
        kernels.gated_act_int8(s["gate_up"], s["q"], s["scales"], s["activation"], LIMIT, s["bias"])
        return {"values": _values(s["q"], s["scales"], s["values"])}
    if s["op"] == "product":
        if s["x"] is not None:
            kernels.quantize_rows(s["x"], s["a"], s["a_scales"])
        kernels.int8_product(s["a"], s["a_scales"], s["laid_out"], s["out"], accumulate=s["accumulate"])
        return {"out": s["out"]}
    up, down = s["laid_out"]
    kernels.rmsnorm_int8(s["x"], s["weight"], s["q"], s["scales"], EPS, add=s["add"])
    kernels.int8_gated(s["q"], s["scales"], up, s["h"], s["h_scales"], s["work"], s["activation"], LIMIT)
    kernels.int8_product(s["h"], s["h_scales"], down, s["out"])
    return {"out": s["out"], "x": s["x"]}


def _plain_normed(x, weight):
    """q and scale of the normed rows of x."""
    q, scale = _in_8_bits(x * weight)
    return q, scale / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)


def _plain_act(g, u, activation):
    if activation == "relu":
        return g.clamp(min=0.0) * u
    if activation == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))) * u
    if activation == "capped_swish":
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        return g * (1.0 / (1.0 + torch.exp(-1.702 * g))) * (u + 1.0)
    return g * (1.0 / (1.0 + torch.exp(-g))) * u


def _plain_norm(s):
    if s["add"] is not None:
        s["x"].add_(s["add"])
    q, scale = _plain_normed(s["x"], s["weight"])
    return {"values": (q * scale).to(torch.bfloat16), "x": s["x"]}


def _plain_activated(gate_up, activation):
    g, u = gate_up.chunk(2, 1)
    return _in_8_bits(_plain_act(g, u, activation).to(torch.bfloat16).float())


def _plain_gated(s):
    gate_up = s["gate_up"].float()
    q, scale = _plain_activated(gate_up if s["bias"] is None else gate_up + s["bias"], s["activation"])
    return {"values": (q * scale).to(torch.bfloat16)}


def _plain_sums(q, scale, w):
    """The integers are added in 32-bit floats, exact below 2^24, where sums of random signs stay."""
    return (q @ w[0].float().T) * scale * w[1]


def _plain_product(s):
    if s["x"] is not None:
        q, scale = _in_8_bits(s["x"].float())
    else:
        q, scale = s["a"][:, :s["K"]].float(), s["a_scales"][:, None]
    v = _plain_sums(q, scale, s["w"])
    s["out"].copy_(s["out"] + v if s["accumulate"] else v)
    return {"out": s["out"]}


def _plain_block(s):
    s["x"].add_(s["add"])
    q, scale = _plain_normed(s["x"], s["weight"])
    h, h_scale = _plain_activated(_plain_sums(q, scale, s["up"]), s["activation"])
    s["out"].copy_(_plain_sums(h, h_scale, s["down"]))
    return {"out": s["out"], "x": s["x"]}


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {"float32": 4, "bfloat16": 2, "none": 0, "int8": 1}
    T = case["T"]
    if case["op"] == "norm":
        n = T * case["D"]
        return {"bytes": n * (5 + (size[case["add"]] + 4 if case["add"] != "none" else 0)) + 4 * (case["D"] + T), "flops": 6 * n}
    if case["op"] == "gated":
        n = T * case["I"]
        return {"bytes": n * (2 * size[case["dtype"]] + 1) + 4 * T, "flops": 12 * n}
    if case["op"] == "product":
        K, N = case["K"], case["N"]
        return {"bytes": N * (K + 4) + T * (K * size[case["rows"]] + 4) + T * N * size[case["out"]] * (2 if case["accumulate"] else 1),
                "flops": 2 * T * K * N}
    H, I = case["H"], case["I"]
    return {"bytes": 3 * H * I + 4 * (2 * I + 2 * H) + T * H * (4 + 4 + 4 + 2), "flops": 6 * T * H * I}


# ---------------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_rows(v):
    top = v.abs().max(dim=1).values
    unit = torch.zeros_like(top)
    unit[top > 0] = 127.0 / top[top > 0]
    return (v * unit[:, None]).round(), top / 127.0


def _exact_normed(x, weight):
    q, scale = _exact_rows(x * weight.double())
    return q, scale * (x.square().sum(1) / x.shape[1] + EPS).rsqrt()


def _exact_h(g, u, activation):
    if activation == "relu":
        h = torch.where(g > 0, g, 0.0) * u
    elif activation == "gelu_tanh":
        h = g * u * torch.sigmoid(2.0 * 0.7978845608028654 * (g + 0.044715 * g ** 3))
    elif activation == "capped_swish":
        g = torch.where(g > LIMIT, LIMIT, g)
        h = g * torch.sigmoid(1.702 * g) * (torch.where(u > LIMIT, LIMIT, torch.where(u < -LIMIT, -LIMIT, u)) + 1.0)
    else:
        h = g * torch.sigmoid(g) * u
    return h.to(torch.bfloat16).double()


def _exact_product(q, scale, w):
    out = torch.empty(q.shape[0], w[0].shape[0], dtype=torch.float64, device=DEV)
    weights = w[0].double() * w[1].double()[:, None]
    for at in range(0, q.shape[0], 1024):
        rows = slice(at, at + 1024)
        out[rows] = (q[rows].double() * scale[rows].double()[:, None]) @ weights.T
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double() + (0.0 if s["add"] is None else s["add"].double())
        q, scale = _exact_normed(x, s["weight"])
        return {"values": q * scale[:, None], "x": x}
    if case["op"] == "gated":
        both = s["gate_up"].double() + (0.0 if s["bias"] is None else s["bias"].double())
        q, scale = _exact_rows(_exact_h(both[:, :case["I"]], both[:, case["I"]:], case["activation"]))
        return {"values": q * scale[:, None]}
    if case["op"] == "product":
        q, scale = (s["a"][:, :case["K"]], s["a_scales"]) if s["x"] is None else _exact_rows(s["x"].double())
        out = _exact_product(q, scale, s["w"])
        return {"out": out + s["out"].double() if case["accumulate"] else out}
    x = s["x"].double() + s["add"].double()
    both = _exact_product(*_exact_normed(x, s["weight"]), s["up"])
    h, h_scale = _exact_rows(_exact_h(both[:, :case["I"]], both[:, case["I"]:], case["activation"]))
    return {"out": _exact_product(h, h_scale, s["down"]), "x": x}
