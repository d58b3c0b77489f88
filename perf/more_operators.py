"""Workloads of the operators around a decoder layer's products: rotary positions in both layouts and scaled for long contexts,
the gated feed-forward block, and 8-bit floating point with a scale for each block of 128, its quantisation and its products.

``listed()`` names the cases, ``draw(rng)`` makes one more of the same ranges, ``prepare(case, seed)`` makes what a program has
in hand before a call, ``run(state)`` is one call (with its gradients in the training cases) and ``work(case)`` the bytes and
operations that it cannot do without.  With ``own`` unset ``run`` computes the same in elementary torch operations in 32 bits;
``exact(case, seed)`` computes it in 64 bits.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 128                       # values that share a scale
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------- cases
def _rotate(name, rows, heads, head_dim, rotary_dim, interleaved, scaling, theta, packed, dtype, train):
    return {"name": name, "kind": "rotate", "rows": rows, "heads": heads, "head_dim": head_dim, "rotary_dim": rotary_dim,
            "interleaved": interleaved, "scaling": scaling, "theta": theta, "packed": packed, "dtype": dtype, "train": train}


def _feed(name, rows, hidden, inter, activation, train):
    return {"name": name, "kind": "feed", "rows": rows, "hidden": hidden, "inter": inter, "activation": activation, "train": train}


def _quantise(name, rows, cols, block_rows, transpose, dtype):
    return {"name": name, "kind": "quantise", "rows": rows, "cols": cols, "block_rows": block_rows, "transpose": transpose,
            "dtype": dtype}


def _linear(name, rows, hidden, out, train):
    return {"name": name, "kind": "linear", "rows": rows, "hidden": hidden, "out": out, "train": train}


def listed():
    return [
        # queries and keys of the newest token of eight sequences far into a long context: what one call costs at least
        _rotate("rotate newest tokens", 8, 40, 128, 128, False, "llama3", 500000.0, False, "bf16", False),
        # queries and keys of a micro-batch of ragged documents of the 220M model
        _rotate("rotate 220m train", 4071, 20, 64, 64, False, "none", 10000.0, True, "bf16", True),
        # one long document, half of every head rotated, neighbouring pairs, frequencies stretched for it
        _rotate("rotate long document", 16384, 24, 128, 64, True, "yarn", 1000000.0, True, "bf16", True),
        # the newest token of one sequence: the weights are read once
        _feed("feed one token", 1, 2048, 8192, "silu", False),
        # the newest tokens of two dozen requests through the 4B model's block
        _feed("feed newest tokens", 24, 2560, 9728, "silu", False),
        # a short ragged micro-batch of the 220M model, another activation
        _feed("feed 220m train", 777, 640, 1728, "gelu_tanh", True),
        # a whole micro-batch of the 4B model
        _feed("feed 4b train", 8192, 2560, 9728, "silu", True),
        # a weight of the 220M model on its way into 8 bits, turned around for the gradient's product
        _quantise("quantise weight", 1728, 640, 128, True, "bf16"),
        # a micro-batch of wide activations, every row by itself
        _quantise("quantise activations", 8192, 9728, 1, False, "bf16"),
        # the newest tokens of eight requests, weight kept in 8 bits
        _linear("linear newest tokens", 8, 2560, 9728, False),
        # a ragged batch of prompts, weight kept in 8 bits
        _linear("linear prompts", 1531, 2048, 8192, False),
        # a whole micro-batch of the 4B model, all three products in 8 bits
        _linear("linear 4b train", 8192, 2560, 9728, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


def _draw(rng):
    kind = rng.choice(("rotate", "feed", "feed", "quantise", "linear", "linear"))
    train = rng.random() < 0.5
    if kind == "rotate":
        head_dim = rng.choice((32, 64, 128, 128, 2 * rng.randrange(1, 100)))
        rotary_dim = rng.choice((head_dim, head_dim, 2 * rng.randrange(1, head_dim // 2 + 1)))
        case = _rotate("", _log_int(rng, 1, 16384), rng.choice((1, 6, 20, 24, 40)), head_dim, rotary_dim, rng.random() < 0.5,
                       rng.choice(("none", "linear", "ntk", "yarn", "llama3")), rng.choice((10000.0, 500000.0, 1000000.0)),
                       rng.random() < 0.7, rng.choice(("bf16", "bf16", "fp32")), train)
    elif kind == "quantise":
        rows, cols = _log_int(rng, 1, 8192), rng.choice((640, 2048, 2560, 9728, rng.randrange(1, 4000)))
        case = _quantise("", rows, cols, rng.choice((1, 128)), rng.random() < 0.5, rng.choice(("bf16", "bf16", "fp32")))
    else:
        # hidden and intermediate sizes of the decoder configurations and of the tiny ones, and whatever lies between
        hidden, inter = rng.choice(((128, 352), (640, 1728), (2048, 6144), (2048, 8192), (2560, 9728), (4096, 12288),
                                    (8 * rng.randrange(1, 400), 8 * rng.randrange(1, 1000))))
        rows = _log_int(rng, 1, 8192)
        if kind == "feed":
            case = _feed("", rows, hidden, inter, rng.choice(("silu", "silu", "gelu", "gelu_tanh", "relu")), train)
        else:
            hidden, out = rng.choice(((hidden, inter), (inter, hidden), (hidden, hidden)))
            case = _linear("", rows, hidden, out, train)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------- inputs
def _scaling(case):
    """The stretching of the frequencies as a model's configuration has it."""
    return {"none": None,
            "linear": {"rope_type": "linear", "factor": 4.0},
            "ntk": {"rope_type": "ntk", "factor": 4.0},
            "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096},
            "llama3": {"rope_type": "llama3", "factor": 32.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                       "original_max_position_embeddings": 8192}}[case["scaling"]]


def _frequencies(case):
    """(angle of each pair at position 1, factor of cosine and sine), in 64 bits."""
    r, theta, s = case["rotary_dim"], case["theta"], _scaling(case) or {}
    i = torch.arange(r // 2, dtype=torch.float64)
    kind, factor = s.get("rope_type"), s.get("factor", 1.0)
    if kind == "ntk" and r > 2:
        theta = theta * factor ** (r / (r - 2))
    inv = theta ** (-2.0 * i / r)
    m = 1.0
    if kind == "linear":
        inv = inv / factor
    elif kind == "yarn":
        turns = s["original_max_position_embeddings"] / (2 * math.pi)
        lo = max(math.floor(r * math.log(turns / 32.0) / (2 * math.log(theta))), 0)
        hi = min(math.ceil(r * math.log(turns / 1.0) / (2 * math.log(theta))), r - 1)
        ramp = ((i - lo) / (hi - lo if hi != lo else 0.001)).clamp(0.0, 1.0)
        inv = inv / factor * ramp + inv * (1.0 - ramp)
        m = 0.1 * math.log(factor) + 1.0
    elif kind == "llama3":
        turns = s["original_max_position_embeddings"] * inv / (2 * math.pi)
        kept = ((turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])).clamp(0.0, 1.0)
        inv = inv / factor * (1.0 - kept) + inv * kept
    return inv, m


def _positions(case, gen):
    rows = case["rows"]
    if not case["packed"]:                        # newest tokens, each of a sequence of its own
        return torch.randint(0, 131072, (rows,), generator=gen, device=DEVICE)
    rng = random.Random(7919 * rows)
    cuts, at = [], 0
    while at < rows:                              # documents one after the other, positions from 0 in each
        n = min(rows - at, _log_int(rng, 16, 16384))
        cuts.append(torch.arange(n))
        at += n
    return torch.cat(cuts).to(DEVICE)


def _hidden(gen, rows, cols):
    """Normalised hidden states: some features that run large, padding at the end."""
    x = torch.randn(rows, cols, generator=gen, device=DEVICE)
    x = x * torch.where(torch.arange(cols, device=DEVICE) % 97 == 5, 12.0, 1.0)
    return x.masked_fill((torch.arange(rows, device=DEVICE) >= rows - rows // 50)[:, None], 0.0)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}

    def mat(rows, cols, std=1.0):
        return (torch.randn(rows, cols, generator=gen, device=DEVICE) * std).bfloat16()

    if case["kind"] == "rotate":
        cols, dtype = case["heads"] * case["head_dim"], DTYPES[case["dtype"]]
        state["x"] = torch.randn(case["rows"], cols, generator=gen, device=DEVICE).to(dtype).requires_grad_(case["train"])
        state["positions"] = _positions(case, gen)
        if case["train"]:
            state["dy"] = torch.randn(case["rows"], cols, generator=gen, device=DEVICE).to(dtype)
        if own:                                   # made once for a model; every layer uses it
            from himuon_b200 import ops
            state["freqs"] = ops.RotaryFrequencies(case["rotary_dim"], case["theta"], _scaling(case), device=DEVICE)
        else:
            inv, state["factor"] = _frequencies(case)
            state["inv"] = inv.to(DEVICE)
        return state
    if case["kind"] == "quantise":
        x = _hidden(gen, case["rows"], case["cols"])
        # rows of very different size, as gradients of rare tokens are
        x = x * torch.exp2(torch.randint(-12, 12, (case["rows"], 1), generator=gen, device=DEVICE).float())
        state["x"] = x.to(DTYPES[case["dtype"]])
        return state
    rows, hidden, train = case["rows"], case["hidden"], case["train"]
    state["x"] = _hidden(gen, rows, hidden).bfloat16().requires_grad_(train)
    std = 1.0 / math.sqrt(hidden * (1 + 143 / 97))             # (of the features that run large)
    if case["kind"] == "feed":
        inter = case["inter"]
        state["wg"], state["wu"], state["wd"] = mat(inter, hidden, std), mat(inter, hidden, std), mat(hidden, inter, 1.0 / math.sqrt(inter))
        for n in ("wg", "wu", "wd"):
            state[n].requires_grad_(train)
        out = hidden
    else:
        out = case["out"]
        w = mat(out, hidden, std)
        if train:
            state["w"] = w.requires_grad_()
        else:                                     # laid out in 8 bits when the model was loaded
            q, s = _plain_quantise(w.float(), 128)
            state["w8"], state["w8_scales"] = q.to(torch.float8_e4m3fn), s
    if train:
        state["dy"] = mat(rows, out, 1.0 / rows)
    return state


# ------------------------------------------------------------------------------------------- one call
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        return {"rotate": _plain_rotate, "feed": _plain_feed, "quantise": _plain_quantised, "linear": _plain_linear}[case["kind"]](state, case)


def _run_own(state, case):
    from himuon_b200 import ops

    if case["kind"] == "rotate":
        y = ops.rotary(state["x"], state["positions"], state["freqs"], case["heads"], case["head_dim"], interleaved=case["interleaved"])
        if not case["train"]:
            return {"y": y}
        return {"y": y.detach(), "dx": torch.autograd.grad(y, state["x"], state["dy"])[0]}
    if case["kind"] == "quantise":
        q = ops.quantize_fp8(state["x"], block_rows=case["block_rows"], transpose=case["transpose"])
        return {"values": q.dequantize(), "scales": q.scales}
    if case["kind"] == "feed":
        leaves = [state[n] for n in ("x", "wg", "wu", "wd")]
        y = ops.gated_mlp(*leaves, activation=case["activation"])
        names = ("dx", "dwg", "dwu", "dwd")
    else:
        leaves = [state["x"], state["w"] if case["train"] else ops.Fp8Blocks(state["w8"], state["w8_scales"], 128)]
        y = ops.fp8_linear(*leaves)
        names = ("dx", "dw")
    if not case["train"]:
        return {"y": y}
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, state["dy"])))}


def _plain_rotate(state, case):
    angles = state["positions"].double()[:, None] * state["inv"]
    cos, sin = ((f(angles) * state["factor"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turn(x, sin):
        x = x.float().view(case["rows"], case["heads"], case["head_dim"])
        head, rest = x[..., :case["rotary_dim"]], x[..., case["rotary_dim"]:]
        a, b = (head[..., 0::2], head[..., 1::2]) if case["interleaved"] else head.chunk(2, -1)
        a, b = a * cos - b * sin, b * cos + a * sin
        head = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
        return torch.cat((head, rest), -1).view(case["rows"], -1).to(DTYPES[case["dtype"]])

    out = {"y": turn(state["x"], sin)}
    if case["train"]:
        out["dx"] = turn(state["dy"], -sin)
    return out


def _plain_quantise(x, block_rows):
    """Values in e4m3 as fp32 and the scales, powers of two, of blocks of (block_rows, 128)."""
    rows, cols = x.shape
    nr, nc = -(-rows // block_rows), -(-cols // BLOCK)
    padded = torch.zeros(nr * block_rows, nc * BLOCK, dtype=x.dtype, device=x.device)
    padded[:rows, :cols] = x
    blocks = padded.view(nr, block_rows, nc, BLOCK)
    mantissa, exponent = torch.frexp(blocks.abs().amax((1, 3)))
    # the least power of two that keeps the largest value at 448 = 0.875 * 2^9 or below
    exponent = torch.where(mantissa == 0, torch.zeros_like(exponent), exponent - 9 + (mantissa > 0.875).int()).clamp(min=-110)
    scales = torch.ldexp(torch.ones_like(mantissa), exponent)
    q = (blocks / scales[:, None, :, None]).float().to(torch.float8_e4m3fn).float()
    return q.view(nr * block_rows, nc * BLOCK)[:rows, :cols], scales.float()


def _plain_values(q, s, block_rows):
    rows, cols = q.shape
    return q * s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_quantised(state, case):
    x = state["x"].float()
    q, s = _plain_quantise(x.t() if case["transpose"] else x, case["block_rows"])
    return {"values": _plain_values(q, s, case["block_rows"]), "scales": s}


def _plain_linear(state, case):
    def q(x, block_rows):                         # what 8 bits keep of x
        return _plain_values(*_plain_quantise(x, block_rows), block_rows)

    x = state["x"].float()
    if not case["train"]:
        return {"y": (q(x, 1) @ _plain_values(state["w8"].float(), state["w8_scales"], 128).t()).bfloat16()}
    w, dy = q(state["w"].float(), 128), state["dy"].float()
    return {"y": (q(x, 1) @ w.t()).bfloat16(), "dx": (q(dy, 1) @ w).bfloat16(),
            "dw": (q(dy.t(), 1) @ q(x.t(), 128).t()).bfloat16()}


def _plain_activation(g, activation):
    """The activation and its derivative."""
    if activation == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if activation == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    if activation == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)
    return torch.clamp(g, min=0.0), (g > 0).to(g.dtype)


def _plain_feed(state, case):
    x, wg, wu, wd = (state[n].float() for n in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _plain_activation(g, case["activation"])
    h = a * u
    out = {"y": (h @ wd.t()).bfloat16()}
    if case["train"]:
        dy = state["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * da, dh * a
        out.update(dx=(dg @ wg + du @ wu).bfloat16(), dwg=(dg.t() @ x).bfloat16(), dwu=(du.t() @ x).bfloat16(),
                   dwd=(dy.t() @ h).bfloat16())
    return out


# ------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    if case["kind"] == "rotate":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["heads"] * case["head_dim"] * size * (4 if case["train"] else 2) + 8), "flops": 0}
    if case["kind"] == "quantise":                # (comes out as the fp32 values that the 8 bits stand for)
        rows, cols = case["rows"], case["cols"]
        scales = -(-rows // case["block_rows"]) * -(-cols // BLOCK)
        return {"bytes": rows * cols * (4 if case["dtype"] == "fp32" else 2) + rows * cols * 4 + 4 * scales, "flops": 0}
    rows, hidden, train = case["rows"], case["hidden"], case["train"]
    if case["kind"] == "feed":
        weights, ends = 3 * hidden * case["inter"], rows * hidden
        return {"bytes": 2 * (weights + 2 * ends) * (2 if train else 1), "flops": (18 if train else 6) * rows * hidden * case["inter"]}
    weight, ends = hidden * case["out"], rows * (hidden + case["out"])
    return {"bytes": 4 * (weight + ends) if train else weight + 2 * ends, "flops": (6 if train else 2) * rows * weight}


# ------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"rotate": _exact_rotate, "feed": _exact_feed, "quantise": _exact_quantised, "linear": _exact_linear}[case["kind"]](state, case)


def _exact_rotate(state, case):
    """Pairs as complex numbers, times e^(i * angle); the gradient is the product with the conjugate."""
    rows, heads, r = case["rows"], case["heads"], case["rotary_dim"]
    inv, factor = _frequencies(case)
    angles = state["positions"].double()[:, None, None] * inv.to(DEVICE)
    wave = torch.polar(torch.full_like(angles, factor), angles)

    def turn(x, wave):
        x = x.detach().double().view(rows, heads, -1).clone()
        z = x[..., :r].reshape(rows, heads, -1, 2) if case["interleaved"] else x[..., :r].reshape(rows, heads, 2, -1).transpose(2, 3)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * wave)
        x[..., :r] = (z if case["interleaved"] else z.transpose(2, 3)).reshape(rows, heads, r)
        return x.view(rows, -1)

    out = {"y": turn(state["x"], wave)}
    if case["train"]:
        out["dx"] = turn(state["dy"], wave.conj())
    return out


def _exact_blocks(x, block_rows):
    """What e4m3 with a power of two for each block keeps of x, and those powers: 3 bits behind the leading one, steps of 2^-9 at
    the least, ties to the even one."""
    x = x.detach().double()
    rows, cols = x.shape
    values, scales = torch.empty_like(x), []
    for r in range(0, rows, block_rows if block_rows > 1 else rows):
        part = x[r:r + block_rows] if block_rows > 1 else x
        row = []
        for c in range(0, cols, BLOCK):
            b = part[:, c:c + BLOCK]
            top = b.abs().amax() if block_rows > 1 else b.abs().amax(1, keepdim=True)
            e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, E4M3_MAX)) / E4M3_MAX))
            e = e + (torch.exp2(e) * E4M3_MAX < top).double()             # (the logarithm may be off by a rounding)
            e = e - (torch.exp2(e - 1) * E4M3_MAX >= top).double() * (top > 0)
            scale = torch.exp2(e.clamp(min=-110))
            y = b / scale
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            values[r:r + part.shape[0], c:c + BLOCK] = torch.round(y / step) * step * scale
            row.append(scale.reshape(-1, 1))
        scales.append(torch.cat(row, 1))
    return values, torch.cat(scales)


def _exact_quantised(state, case):
    x = state["x"].t() if case["transpose"] else state["x"]
    values, scales = _exact_blocks(x, case["block_rows"])
    return {"values": values, "scales": scales}


def _exact_linear(state, case):
    x = state["x"]
    if not case["train"]:
        w8, s = state["w8"].double(), state["w8_scales"].double()
        n, k = w8.shape
        w = w8 * s[torch.arange(n, device=DEVICE) // BLOCK][:, torch.arange(k, device=DEVICE) // BLOCK]
        return {"y": _exact_blocks(x, 1)[0] @ w.T}
    w, dy = _exact_blocks(state["w"], 128)[0], state["dy"]
    return {"y": _exact_blocks(x, 1)[0] @ w.T, "dx": _exact_blocks(dy, 1)[0] @ w,
            "dw": _exact_blocks(dy.t(), 1)[0] @ _exact_blocks(x.t(), 128)[0].T}


def _exact_feed(state, case):
    """Through autograd's own rules, 1024 rows at a time."""
    train = case["train"]
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
           "gelu_tanh": lambda g: torch.nn.functional.gelu(g, approximate="tanh")}[case["activation"]]
    weights = [state[n].detach().double().requires_grad_(train) for n in ("wg", "wu", "wd")]
    sums = [torch.zeros_like(w) for w in weights] if train else []
    ys, dxs = [], []
    for r in range(0, case["rows"], 1024):
        x = state["x"].detach()[r:r + 1024].double().requires_grad_(train)
        with torch.set_grad_enabled(train):
            y = (act(x @ weights[0].T) * (x @ weights[1].T)) @ weights[2].T
        ys.append(y.detach())
        if train:
            dx, *grads = torch.autograd.grad(y, [x, *weights], state["dy"][r:r + 1024].double())
            dxs.append(dx)
            for s, g in zip(sums, grads):
                s += g
    out = {"y": torch.cat(ys)}
    if train:
        out.update(dx=torch.cat(dxs), dwg=sums[0], dwu=sums[1], dwd=sums[2])
    return out
