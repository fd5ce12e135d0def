"""Cases of the 4-bit path: rows and matrices in microscaled 4-bit floats, their
products, the norms around a sublayer with its gate and residual scale, and the
feed-forward that these make together.

`run` computes a case in its plain form (torch operations in float32) or, where
`own` is true, with the calls that a user makes of janas_b200.csrc.ops.  Layer sizes are
those of the library's benchmark (hidden 2,560, feed-forward 9,728, q|k|v 6,144).
"""
import math

import torch

own = False

F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"float32": F32, "bfloat16": BF16}
EPS = 1e-6


def listed():
    return [
        # a decode step's rows ahead of a 4-bit product: latency
        {"name": "quantize rows of 8 users", "op": "quantize", "n": 8, "k": 2560, "dtype": "bfloat16"},
        # float32 rows of a length that is no multiple of a block, or of anything
        {"name": "quantize odd rows", "op": "quantize", "n": 333, "k": 1037, "dtype": "float32"},
        # a gate-up matrix as it is brought to 4 bits when a model is opened
        {"name": "quantize a weight", "op": "quantize", "n": 19456, "k": 2560, "dtype": "bfloat16"},
        # q|k|v of one user's next token
        {"name": "linear of one token", "op": "linear", "n": 1, "m": 6144, "k": 2560, "dtype": "bfloat16",
         "out": "float32"},
        # gate-up of a decode step of eight users: a stream of weights
        {"name": "linear of 8 users", "op": "linear", "n": 8, "m": 19456, "k": 2560, "dtype": "bfloat16",
         "out": "float32"},
        # no size a multiple of a tile, float32 rows
        {"name": "linear odd", "op": "linear", "n": 77, "m": 1003, "k": 1037, "dtype": "float32", "out": "float32"},
        # down of a prompt: a long k and few features
        {"name": "linear down of a prompt", "op": "linear", "n": 2048, "m": 2560, "k": 9728, "dtype": "bfloat16",
         "out": "float32"},
        # gate-up of a prompt, the largest product of a layer
        {"name": "linear gate-up of a prompt", "op": "linear", "n": 2048, "m": 19456, "k": 2560, "dtype": "bfloat16",
         "out": "bfloat16"},
        # between two sublayers of a decode step, RMS norms with the gate of a sandwich block
        {"name": "norms of 8 users", "op": "norms", "n": 8, "dm": 2560, "rms": True, "gate": True, "out": "bfloat16"},
        # the same of a prompt, with layer norms
        {"name": "norms of a prompt", "op": "norms", "n": 2048, "dm": 2560, "rms": False, "gate": True,
         "out": "bfloat16"},
        # a whole feed-forward in 4 bits, from the mixer's result to its own: a decode step
        {"name": "feed-forward of 8 users", "op": "ffn", "n": 8, "dm": 2560, "ff": 9728, "rms": True, "gate": False},
        # and a prompt
        {"name": "feed-forward of a prompt", "op": "ffn", "n": 2048, "dm": 2560, "ff": 9728, "rms": True,
         "gate": False},
    ]


def _spread(rng, low, high):
    """A size between low and high, evenly over the logarithm; one in three a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.33 and v >= 64:
        v -= v % 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "norms", "ffn"])
    dtype = rng.choice(["float32", "bfloat16"])
    n = _spread(rng, 1, 2048)
    if op == "quantize":
        return {"op": op, "n": _spread(rng, 1, 16384), "k": _spread(rng, 16, 2560), "dtype": dtype}
    if op == "linear":
        m, k = _spread(rng, 16, 19456), _spread(rng, 16, 9728)
        while n * m * k > 2048 * 19456 * 2560:
            m = max(16, m // 2)
        return {"op": op, "n": n, "m": m, "k": k, "dtype": dtype, "out": rng.choice(["float32", "bfloat16"])}
    rms, gate = rng.random() < 0.6, rng.random() < 0.6
    if op == "norms":
        return {"op": op, "n": n, "dm": _spread(rng, 32, 2560), "rms": rms, "gate": gate, "out": dtype}
    return {"op": op, "n": n, "dm": _spread(rng, 64, 2560), "ff": _spread(rng, 64, 9728), "rms": rms, "gate": gate}


def _normal(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _rows(g, n, k, dtype):
    """Rows as a norm leaves them: mostly around one, a few channels many times larger."""
    x = torch.randn(n, k, generator=g, device="cuda")
    x[:, :: max(1, k // 5)] *= 8.0
    return x.to(dtype)


def _weight(g, m, k):
    """A matrix of 4-bit values, held in bfloat16 (exactly), as a 4-bit checkpoint stands for it."""
    return _plain_values(_normal(g, m, k, scale=0.02)).to(BF16)


def _kept(w):
    """The weight as the user's program keeps it: the library's 4-bit matrix, or the values as floats."""
    if own:
        from janas_b200.csrc import ops
        return ops.mx4_quantize(w)
    return w.float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, n = case["op"], case["n"]
    if op == "quantize":
        return {"case": case, "x": _rows(g, n, case["k"], TYPES[case["dtype"]])}
    if op == "linear":
        return {"case": case, "a": _rows(g, n, case["k"], TYPES[case["dtype"]]),
                "w": _kept(_weight(g, case["m"], case["k"]))}
    dm = case["dm"]
    s = {"case": case, "x": _normal(g, n, dm, scale=2.0), "y": _normal(g, n, dm),
         "post_w": 1 + _normal(g, dm, scale=0.1), "scale": 0.5 + _normal(g, dm, scale=0.1),
         "next_w": 1 + _normal(g, dm, scale=0.1), "post_b": None, "next_b": None, "g": None, "g_bias": None}
    if not case["rms"]:
        s["post_b"], s["next_b"] = _normal(g, dm, scale=0.02), _normal(g, dm, scale=0.02)
    if case["gate"]:
        s["g"], s["g_bias"] = _normal(g, n, dm), _normal(g, dm, scale=0.1)
    if op == "ffn":
        s["gate_up"] = _kept(_weight(g, 2 * case["ff"], dm))
        s["down"] = _kept(_weight(g, dm, case["ff"]))
    return s


# ------------------------------------------------------------------ the plain form, in float32
def _plain_values(x):
    """What x stands for in blocks of 32 with a power of two each and eight magnitudes up to 6."""
    x = x.float()
    n, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % 32)).view(n, -1, 32)
    # the power of two's exponent + 127, from the bits of the largest magnitude
    e = ((b.abs().amax(-1, keepdim=True).view(torch.int32) >> 23) - 2).clamp(min=0)
    power = torch.where(e > 0, (e << 23).view(F32), 2.0 ** -127)
    v = b * ((254 - e) << 23).view(F32)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.copysign(q, v) * power).view(n, -1)[:, :k].contiguous()


def _plain_norm(t, w, b, rms):
    if not rms:
        t = t - t.mean(-1, keepdim=True)
    t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * w
    return t if b is None else t + b


def _plain_norms(s):
    """The residual stream with the sublayer's result added, in place, and its next norm."""
    rms, t = s["case"]["rms"], s["y"]
    if s["g"] is not None:
        t = t * torch.sigmoid(s["g"] + s["g_bias"])
    s["x"] += s["scale"] * _plain_norm(t, s["post_w"], s["post_b"], rms)
    return _plain_norm(s["x"], s["next_w"], s["next_b"], rms)


def run(s):
    case = s["case"]
    if own:
        return _own(s)
    if case["op"] == "quantize":
        return _plain_values(s["x"]).to(BF16)
    if case["op"] == "linear":
        return (_plain_values(s["a"]) @ s["w"].t()).to(TYPES[case["out"]])
    h = _plain_norms(s)
    if case["op"] == "norms":
        return {"x": s["x"], "h": h.to(TYPES[case["out"]])}
    z = _plain_values(h) @ s["gate_up"].t()
    gate, up = z[:, :case["ff"]], z[:, case["ff"]:]
    return {"x": s["x"], "y": (_plain_values(gate * torch.sigmoid(gate) * up) @ s["down"].t()).to(BF16)}


# ------------------------------------------------------------------ the library's calls
def _own(s):
    from janas_b200.csrc import ops
    case = s["case"]
    if case["op"] == "quantize":
        return ops.mx4_values(ops.mx4_quantize(s["x"]), BF16)
    if case["op"] == "linear":
        return ops.linear_mx4(s["a"], s["w"], TYPES[case["out"]])
    h = ops.norm_residual_norm(s["x"], s["y"], s["post_w"], s["next_w"], EPS, rms=case["rms"], y_gate=s["g"],
                               gate_bias=s["g_bias"], scale=s["scale"], post_bias=s["post_b"], next_bias=s["next_b"],
                               out="mx4" if case["op"] == "ffn" else TYPES[case["out"]])
    if case["op"] == "norms":
        return {"x": s["x"], "h": h}
    z = ops.linear_mx4(h, s["gate_up"])
    return {"x": s["x"], "y": ops.linear_mx4(ops.mx4_gated_unit(z), s["down"], BF16)}


def work(case):
    op, n = case["op"], case["n"]
    size = {"float32": 4, "bfloat16": 2}
    packed = 17 / 32
    if op == "quantize":
        return {"bytes": n * case["k"] * (size[case["dtype"]] + 2), "flops": 2 * n * case["k"]}
    if op == "linear":
        m, k = case["m"], case["k"]
        return {"bytes": n * k * size[case["dtype"]] + m * k * packed + n * m * size[case["out"]], "flops": 2 * n * m * k}
    dm = case["dm"]
    rows = n * dm * (4 + 4 + 4 + (4 if case["gate"] else 0))
    if op == "norms":
        return {"bytes": rows + n * dm * size[case["out"]], "flops": 20 * n * dm}
    ff = case["ff"]
    return {"bytes": rows + n * dm * 2 + packed * 3 * ff * dm, "flops": 2 * n * 3 * ff * dm}


# ------------------------------------------------------------------ the definition, in 64 bits
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values(x):
    """Each value is the nearest of sign * grid * 2^e, a tie going to the one whose index in the grid is even."""
    n, k = x.shape
    out = torch.zeros(n, -(-k // 32) * 32, dtype=torch.float64, device=x.device)
    out[:, :k] = x.double()
    out = out.view(-1, 32)
    powers = torch.tensor([2.0 ** i for i in range(-127, 128)], dtype=torch.float64, device=x.device)
    for at in range(0, out.shape[0], 1 << 18):
        b = out[at:at + (1 << 18)]
        top = b.abs().max(dim=1).values
        # top = f 2^e with f in [0.5, 1): two below the largest power of two in it
        scale = powers[(torch.frexp(top).exponent.long() - 3).clamp(min=-127) + 127]
        v = b.abs() / scale[:, None]
        best = torch.zeros_like(v)
        for i in range(7):
            low, high = _GRID[i], _GRID[i + 1]
            middle = (low + high) / 2
            best = torch.where(v >= middle if i % 2 else v > middle, torch.full_like(v, high), best)
        b.copy_(torch.sign(b) * best * scale[:, None])
    return out.view(n, -1)[:, :k]


def _exact_norm(t, w, b, rms):
    mean = torch.zeros_like(t[:, :1]) if rms else t.sum(1, keepdim=True) / t.shape[1]
    d = t - mean
    r = d / torch.sqrt((d ** 2).sum(1, keepdim=True) / t.shape[1] + EPS) * w.double()
    return r + b.double() if b is not None else r


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "quantize":
        return _exact_values(s["x"])
    if op == "linear":
        return torch.matmul(_exact_values(s["a"]), s["w"].double().T)
    y = s["y"].double()
    if s["g"] is not None:
        y = y / (1 + torch.exp(-(s["g"].double() + s["g_bias"].double())))
    x = s["x"].double() + s["scale"].double() * _exact_norm(y, s["post_w"], s["post_b"], case["rms"])
    h = _exact_norm(x, s["next_w"], s["next_b"], case["rms"])
    if op == "norms":
        return {"x": x, "h": h}
    z = torch.matmul(_exact_values(h), s["gate_up"].double().T)
    gate, up = z.chunk(2, dim=1)
    unit = gate / (1 + torch.exp(-gate)) * up
    return {"x": x, "y": torch.matmul(_exact_values(unit), s["down"].double().T)}
