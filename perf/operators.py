"""The block-scaled (MX) operators as measurable cases: quantisation, RMS norm with the residual's addition, gated
activation and the product with 4-bit weights, in a plain torch form and through the framework's entry points.

Blocks are 32 values along the last axis with one power-of-two scale each; "mxfp8" holds e4m3 elements, "mxfp4" e2m1.
What an operator holds in 8 or 4 bits is returned as the values that it stands for, in bfloat16: an element has at most
four significant bits, so that type holds it as it is."""
import math

import torch

own = False

BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


# ----------------------------------------------------------------------------- the cases


def listed():
    return [
        # the text stage's tokens of two prompts on their way into a 4-bit product
        {"name": "quantise-4bit-small", "op": "quantise", "rows": 154, "k": 1024, "pad": 0, "dtype": "bf16", "fmt": "mxfp4"},
        # the widest token matrix of a large batch
        {"name": "quantise-8bit-large", "op": "quantise", "rows": 16384, "k": 5120, "pad": 0, "dtype": "fp16", "fmt": "mxfp8"},
        # one new token between two layers: latency alone
        {"name": "norm-one-token", "op": "norm", "rows": 1, "k": 1280, "pad": 0, "dtype": "bf16", "fmt": "mxfp8", "res": True},
        # odd rows and an odd width, read out of a wider buffer, 16-bit result
        {"name": "norm-ragged", "op": "norm", "rows": 1001, "k": 1283, "pad": 5, "dtype": "fp16", "fmt": "none", "res": True},
        # a long prompt's residual stream in front of a projection
        {"name": "norm-large", "op": "norm", "rows": 16384, "k": 5120, "pad": 0, "dtype": "bf16", "fmt": "mxfp8", "res": True},
        # the feed-forward gate of two prompts
        {"name": "gate-small", "op": "gate", "rows": 154, "k": 4096, "pad": 0, "dtype": "fp16", "fmt": "mxfp8", "act": "gelu"},
        # the feed-forward gate of a large batch, on to a 4-bit product
        {"name": "gate-large", "op": "gate", "rows": 16384, "k": 5120, "pad": 0, "dtype": "bf16", "fmt": "mxfp4", "act": "silu"},
        # one token through a wide projection: the weights' bytes are the work
        {"name": "linear-one-token", "op": "linear", "rows": 1, "n": 10240, "k": 5120, "pad": 0, "dtype": "bf16", "fmt": "mxfp8", "bias": False, "res": False},
        # one token each of a serving batch, back into the residual stream
        {"name": "linear-batch", "op": "linear", "rows": 48, "n": 5120, "k": 10240, "pad": 0, "dtype": "bf16", "fmt": "mxfp8", "bias": False, "res": True},
        # three prompts: rows that fill no tile, a bias
        {"name": "linear-prompts", "op": "linear", "rows": 231, "n": 1280, "k": 1024, "pad": 0, "dtype": "fp16", "fmt": "mxfp8", "bias": True, "res": False},
        # the gate projection of an image's tokens, 8-bit operands
        {"name": "linear-8bit-large", "op": "linear", "rows": 4096, "n": 10240, "k": 1280, "pad": 0, "dtype": "fp16", "fmt": "mxfp8", "bias": True, "res": False},
        # the largest product, 4-bit operands on both sides
        {"name": "linear-4bit-large", "op": "linear", "rows": 8192, "n": 10240, "k": 5120, "pad": 0, "dtype": "bf16", "fmt": "mxfp4", "bias": False, "res": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantise", "norm", "gate", "linear", "linear", "linear"])
    case = {"op": op, "dtype": rng.choice(sorted(DTYPES)), "pad": rng.choice([0, 0, 8, 24, rng.randint(1, 40)])}
    if op == "linear":
        case["n"] = _log(rng, 64, 10240)
        case["k"] = _log(rng, 64, 10240)
        if rng.random() < 0.5:      # widths of models are mostly round
            case["n"], case["k"] = -(-case["n"] // 64) * 64, -(-case["k"] // 64) * 64
        most = min(8192, 8192 * 10240 * 5120 // (case["n"] * case["k"]))
        case["rows"] = _log(rng, 1, most)
        case.update(fmt=rng.choice(["mxfp4", "mxfp8"]), bias=rng.random() < 0.5, res=rng.random() < 0.5)
        return case
    case["k"] = _log(rng, 32, 10240)
    if rng.random() < 0.5:
        case["k"] = -(-case["k"] // 32) * 32
    most = min(16384, 16384 * 5120 // case["k"])
    case["rows"] = _log(rng, 1, most)
    case["fmt"] = rng.choice(["mxfp4", "mxfp8"] if op == "quantise" else ["mxfp4", "mxfp8", "none"])
    if op == "norm":
        case["res"] = rng.random() < 0.7
    if op == "gate":
        case["act"] = rng.choice(["gelu", "silu"])
    return case


# ----------------------------------------------------------------------------- inputs


def _inputs(case, seed):
    """Every tensor of a case from the seed alone: activations with a few channels ten times the others, as the residual
    streams of transformers have them, weights of the usual spread."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, k, dt = case["rows"], case["k"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    def matrix(width, loud):
        m = randn(rows, width + case["pad"])
        if loud:
            at = torch.randint(0, width, (max(1, width // 100),), generator=g, device="cuda")
            m[:, at] *= 10.0
        return m.to(dt)[:, :width]

    d = {"x": matrix(2 * k if case["op"] == "gate" else k, case["op"] != "gate")}
    if case["op"] == "norm":
        d["gamma"] = 1.0 + 0.1 * randn(k)
        d["res"] = matrix(k, True) if case["res"] else None
    if case["op"] == "linear":
        d["w"] = randn(case["n"], k) * k ** -0.5
        d["bias"] = randn(case["n"]) if case["bias"] else None
        d["res"] = randn(rows, case["n"]).to(dt) if case["res"] else None
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "linear":      # weights are quantised and laid out once, when a model is loaded
        w, bias = d.pop("w"), d.pop("bias")
        if own:
            from stablediffusion_amd import ops
            d["pw"] = ops.pack_linear_mx(w, bias)
        else:
            d["wq"], d["bias"] = _mx_values(w, "mxfp4"), bias
    d["case"] = dict(case)
    return d


# ----------------------------------------------------------------------------- the plain form


def _mx_values(x, fmt):
    """x (float32, [..., K]) -> the float32 values that its MX form stands for."""
    k = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(*x.shape[:-1], -1, BLOCK)
    biased = b.abs().amax(dim=-1, keepdim=True).view(torch.int32) >> 23     # floor(log2 amax) + 127
    byte = (biased - (2 if fmt == "mxfp4" else 8)).clamp(min=0)
    b = b * ((254 - byte) << 23).view(torch.float32)                        # the exact reciprocal of the scale
    if fmt == "mxfp8":
        b = b.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    else:
        a = b.abs().clamp(max=6.0)
        step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
        b = torch.round(a / step) * step * torch.sign(b)
    scale = torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)  # byte 0 is 2^-127, a subnormal
    b = torch.where(biased < 255, b * scale, torch.nan)                     # a block with NaN or infinity in it
    return b.reshape(*x.shape[:-1], -1)[..., :k]


def _held(y, fmt, dtype):
    return y.to(dtype) if fmt == "none" else _mx_values(y, fmt).to(torch.bfloat16)


def _plain(s):
    case = s["case"]
    x, fmt, dt = s["x"].float(), case["fmt"], DTYPES[case["dtype"]]
    if case["op"] == "quantise":
        return {"y": _held(x, fmt, dt)}
    if case["op"] == "norm":
        out = {}
        if s["res"] is not None:
            x = x + s["res"].float()
            out["s"] = x.to(dt)
        y = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * s["gamma"]
        out["y"] = _held(y, fmt, dt)
        return out
    if case["op"] == "gate":
        a, b = x.chunk(2, dim=-1)
        b = 0.5 * b * torch.special.erfc(b * -math.sqrt(0.5)) if case["act"] == "gelu" else b / (1.0 + torch.exp(-b))
        return {"y": _held(a * b, fmt, dt)}
    y = _mx_values(x, fmt) @ s["wq"].t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["res"] is not None:
        y = y + s["res"].float()
    return {"y": y.to(dt)}


def run(state):
    if not own:
        return _plain(state)
    from stablediffusion_amd import ops
    case = state["case"]
    fmt = None if case["fmt"] == "none" else case["fmt"]

    def values(y):
        return y if fmt is None else ops.mx_dequantize(y, torch.bfloat16)

    if case["op"] == "quantise":
        return {"y": values(ops.mx_quantize(state["x"], fmt))}
    if case["op"] == "norm":
        if state["res"] is None:
            return {"y": values(ops.rmsnorm(state["x"], state["gamma"], EPS, fmt=fmt))}
        y, s = ops.rmsnorm(state["x"], state["gamma"], EPS, res=state["res"], fmt=fmt)
        return {"s": s, "y": values(y)}
    if case["op"] == "gate":
        return {"y": values(ops.gated(state["x"], act=case["act"], fmt=fmt))}
    return {"y": ops.linear_mx(state["x"], state["pw"], fmt=fmt, res=state["res"])}


# ----------------------------------------------------------------------------- the work and the definition


def work(case):
    """x, the residual, the parameters read once, the results written once (the weights in 4 bits and their scales)."""
    rows, k = case["rows"], case["k"]
    m = 2 * rows * k
    if case["op"] == "quantise":
        return {"bytes": 2 * m, "flops": 4 * rows * k}
    if case["op"] == "norm":
        return {"bytes": (4 if case["res"] else 2) * m + 4 * k, "flops": 6 * rows * k}
    if case["op"] == "gate":
        return {"bytes": 3 * m, "flops": 12 * rows * k}
    n = case["n"]
    return {"bytes": m + n * k * 17 / 32 + 2 * rows * n * (2 if case["res"] else 1) + (4 * n if case["bias"] else 0),
            "flops": 2 * rows * n * k}


def _power(e):
    """2^e in float64, exactly, for e in [-1022, 1023]."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_mx(x, fmt):
    """The MX values of float64 x from the definition: the block's exponent is that of its largest magnitude less the
    format's largest one; an element is the nearest multiple of its own step, ties to the even multiple."""
    emax, emin, digits, most = (2, 0, 1, 6.0) if fmt == "mxfp4" else (8, -6, 3, 448.0)
    rows, k = x.shape
    full = torch.zeros(rows, -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :k] = x
    for_blocks = full.view(rows, -1, BLOCK)
    top = torch.frexp(for_blocks.abs().max(dim=2, keepdim=True).values)[1] - 1 - emax
    scale = _power(top.clamp(min=-127))
    v = for_blocks / scale
    step = _power((torch.frexp(v)[1] - 1).clamp(min=emin) - digits)
    v = (torch.round(v / step) * step).clamp(-most, most)
    return (v * scale).view(rows, -1)[:, :k]


def exact(case, seed):
    d = _inputs(case, seed)
    x, fmt = d["x"].double(), case["fmt"]

    def held(y):
        return y if fmt == "none" else _exact_mx(y, fmt)

    if case["op"] == "quantise":
        return {"y": held(x)}
    if case["op"] == "norm":
        out = {}
        if d["res"] is not None:
            x = x + d["res"].double()
            out["s"] = x
        out["y"] = held(x / torch.sqrt((x * x).sum(dim=1, keepdim=True) / case["k"] + EPS) * d["gamma"].double())
        return out
    if case["op"] == "gate":
        half = case["k"]
        a, b = x[:, :half], x[:, half:]
        b = b * torch.special.ndtr(b) if case["act"] == "gelu" else b * torch.sigmoid(b)
        return {"y": held(a * b)}
    y = _exact_mx(x, fmt) @ _exact_mx(d["w"].double(), "mxfp4").t()
    if d["bias"] is not None:
        y = y + d["bias"].double()
    if d["res"] is not None:
        y = y + d["res"].double()
    return {"y": y}
