"""The operators around the 8-bit and fused-epilogue projections of a transformer block, as a user's program calls them.

Each case is one call: the residual's addition with the RMS norm behind it (rows of the tensor type, or 8-bit rows with a scale each),
rows to 8 bits, and a linear layer with bias, activation and residual in its epilogue (16-bit operands, INT8 weights, or both operands
INT8). Widths are those of the supported models (1152 PixArt-Sigma, 2240 Sana, 5120 U-Net, 6144 Krea 2) and powers of two; rows run
from the single token of a serving step over drafts and prompts to an image with its text.
"""
import math

import torch

own = False      # false: the plain forms below; true: the framework's operators

EPS = 1e-6
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the norm in front of an 8-bit projection, one token of a serving step: a launch
        {"name": "norm_int8_token_6144", "op": "norm", "int8": True, "type": "bf16", "rows": 1, "cols": 6144},
        # the same for a batch of prompts, an odd number of rows
        {"name": "norm_int8_333x2240", "op": "norm", "int8": True, "type": "fp16", "rows": 333, "cols": 2240},
        # the norm of a 16-bit block at 1024 x 1024 with 512 tokens of text
        {"name": "norm_4608x6144", "op": "norm", "int8": False, "type": "bf16", "rows": 4608, "cols": 6144},
        # hidden rows of a drafted continuation on their way into the second product of an MLP
        {"name": "rows_int8_24x16384", "op": "rows", "type": "bf16", "rows": 24, "cols": 16384},
        # hidden rows of an image block with a 77-token prompt
        {"name": "rows_int8_4173x4608", "op": "rows", "type": "fp16", "rows": 4173, "cols": 4608},
        # first product of an MLP for one token, 16-bit weights: the smallest linear layer
        {"name": "linear_token_1152", "op": "linear", "kind": "w16", "type": "bf16", "rows": 1, "k": 1152, "n": 4608, "act": "gelu_tanh", "bias": True, "residual": False},
        # the same of a large model with both operands in 8 bits: the weights' bytes are the time
        {"name": "linear_token_6144_w8a8", "op": "linear", "kind": "w8a8", "type": "bf16", "rows": 1, "k": 6144, "n": 16384, "act": "silu", "bias": False, "residual": False},
        # second product for a draft of 20 tokens, INT8 weights, the residual added
        {"name": "linear_draft_16384_w8", "op": "linear", "kind": "w8", "type": "bf16", "rows": 20, "k": 16384, "n": 6144, "act": "none", "bias": False, "residual": True},
        # an odd number of rows and a contraction that is no multiple of a tile's depth
        {"name": "linear_1031x1160", "op": "linear", "kind": "w16", "type": "fp16", "rows": 1031, "k": 1160, "n": 4608, "act": "gelu_tanh", "bias": True, "residual": True},
        # second product of a PixArt-Sigma MLP at 1024 x 1024 in 8 bits
        {"name": "linear_4096x4608_w8a8", "op": "linear", "kind": "w8a8", "type": "fp16", "rows": 4096, "k": 4608, "n": 1152, "act": "none", "bias": True, "residual": True},
        # first product of the MLP of a large image model, 16 bits and 8 bits: the matrix pipes are the time
        {"name": "linear_4608x6144", "op": "linear", "kind": "w16", "type": "bf16", "rows": 4608, "k": 6144, "n": 16384, "act": "gelu_tanh", "bias": True, "residual": False},
        {"name": "linear_4608x6144_w8a8", "op": "linear", "kind": "w8a8", "type": "bf16", "rows": 4608, "k": 6144, "n": 16384, "act": "gelu", "bias": True, "residual": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    most = max(2 * c["rows"] * c["k"] * c["n"] for c in listed() if c["op"] == "linear")
    widest = max(c["rows"] * c["cols"] for c in listed() if c["op"] != "linear")
    while True:
        op, rows, type_ = rng.choice(["norm", "rows", "linear", "linear", "linear"]), _log_int(rng, 1, 4608), rng.choice(["fp16", "bf16"])
        if op != "linear":
            cols = 8 * _log_int(rng, 40, 2048)
            if rows * cols <= widest:
                return {"op": op, "type": type_, "rows": rows, "cols": cols, **({"int8": rng.random() < 0.6} if op == "norm" else {})}
            continue
        kind = rng.choice(["w16", "w8", "w8a8"])
        step = 16 if kind == "w8a8" else 8
        k, n = step * _log_int(rng, 320 // step, 16384 // step), 8 * _log_int(rng, 40, 2048)
        if 2 * rows * k * n <= most:
            return {"op": op, "kind": kind, "type": type_, "rows": rows, "k": k, "n": n, "act": rng.choice(["none", "gelu", "gelu_tanh", "silu"]),
                    "bias": rng.random() < 0.6, "residual": rng.random() < 0.5}


def _integers(x):
    """Rows of x as 8-bit integers, and the scale of each: what a user's quantised checkpoint or the operator in front holds."""
    most = x.abs().amax(dim=1, keepdim=True)
    return torch.round(x * (127.0 / most)).to(torch.int8), (most / 127.0).squeeze(1).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % 100003) + 17)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] != "linear":
        # a few channels of a residual stream are much larger than the others
        loud = torch.exp(1.2 * normal(case["cols"]).clamp(-2.5, 2.5))
        s["x"] = (normal(case["rows"], case["cols"]) * loud).to(t)
        if case["op"] == "norm":
            s["r"] = (0.5 * normal(case["rows"], case["cols"]) * loud).to(t)
            s["gain"] = (1 + 0.2 * normal(case["cols"])).to(t)
        return s
    m, k, n = case["rows"], case["k"], case["n"]
    x, w = normal(m, k), normal(n, k) / math.sqrt(k)
    if case["kind"] == "w8a8":
        s["x"], s["x_scales"] = _integers(x)
    else:
        s["x"], s["x_scales"] = x.to(t), None
    if case["kind"] == "w16":
        s["w"], s["w_scales"] = w.to(t), None
    else:
        s["w"], s["w_scales"] = _integers(w)
    s["bias"] = (0.5 * normal(n)).to(t) if case["bias"] else None
    s["residual"] = normal(m, n).to(t) if case["residual"] else None
    return s


def _plain_rows_int8(z, rstd):
    most = z.abs().amax(dim=1, keepdim=True)
    some = torch.where(most > 0, most, torch.ones_like(most))
    # (64 bits: which integer a value next to the middle of two becomes must not hang on the division's rounding)
    q = torch.round(z.double() * 127.0 / some.double()).float()
    scale = most * rstd / 127.0
    return q * scale, scale.squeeze(1)


def _plain(s):
    case, t = s["case"], TYPES[s["case"]["type"]]
    if case["op"] == "rows":
        x = s["x"].float()
        values, scales = _plain_rows_int8(x, torch.ones_like(x[:, :1]))
        return {"values": values, "scales": scales}
    if case["op"] == "norm":
        total = (s["x"].float() + s["r"].float()).to(t)
        h, gain = total.float(), s["gain"].float()
        rstd = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
        if not case["int8"]:
            return {"sum": total, "values": (h * rstd * gain).to(t)}
        values, scales = _plain_rows_int8(h * gain, rstd)
        return {"sum": total, "values": values, "scales": scales}
    y = torch.matmul(s["x"].float(), s["w"].float().t())
    if s["w_scales"] is not None:
        y = y * s["w_scales"]
    if s["x_scales"] is not None:
        y = y * s["x_scales"][:, None]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = 0.5 * y * torch.erfc(y * -math.sqrt(0.5))
    elif case["act"] == "gelu_tanh":
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(t)


def run(s):
    if not own:
        return _plain(s)
    import brodiffusion_amd as bd
    case = s["case"]
    if case["op"] == "linear":
        return bd.linear_act(s["x"], s["w"], s["bias"], activation=case["act"], residual=s["residual"], x_scales=s["x_scales"], w_scales=s["w_scales"],
                             dtype=TYPES[case["type"]])
    if case["op"] == "norm" and not case["int8"]:
        total, values = bd.add_rms_norm(s["x"], s["r"], s["gain"], EPS)
        return {"sum": total, "values": values}
    # (8-bit rows are compared as the numbers that they stand for: the product with their scale is part of the pass)
    if case["op"] == "norm":
        total, q, scales = bd.add_rms_norm_int8(s["x"], s["r"], s["gain"], EPS)
        return {"sum": total, "values": torch.mul(q, scales[:, None]), "scales": scales}
    q, scales = bd.quantize_rows_int8(s["x"])
    return {"values": torch.mul(q, scales[:, None]), "scales": scales}


def work(case):
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        x_bytes, w_bytes = (1 if case["kind"] == "w8a8" else 2), (2 if case["kind"] == "w16" else 1)
        return {"bytes": m * k * x_bytes + n * k * w_bytes + 2 * m * n * (2 if case["residual"] else 1) + 2 * n, "flops": 2 * m * n * k}
    count = case["rows"] * case["cols"]
    if case["op"] == "rows":
        return {"bytes": 2 * count + count + 4 * case["rows"], "flops": 4 * count}
    return {"bytes": 4 * count + 2 * count + (1 if case["int8"] else 2) * count + 2 * case["cols"], "flops": 8 * count}


def _exact_rows(z, rstd):
    """Rows z in 64 bits as multiples of their largest magnitude / 127, times rstd."""
    a = z.abs().max(dim=1).values
    steps = torch.zeros_like(z)
    some = a > 0
    steps[some] = torch.round(127 * z[some] / a[some, None])
    scales = a * rstd / 127
    return steps * scales[:, None], scales


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        values, scales = _exact_rows(s["x"].double(), 1.0)
        return {"values": values, "scales": scales}
    if case["op"] == "norm":
        total = s["x"].double() + s["r"].double()
        h = total.to(TYPES[case["type"]]).double()     # the norm is of the stored sum
        rstd = (h.pow(2).sum(dim=1) / case["cols"] + EPS).pow(-0.5)
        z = h * s["gain"].double()
        if not case["int8"]:
            return {"sum": total, "values": z * rstd[:, None]}
        values, scales = _exact_rows(z, rstd)
        return {"sum": total, "values": values, "scales": scales}
    x, w = s["x"].double(), s["w"].double()
    if s["x_scales"] is not None:
        x *= s["x_scales"].double()[:, None]
    if s["w_scales"] is not None:
        w *= s["w_scales"].double()[:, None]
    y = x @ w.t()
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "gelu":
        y = y * torch.erfc(y * -(0.5 ** 0.5)) / 2
    elif case["act"] == "gelu_tanh":
        y = y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y.pow(3)))) / 2
    if s["residual"] is not None:
        y += s["residual"].double()
    return y
