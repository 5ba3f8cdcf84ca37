"""The steps of a transformer block around its attention and its MLP, with the weights of its projections in 4 bits, as a user's program calls them.

Each case is one call. `norm`: the step between two blocks' products, a block's output into the residual stream (its own norm behind it, a gate, a factor
of the stream) with the norm in front of the next block, modulated where the model does that. `linear`: a projection whose weights are 4-bit integers
with a scale, and in some checkpoints a zero point, for each group of the contraction. Widths are those of the supported models (1152 PixArt-Sigma,
2240 Sana, 5120 U-Net, 6144 Krea 2) and powers of two; rows run from the single token of a serving step over drafts and prompts to an image with its text.
"""
import math

import torch

own = False      # false: the plain forms below; true: the framework's operators

EPS = 1e-6
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # both norms of a block that has one on either side, one token of a serving step: a launch
        {"name": "norm_token_6144", "op": "norm", "type": "bf16", "items": 1, "rows": 1, "cols": 6144, "post": "rms", "pre": "rms", "modulated": False, "gate": True, "alpha": 1.0},
        # nine prompts of 37 tokens, each with a gate and a modulation of its own
        {"name": "norm_9x37x2240", "op": "norm", "type": "fp16", "items": 9, "rows": 37, "cols": 2240, "post": "none", "pre": "layer", "modulated": True, "gate": True, "alpha": 1.0},
        # two images of a guided step, norms on both sides and a factor of the residual stream
        {"name": "norm_2x2087x1152", "op": "norm", "type": "fp16", "items": 2, "rows": 2087, "cols": 1152, "post": "rms", "pre": "rms", "modulated": True, "gate": True, "alpha": 0.8125},
        # an image block at 1024 x 1024 with 512 tokens of text
        {"name": "norm_4608x6144", "op": "norm", "type": "bf16", "items": 1, "rows": 4608, "cols": 6144, "post": "none", "pre": "layer", "modulated": True, "gate": True, "alpha": 1.0},
        # first product of an MLP for one token: the smallest linear layer
        {"name": "linear_token_1152", "op": "linear", "type": "fp16", "rows": 1, "k": 1152, "n": 4608, "group": 64, "zeros": False, "act": "gelu_tanh", "bias": True, "residual": False},
        # the same of a large model: the weights' bytes are the time
        {"name": "linear_token_6144", "op": "linear", "type": "bf16", "rows": 1, "k": 6144, "n": 16384, "group": 128, "zeros": False, "act": "silu", "bias": False, "residual": False},
        # second product for a draft of 20 tokens, zero points, the residual added
        {"name": "linear_draft_16384", "op": "linear", "type": "bf16", "rows": 20, "k": 16384, "n": 6144, "group": 128, "zeros": True, "act": "none", "bias": False, "residual": True},
        # a 77-token prompt, small groups
        {"name": "linear_77x4608", "op": "linear", "type": "fp16", "rows": 77, "k": 4608, "n": 1152, "group": 32, "zeros": False, "act": "none", "bias": True, "residual": False},
        # a batch of prompts
        {"name": "linear_333x2240", "op": "linear", "type": "bf16", "rows": 333, "k": 2240, "n": 6720, "group": 64, "zeros": True, "act": "silu", "bias": False, "residual": False},
        # an odd number of rows and a contraction that ends inside a group
        {"name": "linear_1031x1160", "op": "linear", "type": "fp16", "rows": 1031, "k": 1160, "n": 4608, "group": 128, "zeros": False, "act": "gelu", "bias": True, "residual": True},
        # second product of a PixArt-Sigma MLP at 1024 x 1024
        {"name": "linear_4096x4608", "op": "linear", "type": "fp16", "rows": 4096, "k": 4608, "n": 1152, "group": 64, "zeros": False, "act": "none", "bias": True, "residual": True},
        # first product of the MLP of a large image model: the matrix pipes are the time
        {"name": "linear_4608x6144", "op": "linear", "type": "bf16", "rows": 4608, "k": 6144, "n": 16384, "group": 128, "zeros": False, "act": "gelu_tanh", "bias": True, "residual": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    most = max(2 * c["rows"] * c["k"] * c["n"] for c in listed() if c["op"] == "linear")
    widest = max(c["items"] * c["rows"] * c["cols"] for c in listed() if c["op"] == "norm")
    while True:
        rows, type_ = _log_int(rng, 1, 4608), rng.choice(["fp16", "bf16"])
        if rng.random() < 0.4:
            items, cols = _log_int(rng, 1, 12), 8 * _log_int(rng, 16, 2048)
            if items * rows * cols <= widest:
                return {"op": "norm", "type": type_, "items": items, "rows": rows, "cols": cols, "post": rng.choice(["none", "rms", "layer"]), "pre": rng.choice(["rms", "layer"]),
                        "modulated": rng.random() < 0.6, "gate": rng.random() < 0.8, "alpha": rng.choice([1.0, 1.0, 0.8125, 1.7])}
            continue
        k, n = 8 * _log_int(rng, 16, 2048), 8 * _log_int(rng, 16, 2048)
        if 2 * rows * k * n <= most:
            return {"op": "linear", "type": type_, "rows": rows, "k": k, "n": n, "group": rng.choice([32, 64, 128, 128]), "zeros": rng.random() < 0.5,
                    "act": rng.choice(["none", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.6, "residual": rng.random() < 0.5}


def _four_bits(w, group, zeros, t):
    """w (n, k) as a 4-bit checkpoint holds it: two integers to a byte, the first in the low half, and a scale (and a zero point) of each group."""
    n, k = w.shape
    pad = -k % group
    blocks = torch.nn.functional.pad(w, (0, pad)).view(n, -1, group)
    if zeros:
        low, high = blocks.amin(dim=2).clamp(max=0), blocks.amax(dim=2).clamp(min=0)
        scales = ((high - low) / 15).clamp(min=1e-6).to(t)
        zero = torch.round(-low / scales.float()).clamp(0, 15)
    else:
        scales = (blocks.abs().amax(dim=2) / 7.5).clamp(min=1e-6).to(t)
        zero = torch.full_like(scales, 8, dtype=torch.float32)
    q = torch.round(blocks / scales.float()[:, :, None] + zero[:, :, None]).clamp(0, 15).to(torch.uint8).view(n, -1)[:, :k]
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scales, zero.to(torch.uint8) if zeros else None


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % 100003) + 23)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "norm":
        items, rows, cols = case["items"], case["rows"], case["cols"]
        # a few channels of a residual stream are much larger than the others
        loud = torch.exp(1.2 * normal(cols).clamp(-2.5, 2.5))
        s["x"] = (normal(items, rows, cols) * loud + 0.3).to(t)
        s["branch"] = (0.5 * normal(items, rows, cols) * loud).to(t)
        # gate, scale and shift are cut out of one row of modulation for each item, as the models make them
        vectors = (0.5 * normal(items, 6 * cols)).to(t)
        s["gate"] = vectors[:, :cols] if case["gate"] else None
        s["scale"], s["shift"] = (vectors[:, cols:2 * cols], vectors[:, 2 * cols:3 * cols]) if case["modulated"] else (None, None)
        s["post_gain"] = (1 + 0.2 * normal(cols)).to(t) if case["post"] == "rms" else None
        s["gain"] = (1 + 0.2 * normal(cols)).to(t) if case["pre"] == "rms" else None
        return s
    m, k, n = case["rows"], case["k"], case["n"]
    x = normal(m, k)
    # (hidden rows behind an activation are not centred)
    s["x"] = (x * torch.sigmoid(x) if k > n else x).to(t)
    s["q"], s["scales"], s["zeros"] = _four_bits(normal(n, k) / math.sqrt(k), case["group"], case["zeros"], t)
    s["bias"] = (0.5 * normal(n)).to(t) if case["bias"] else None
    s["residual"] = normal(m, n).to(t) if case["residual"] else None
    if own:
        import brodiffusion_amd as bd
        s["w"] = bd.pack_int4(s["q"], s["scales"], s["zeros"], group=case["group"])
    return s


def _plain_norm(x, kind, gain):
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    return x if gain is None else x * gain.float()


def _plain(s):
    case, t = s["case"], TYPES[s["case"]["type"]]
    if case["op"] == "norm":
        b = s["branch"].float()
        if case["post"] != "none":
            b = _plain_norm(b, case["post"], s["post_gain"])
        if s["gate"] is not None:
            b = b * s["gate"].float()[:, None, :]
        total = (s["x"].float() * case["alpha"] + b).to(t)
        y = _plain_norm(total.float(), case["pre"], s["gain"])
        if case["modulated"]:
            y = y * (1 + s["scale"].float()[:, None, :]) + s["shift"].float()[:, None, :]
        return {"sum": total, "values": y.to(t)}
    n, k = case["n"], case["k"]
    q = torch.stack((s["q"] & 15, s["q"] >> 4), dim=2).view(n, k).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(case["group"], dim=1)[:, :k]
    w = (q - zero) * s["scales"].float().repeat_interleave(case["group"], dim=1)[:, :k]
    y = torch.matmul(s["x"].float(), w.t())
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
        return bd.linear_int4(s["x"], s["w"], s["bias"], activation=case["act"], residual=s["residual"])
    total, values = bd.gate_add_norm(s["x"], s["branch"], gate=s["gate"], post=case["post"], post_gain=s["post_gain"], residual_scale=case["alpha"], norm=case["pre"], gain=s["gain"],
                                     scale=s["scale"], shift=s["shift"], eps=EPS)
    return {"sum": total, "values": values}


def work(case):
    if case["op"] == "linear":
        m, k, n, groups = case["rows"], case["k"], case["n"], -(-case["k"] // case["group"])
        weights = n * k // 2 + n * groups * (3 if case["zeros"] else 2)
        return {"bytes": weights + 2 * m * k + 2 * m * n * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    count, cols = case["items"] * case["rows"] * case["cols"], case["cols"]
    vectors = case["items"] * cols * ((1 if case["gate"] else 0) + (2 if case["modulated"] else 0)) + cols * ((1 if case["post"] == "rms" else 0) + (1 if case["pre"] == "rms" else 0))
    return {"bytes": 2 * (4 * count + vectors), "flops": 16 * count}


def _exact_norm(x, kind, gain):
    if kind == "layer":
        x = x - x.sum(dim=-1, keepdim=True) / x.shape[-1]
    x = x * (x.pow(2).sum(dim=-1, keepdim=True) / x.shape[-1] + EPS).pow(-0.5)
    return x if gain is None else x * gain.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        b = s["branch"].double()
        if case["post"] != "none":
            b = _exact_norm(b, case["post"], s["post_gain"])
        if s["gate"] is not None:
            b = b * s["gate"].double().unsqueeze(1)
        total = s["x"].double() * case["alpha"] + b
        y = _exact_norm(total.to(TYPES[case["type"]]).double(), case["pre"], s["gain"])     # the norm is of the stored sum
        if case["modulated"]:
            y = y + y * s["scale"].double().unsqueeze(1) + s["shift"].double().unsqueeze(1)
        return {"sum": total, "values": y}
    n, k, group = case["n"], case["k"], case["group"]
    w = torch.empty(n, k, dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = s["q"] % 16, s["q"] // 16
    for g in range(s["scales"].shape[1]):
        part = w[:, g * group:(g + 1) * group]
        part -= 8 if s["zeros"] is None else s["zeros"][:, g:g + 1].double()
        part *= s["scales"][:, g:g + 1].double()
    y = s["x"].double() @ w.t()
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
