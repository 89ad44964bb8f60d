"""Operators of the 8-bit feed-forward path, as a serving program calls them, beside their plain forms.

  quantize   rows of activations -> 8-bit codes and a scale per row
  linear     x W^T with x quantised per row and W per output channel, sums in integers; or the gated pair act(x G^T) * (x U^T)
  norm       residual update of a block (norm behind it, gate, residual scales) and the norm in front of the next one, its result in the
             activations' type or as 8-bit codes

`exact` restates each from its definition in 64 bits.  Codes are defined by 32-bit arithmetic (one rounding for 127 / a, one for the product, ties
of the final rounding to even), so they have no 64-bit value of their own.
"""
from __future__ import annotations

import math

import torch

import __graft_entry__ as entry

own = False

DTYPES = dict(fp32=torch.float32, fp16=torch.float16, bf16=torch.bfloat16)
TINY = 2.0 ** -116           # rows whose largest value lies below are held as zeros
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token's activations in front of a down projection
        dict(name="quantize 1x3584", kind="quantize", rows=1, cols=3584, dtype="bf16", pad=0),
        # a full prompt pass
        dict(name="quantize 65536x3584", kind="quantize", rows=65536, cols=3584, dtype="fp16", pad=0),
        # one user: gate and up of the next token
        dict(name="glu 1 x 1024 -> 3584", kind="linear", rows=1, cols=1024, out=3584, dtype="fp16", out_dtype="fp16", act="silu", pad=0),
        # a small serving batch through a wider model's output projection
        dict(name="linear 16 x 4096 -> 4096", kind="linear", rows=16, cols=4096, out=4096, dtype="bf16", out_dtype="bf16", act="", pad=0),
        # a full serving batch: logits of a step
        dict(name="linear 128 x 1024 -> 32768", kind="linear", rows=128, cols=1024, out=32768, dtype="fp16", out_dtype="fp32", act="", pad=0),
        # ragged prompts: odd sizes everywhere, rows taken out of a wider buffer
        dict(name="linear 999 x 1000 -> 2313", kind="linear", rows=999, cols=1000, out=2313, dtype="bf16", out_dtype="bf16", act="", pad=24),
        # prompts of a few kilotokens, gate and up
        dict(name="glu 8192 x 1024 -> 3584", kind="linear", rows=8192, cols=1024, out=3584, dtype="fp16", out_dtype="fp16", act="silu", pad=0),
        # a full prompt pass, down projection
        dict(name="linear 65536 x 3584 -> 1024", kind="linear", rows=65536, cols=3584, out=1024, dtype="fp16", out_dtype="fp32", act="", pad=0),
        # one token: residual update and the codes for the next product
        dict(name="norm 1x1024 codes", kind="norm", rows=1, cols=1024, dtype="fp16", x_dtype="fp32", post=False, gate="", codes=True, x_scale=1.0, y_scale=1.0),
        # ragged prompts through a block with norms on both sides and a gate
        dict(name="norm 777x2050 gated", kind="norm", rows=777, cols=2050, dtype="bf16", x_dtype="bf16", post=True, gate="sigmoid", codes=False, x_scale=1.0,
             y_scale=0.25),
        # prompts of a wider model, norms on both sides, learned gate per channel and scaled residual
        dict(name="norm 16384x4096", kind="norm", rows=16384, cols=4096, dtype="bf16", x_dtype="fp32", post=True, gate="channel", codes=False, x_scale=0.9,
             y_scale=1.0),
        # a full prompt pass in front of gate and up
        dict(name="norm 65536x1024 codes", kind="norm", rows=65536, cols=1024, dtype="fp16", x_dtype="fp32", post=False, gate="", codes=True, x_scale=1.0, y_scale=1.0),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    def size(a, b):
        """Half of them multiples of 64, the others as they come."""
        n = log(a, b)
        return max(64, n // 64 * 64) if rng.random() < 0.5 else n

    kind = rng.choice(["quantize", "linear", "linear", "linear", "norm", "norm"])
    dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
    if kind == "quantize":
        cols = size(1, 16384)
        return dict(kind=kind, rows=log(1, max(1, min(65536, 65536 * 3584 // cols // (2 if dtype == "fp32" else 1)))), cols=cols, dtype=dtype,
                    pad=rng.choice([0, 0, 8, 5]))
    if kind == "linear":
        cols, out = size(16, 8192), size(1, 16384)
        act = rng.choice(["", "", "silu", "gelu"])
        if act:
            out = min(out, 8192)
        n = 2 * out if act else out
        most = min(65536, 65536 * 1024 * 3584 // (cols * n), 65536 * 1024 * 2 // (cols + n))
        return dict(kind=kind, rows=log(1, max(1, most)), cols=cols, out=out, dtype=dtype, out_dtype=rng.choice(["fp32", dtype]), act=act,
                    pad=rng.choice([0, 0, 16, 3]))
    cols = size(4, 8192)
    gate = rng.choice(["", "", "channel", "token", "sigmoid"])
    post = rng.random() < 0.5
    # 8-bit results in the forms whose 32-bit steps are all element by element: a norm behind the block or a sigmoid differs in its last place from one
    # summation order or library to the next, and with it a code here and there
    return dict(kind=kind, rows=log(1, max(1, min(65536, 65536 * 512 // cols))), cols=cols, dtype=dtype, x_dtype=rng.choice(["fp32", dtype]), post=post, gate=gate,
                codes=not post and gate != "sigmoid" and rng.random() < 0.6, x_scale=rng.choice([1.0, 1.0, 0.9]), y_scale=rng.choice([1.0, 0.25, 1.5]))


# ---- inputs --------------------------------------------------------------------------------------------------------------------
class Draws:
    """Random tensors on the GPU, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 11)

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, device="cuda", generator=self.g) * std

    def rows(self, rows, cols, dtype, pad=0):
        """Activations: a few channels far larger than the rest, rows of different size, now and then a row of padding (zeros)."""
        x = self.normal(rows, cols + pad)
        loud = torch.rand(cols + pad, device="cuda", generator=self.g) < 0.01
        x *= torch.where(loud, 12.0, 1.0)
        x *= torch.exp(self.normal(rows, 1, std=0.7))
        x *= (torch.rand(rows, 1, device="cuda", generator=self.g) >= 0.01) | (torch.arange(rows, device="cuda")[:, None] == 0)
        return x.to(DTYPES[dtype])[:, :cols]


def inputs(case, seed):
    d = Draws(seed)
    if case["kind"] == "quantize":
        return dict(x=d.rows(case["rows"], case["cols"], case["dtype"], case["pad"]))
    if case["kind"] == "linear":
        w = [d.normal(case["out"], case["cols"], std=0.02).bfloat16() for _ in range(2 if case["act"] else 1)]
        return dict(w=w, x=d.rows(case["rows"], case["cols"], case["dtype"], case["pad"]))
    rows, cols, t = case["rows"], case["cols"], case["dtype"]
    s = dict(x=d.rows(rows, cols, case["x_dtype"]), y=d.rows(rows, cols, t), pre=1.0 + d.normal(cols, std=0.1), post=None, gate=None)
    if case["post"]:
        s["post"] = 1.0 + d.normal(cols, std=0.1)
    if case["gate"]:
        s["gate"] = d.normal(*((cols,) if case["gate"] == "channel" else (rows, cols))).to(DTYPES[t])
    return s


def prepare(case, seed):
    s = dict(case=case, **inputs(case, seed))
    if case["kind"] == "linear":
        w = s.pop("w")
        if own:
            ops = entry.load_ops()
            act = dict(silu=ops.ACT_SILU, gelu=ops.ACT_GELU_TANH).get(case["act"])
            s["layer"] = ops.Int8GatedLinear(w[0], w[1], act) if case["act"] else ops.Int8Linear(w[0])
        else:
            s["layer"] = [plain_codes(m) for m in w]
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------------------
def plain_codes(x):
    """(codes as fp32, scale per row) of fp32, fp16 or bf16 rows."""
    x = x.float()
    a = x.abs().amax(-1, keepdim=True)
    top = torch.full_like(a, 127.0)
    kept = a >= TINY
    inv = torch.where(kept, top / a, torch.zeros_like(a))
    scale = torch.where(kept, a / top, torch.zeros_like(a))
    return torch.round(x * inv), scale[:, 0]


def activation(g, act):
    """SiLU, or GELU in its tanh form, 0.5 g (1 + tanh(p / 2)) = g / (1 + e^-p)."""
    p = g if act == "silu" else math.sqrt(8.0 / math.pi) * (g + 0.044715 * g * g * g)
    return g / (1.0 + torch.exp(-p))


def plain_linear(x, layer, act, dtype):
    codes, scale = plain_codes(x)
    parts = [torch.matmul(codes, cw.t()) * scale[:, None] * sw for cw, sw in layer]
    return (activation(parts[0], act) * parts[1] if act else parts[0]).to(dtype)


def plain_rms(v):
    return torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)


def plain_norm(case, s):
    x, z = s["x"].float(), s["y"].float()
    if s["post"] is not None:
        z = z / plain_rms(z) * s["post"]
    if s["gate"] is not None:
        g = s["gate"].float()
        z = z * (1.0 / (1.0 + torch.exp(-g)) if case["gate"] == "sigmoid" else g)
    new = x * case["x_scale"] + z * case["y_scale"]
    if not case["codes"]:
        return dict(x=new.to(s["x"].dtype), n=(new / plain_rms(new) * s["pre"]).to(DTYPES[case["dtype"]]))
    codes, scale = plain_codes(new * s["pre"])
    return dict(x=new.to(s["x"].dtype), codes=codes.to(torch.int8), scale=scale / plain_rms(new)[:, 0])


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        ops = entry.load_ops()
        if kind == "quantize":
            codes, scale = ops.quantize_rows(state["x"])
            return dict(codes=codes, scale=scale)
        if kind == "linear":
            return state["layer"].forward(state["x"], out_dtype=DTYPES[case["out_dtype"]])
        out = ops.norm_block(state["x"], state["y"], pre_w=state["pre"], post_w=state["post"], gate=state["gate"], sigmoid_gate=case["gate"] == "sigmoid",
                             x_scale=case["x_scale"], y_scale=case["y_scale"], eps=EPS, out_dtype=None if case["codes"] else DTYPES[case["dtype"]])
        return dict(zip(("x", "codes", "scale") if case["codes"] else ("x", "n"), out))
    if kind == "quantize":
        codes, scale = plain_codes(state["x"])
        return dict(codes=codes.to(torch.int8), scale=scale)
    if kind == "linear":
        return plain_linear(state["x"], state["layer"], case["act"], DTYPES[case["out_dtype"]])
    return plain_norm(case, state)


def work(case):
    e = dict(fp32=4, fp16=2, bf16=2)
    rows, cols = case["rows"], case["cols"]
    if case["kind"] == "quantize":
        return dict(bytes=rows * (cols * (e[case["dtype"]] + 1) + 4), flops=3 * rows * cols)
    if case["kind"] == "linear":
        n = case["out"] * (2 if case["act"] else 1)
        return dict(bytes=rows * cols * e[case["dtype"]] + n * (cols + 4) + rows * case["out"] * e[case["out_dtype"]], flops=2 * rows * n * cols)
    one = rows * cols
    gate = {"": 0, "channel": cols}.get(case["gate"], one) * e[case["dtype"]]
    out = one + 4 * rows if case["codes"] else one * e[case["dtype"]]
    return dict(bytes=one * (2 * e[case["x_dtype"]] + e[case["dtype"]]) + gate + 4 * cols * (2 if case["post"] else 1) + out, flops=10 * one)


# ---- definitions in 64 bits -----------------------------------------------------------------------------------------------------------
def codes_by_definition(m):
    """Codes as float64 (what 32-bit arithmetic makes of them) and the scales a / 127."""
    m32 = m.to(torch.float32)
    largest = m32.abs().max(dim=1).values
    held = largest >= TINY
    factor = torch.div(torch.tensor([127.0], device=m.device), largest)
    codes = torch.round(torch.mul(m32, torch.where(held, factor, torch.zeros_like(factor)).unsqueeze(1))).double()
    return codes, torch.where(held, largest.double() / 127.0, torch.zeros_like(largest, dtype=torch.float64))


def exact(case, seed):
    s = inputs(case, seed)
    if case["kind"] == "quantize":
        return dict(codes=None, scale=codes_by_definition(s["x"])[1])
    if case["kind"] == "linear":
        cx, sx = codes_by_definition(s["x"])
        parts = []
        for w in s["w"]:
            cw, sw = codes_by_definition(w)
            out = torch.mm(cx, cw.T)
            out *= sx.unsqueeze(1)
            out *= sw.unsqueeze(0)
            parts.append(out)
        if case["act"] == "silu":
            return parts[0] * torch.sigmoid(parts[0]) * parts[1]
        if case["act"] == "gelu":
            return parts[0] * torch.sigmoid((8.0 / math.pi) ** 0.5 * (parts[0] + 0.044715 * parts[0] ** 3)) * parts[1]
        return parts[0]
    x, z = s["x"].double(), s["y"].double()
    if case["post"]:
        z = z * s["post"].double() * torch.rsqrt((z ** 2).mean(1, keepdim=True) + EPS)
    if case["gate"]:
        g = s["gate"].double()
        z = z * (torch.sigmoid(g) if case["gate"] == "sigmoid" else g)
    new = case["x_scale"] * x + case["y_scale"] * z
    inv = torch.rsqrt((new ** 2).mean(1, keepdim=True) + EPS)
    t = new * s["pre"].double()
    if not case["codes"]:
        return dict(x=new, n=t * inv)
    largest = t.abs().max(dim=1).values
    return dict(x=new, codes=None, scale=torch.where(largest >= TINY, largest / 127.0 * inv[:, 0], torch.zeros_like(largest)))
