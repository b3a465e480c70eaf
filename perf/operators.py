"""Dense operators beside the routed layer, as measured cases.

The gated feed-forward block (the shared expert that every token passes),
its training step, the 4-bit microscaled quantiser, the product of two
4-bit operands and the 4-bit serving form of the block. `run` computes a
case either in its plain form (elementary torch operations in 32 bits,
rounded once) or, with `own` set, through the package's entry points;
`exact` restates it in 64 bits.

Layouts shared by both forms: w13 is [2I, H] with the up rows first and the
gate rows after them, w2 is [H, I]. A 4-bit matrix [R, K] is held as codes
uint8 [R, K / 2] (element 2j in the low nibble of byte j) and exponent bytes
uint8 [ceil(R / 128), ceil(K / 128), 32, 4, 4]: the byte of row r and
32-column block b is at [r // 128, b // 4, r % 32, r % 128 // 32, b % 4].
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a chat through the shared expert: latency of two weight streams
        {"name": "ffn_token_1", "op": "ffn", "t": 1, "h": 7168, "i": 2048, "type": "bf16", "act": "silu"},
        # a full decode batch, in the other 16-bit type and activation
        {"name": "ffn_decode_64", "op": "ffn", "t": 64, "h": 7168, "i": 2048, "type": "fp16", "act": "gelu_tanh"},
        # a ragged prompt of the benchmark's sequence lengths
        {"name": "ffn_prompt_901", "op": "ffn", "t": 901, "h": 7168, "i": 2048, "type": "bf16", "act": "silu"},
        # the expert-parallel batch: large prefill
        {"name": "ffn_prefill_8192", "op": "ffn", "t": 8192, "h": 7168, "i": 2048, "type": "bf16", "act": "silu"},
        # fine-tuning step of a small block with odd sizes and a ragged batch
        {"name": "train_ragged_333", "op": "train", "t": 333, "h": 1032, "i": 520, "type": "fp16", "act": "gelu_tanh"},
        # training step of the shared expert on the prefill batch
        {"name": "train_4096", "op": "train", "t": 4096, "h": 7168, "i": 2048, "type": "bf16", "act": "silu"},
        # activations of a decode batch into 4 bits
        {"name": "quantize_53", "op": "quantize", "t": 53, "h": 7168, "type": "fp16"},
        # activations of the stress batch into 4 bits
        {"name": "quantize_16384", "op": "quantize", "t": 16384, "h": 7168, "type": "bf16"},
        # one token through a 4-bit projection
        {"name": "mx_linear_1", "op": "mx_linear", "t": 1, "n": 4096, "h": 7168, "type": "bf16"},
        # a prefill batch through a 4-bit projection
        {"name": "mx_linear_8192", "op": "mx_linear", "t": 8192, "n": 4096, "h": 7168, "type": "bf16"},
        # a decode batch through the block with 4-bit weights
        {"name": "mx_ffn_16", "op": "mx_ffn", "t": 16, "h": 7168, "i": 2048, "type": "bf16", "act": "silu"},
        # a prefill batch through the block with 4-bit weights
        {"name": "mx_ffn_4096", "op": "mx_ffn", "t": 4096, "h": 7168, "i": 2048, "type": "bf16", "act": "silu"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "train", "quantize", "mx_linear", "mx_ffn"])
    kind = rng.choice(["bf16", "fp16"])
    if op in ("ffn", "train"):
        top = 8192 if op == "ffn" else 4096
        return {"op": op, "t": _log(rng, 1, top), "h": 8 * _log(rng, 32, 896), "i": 8 * _log(rng, 16, 256),
                "type": kind, "act": rng.choice(["silu", "gelu_tanh"])}
    if op == "quantize":
        return {"op": op, "t": _log(rng, 1, 16384), "h": 32 * _log(rng, 1, 224), "type": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "mx_linear":
        return {"op": op, "t": _log(rng, 1, 8192), "n": _log(rng, 128, 4096), "h": 32 * _log(rng, 4, 224), "type": kind}
    return {"op": op, "t": _log(rng, 1, 4096), "h": 32 * _log(rng, 16, 224), "i": 32 * _log(rng, 16, 64),
            "type": kind, "act": rng.choice(["silu", "gelu_tanh"])}


def work(case):
    op, t, h = case["op"], case["t"], case["h"]
    e = 4 if case["type"] == "fp32" else 2
    if op == "ffn":
        i = case["i"]
        return {"bytes": e * (2 * t * h + 3 * h * i), "flops": 6 * t * h * i}
    if op == "train":
        # in: x, the output's gradient and the weights; out: y, x's gradient and the weights' gradients
        i = case["i"]
        return {"bytes": e * (4 * t * h + 6 * h * i), "flops": 18 * t * h * i}
    if op == "quantize":
        # in: the rows; out: codes and exponents, and the values they stand for
        return {"bytes": t * h * (e + 0.5 + 1 / 32 + 2), "flops": 4 * t * h}
    four = 0.5 + 1 / 32
    if op == "mx_linear":
        n = case["n"]
        return {"bytes": e * t * (h + n) + four * n * h, "flops": 2 * t * h * n}
    i = case["i"]
    return {"bytes": e * 2 * t * h + four * 3 * h * i, "flops": 6 * t * h * i}


# ------------------------------------------------------------------ inputs
def _weights(rows, cols, kind, gen):
    return (torch.randn(rows, cols, generator=gen, device="cuda") * cols ** -0.5).to(kind)


def _activations(t, h, kind, gen):
    """Normal rows of unequal size with a few large channels, as hidden states have them."""
    x = torch.randn(t, h, generator=gen, device="cuda")
    x *= torch.exp2(torch.randn(t, 1, generator=gen, device="cuda") * 0.5)
    loud = torch.rand(h, generator=gen, device="cuda") < 0.01
    return torch.where(loud, x * 8, x).to(kind)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, t, h = _TYPES[case["type"]], case["t"], case["h"]
    s = dict(case, x=_activations(t, h, kind, gen))
    if case["op"] in ("ffn", "train"):
        s["w13"] = _weights(2 * case["i"], h, kind, gen)
        s["w2"] = _weights(h, case["i"], kind, gen)
    if case["op"] == "train":
        s["dy"] = _weights(t, h, kind, gen)
    if case["op"] == "mx_linear":
        s["w"] = _four_bits(_weights(case["n"], h, torch.float32, gen))
    if case["op"] == "mx_ffn":
        s["w13"] = _four_bits(_weights(2 * case["i"], h, torch.float32, gen))
        s["w2"] = _four_bits(_weights(h, case["i"], torch.float32, gen))
    return s


# --------------------------------------------------------------- plain form
def _act(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    return 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))


def _act_slope(g, name):
    if name == "silu":
        s = torch.sigmoid(g)
        return s * (1 + g * (1 - s))
    th = torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))
    return 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * 0.7978845608028654 * (1 + 0.134145 * g * g)


def _plain_quantize(x):
    """Values (fp32, the elements in units of their block's scale) and exponents [R, K / 32] of fp32 rows."""
    b = x.reshape(x.shape[0], -1, 32)
    top = torch.frexp(b.abs().amax(dim=2))
    e = torch.where(top.mantissa == 0, -127, (top.exponent - 3).clamp(-127, 127))
    v = torch.ldexp(b, -e.unsqueeze(2))
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.round(a / step) * step).clamp(max=6.0).copysign(v), e


def _four_bits(x):
    """Codes and tiled exponent bytes of fp32 rows."""
    v, e = _plain_quantize(x)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    c = torch.searchsorted(grid, v.abs()).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
    c = c.reshape(x.shape[0], -1, 2)
    rows, blocks = e.shape
    full = torch.zeros(-(-rows // 128) * 128, -(-blocks // 4) * 4, dtype=torch.uint8, device=x.device)
    full[:rows, :blocks] = (e + 127).to(torch.uint8)
    tiled = full.reshape(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()
    return c[:, :, 0] | c[:, :, 1] << 4, tiled


def _values(codes, tiled, to=torch.float32):
    """The matrix that codes and tiled exponents stand for."""
    rows, half = codes.shape
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device, dtype=to)
    grid = torch.cat([grid, -grid])
    v = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], dim=2).reshape(rows, -1, 32)
    e = tiled.permute(0, 3, 2, 1, 4).reshape(tiled.shape[0] * 128, -1)[:rows, : half // 16]
    return torch.ldexp(v, e.to(torch.int32).unsqueeze(2) - 127).reshape(rows, -1)


def _plain_rounded(x):
    v, e = _plain_quantize(x)
    return torch.ldexp(v, e.unsqueeze(2)).reshape(x.shape)


def _plain(s):
    kind, x = _TYPES[s["type"]], s["x"].float()
    op = s["op"]
    if op == "quantize":
        return _plain_rounded(x).to(torch.bfloat16)
    if op == "mx_linear":
        return (_plain_rounded(x) @ _values(*s["w"]).t()).to(kind)
    if op == "mx_ffn":
        u, g = (_plain_rounded(x) @ _values(*s["w13"]).t()).chunk(2, dim=1)
        return (_plain_rounded(_act(g, s["act"]) * u) @ _values(*s["w2"]).t()).to(kind)
    w13, w2 = s["w13"].float(), s["w2"].float()
    u, g = (x @ w13.t()).chunk(2, dim=1)
    a = _act(g, s["act"])
    hid = a * u
    y = (hid @ w2.t()).to(kind)
    if op == "ffn":
        return y
    dy = s["dy"].float()
    dh = dy @ w2
    du_dg = torch.cat([dh * a, dh * u * _act_slope(g, s["act"])], dim=1)
    return {"y": y, "dx": (du_dg @ w13).to(kind), "dw13": (du_dg.t() @ x).to(kind), "dw2": (dy.t() @ hid).to(kind)}


# --------------------------------------------------------- the package's calls
def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashinfer-bench-avengers_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ffn_host

    return ffn_host


def _own(s):
    f, op = _package(), s["op"]
    if op == "ffn":
        return f.gated_ffn(s["x"], s["w13"], s["w2"], s["act"])
    if op == "train":
        y, saved = f.gated_ffn_forward(s["x"], s["w13"], s["w2"], s["act"])
        dx, dw13, dw2 = f.gated_ffn_backward(s["dy"], s["x"], s["w13"], s["w2"], saved, s["act"])
        return {"y": y, "dx": dx, "dw13": dw13, "dw2": dw2}
    if op == "quantize":
        return f.mxfp4_dequantize(*f.mxfp4_quantize(s["x"]), torch.bfloat16)
    if op == "mx_linear":
        return f.mxfp4_linear(s["x"], *s["w"])
    return f.mxfp4_gated_ffn(s["x"], *s["w13"], *s["w2"], s["act"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------ 64-bit definition
def _nearest_four_bits(x):
    """Each 32-block of fp64 rows on the grid of e2m1 numbers times 2^(floor(log2 max) - 2): the nearest, a tie to
    the neighbour with the even last bit, beyond 6 the 6."""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(dim=2, keepdim=True)
    m, p = torch.frexp(top)
    unit = torch.where(top > 0, torch.exp2((p - 3).clamp(-127, 127).double()), torch.ones_like(top))
    q = b / unit
    a = q.abs()
    out = torch.zeros_like(a)
    # midpoints between neighbours; a tie goes up where the upper neighbour's code is even
    for mid, value, up in ((0.25, 0.5, False), (0.75, 1.0, True), (1.25, 1.5, False), (1.75, 2.0, True), (2.5, 3.0, False),
                           (3.5, 4.0, True), (5.0, 6.0, False)):
        out = torch.where(a >= mid if up else a > mid, value, out)
    return (out * unit * torch.sign(q)).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    x, op = s["x"].double(), case["op"]
    if op == "quantize":
        return _nearest_four_bits(x)
    if op == "mx_linear":
        return torch.mm(_nearest_four_bits(x), _values(*s["w"], torch.float64).T)
    four = op == "mx_ffn"
    w13, w2 = (_values(*s[k], torch.float64) if four else s[k].double() for k in ("w13", "w2"))
    i = case["i"]
    if four:
        x = _nearest_four_bits(x)
    up, gate = torch.mm(x, w13[:i].T), torch.mm(x, w13[i:].T)
    if case["act"] == "silu":
        sig = 1 / (1 + torch.exp(-gate))
        value, slope = gate * sig, sig + gate * sig * (1 - sig)
    else:
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (gate + 0.044715 * gate ** 3))
        value = gate * (1 + th) / 2
        slope = (1 + th) / 2 + gate / 2 * (1 - th ** 2) * c * (1 + 3 * 0.044715 * gate ** 2)
    hid = value * up
    if four:
        hid = _nearest_four_bits(hid)
    y = torch.mm(hid, w2.T)
    if op != "train":
        return y
    dy = s["dy"].double()
    dh = torch.mm(dy, w2)
    dup, dgate = dh * value, dh * up * slope
    return {"y": y, "dx": torch.mm(dup, w13[:i]) + torch.mm(dgate, w13[i:]),
            "dw13": torch.cat([torch.mm(dup.T, x), torch.mm(dgate.T, x)]), "dw2": torch.mm(dy.T, hid)}
