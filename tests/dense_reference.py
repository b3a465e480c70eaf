"""Plain 64-bit forms of the dense operators, with element-wise bounds on how
far a kernel may be from them.

Bounds count, for every element:
  * the last rounding, u = 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32) times the
    value, and half the smallest step of fp16's subnormals, 2^-25;
  * the rounding of the 16-bit intermediates (h, du, dg), carried through the
    product that reads them by the absolute values of its other operand; for up
    to 64 tokens y and dx read them as two 16-bit numbers, so the rounding
    there is u squared of the value;
  * the fp32 sums: a sum of k products is k / 16 additions of 16-term blocks,
    each addition off by at most 2^-23 of the sum of magnitudes (a tensor core
    may truncate), so GAMMA(k) = (k / 16 + 16) 2^-23 times that sum;
  * the activation: 4e-6 relative (fast exponential and division).
Splitting K over a cluster adds at most 8 additions, within the 16.
"""
from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
ACT = 4e-6
TWO_PART = 64


def gamma(k: int) -> float:
    return (k / 16 + 16) * 2.0 ** -23


def act(g: torch.Tensor, name: str):
    """act(g), act'(g) in 64 bits."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def ffn(x, w13, w2, name, dy=None):
    """Values and bounds of the block (and, given dy, of its gradients) on the
    inputs' own values: dict name -> (value, bound)."""
    dt = x.dtype
    u_, tiny = U[dt], TINY[dt]
    x, w13, w2 = x.double(), w13.double(), w2.double()
    inter = w2.shape[1]
    H, T = x.shape[1], x.shape[0]
    pre = x @ w13.T
    e_pre = gamma(H) * (x.abs() @ w13.abs().T)
    up, gate = pre[:, :inter], pre[:, inter:]
    e_up, e_gate = e_pre[:, :inter], e_pre[:, inter:]
    a, da = act(gate, name)
    # |act'| and |act''| of both activations stay below 1.2
    e_a = 1.2 * e_gate + ACT * a.abs()
    h = a * up
    e_h = e_a * up.abs() + a.abs() * e_up + e_a * e_up
    r_h = e_h + u_ * (h.abs() + e_h) + tiny            # after the rounding to 16 bits
    y_h = e_h + u_ * u_ * (h.abs() + e_h) + tiny if T <= TWO_PART else r_h
    y = h @ w2.T
    # two parts: twice the terms in the sum
    e_y = y_h @ w2.abs().T + (2 if T <= TWO_PART else 1) * gamma(inter) * ((h.abs() + r_h) @ w2.abs().T)
    out = {"y": (y, e_y + u_ * (y.abs() + e_y) + tiny)}
    if dy is None:
        return out
    dy = dy.double()
    dh = dy @ w2
    e_dh = gamma(H) * (dy.abs() @ w2.abs())
    e_da = 1.2 * e_gate + ACT * (1 + gate.abs())
    du, dg = dh * a, dh * up * da
    e_du = e_dh * (a.abs() + e_a) + dh.abs() * e_a
    e_dg = (dh.abs() + e_dh) * (up.abs() + e_up) * (da.abs() + e_da) - dg.abs()
    d = torch.cat([du, dg], 1)
    e_d = torch.cat([e_du, e_dg], 1)
    r_d = e_d + u_ * (d.abs() + e_d) + tiny

    # dx of few tokens reads [du | dg] in two parts, like y
    d_x = e_d + u_ * u_ * (d.abs() + e_d) + tiny if T <= TWO_PART else r_d

    def product(left, e_left, right, k, parts=1):
        v = left @ right
        m = e_left @ right.abs()
        e = m + parts * gamma(k) * (left.abs() @ right.abs() + m)
        return v, e + u_ * (v.abs() + e) + tiny

    out["dx"] = product(d, d_x, w13, 2 * inter, 2 if T <= TWO_PART else 1)
    out["dw13"] = product(d.T, r_d.T, x, T)
    v, e = product(h.T, r_h.T, dy, T)
    out["dw2"] = (v.T, e.T)
    return out


def assert_within(got: torch.Tensor, want, what: str = "") -> None:
    value, bound = want
    assert got.shape == value.shape
    off = (got.double() - value).abs() - bound.to(got.device)
    worst = off.max().item() if off.numel() else 0.0
    assert not torch.isnan(off).any(), f"{what}: NaN"
    assert worst <= 0.0, f"{what}: {int((off > 0).sum())} of {off.numel()} elements beyond the bound, by {worst:g}"


# ------------------------------------------------------------------ 4 bits
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def mx_quantize(x: torch.Tensor):
    """Codes [R, K / 2] and exponent bytes in mxfp4_scale_shape, element by
    element from the definition (64 bits, CPU)."""
    x = x.detach().cpu().double()
    R, K = x.shape
    b = x.reshape(R, K // 32, 32)
    amax = b.abs().amax(2)
    bad = ~torch.isfinite(b).all(2)
    safe = torch.where(bad | (amax == 0), torch.ones_like(amax), amax)
    m, e = torch.frexp(safe)                       # safe = m 2^e, m in [0.5, 1)
    e = (e - 1 - 2).clamp(min=-127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    v = b / torch.exp2(e.double())[:, :, None]
    v = torch.where(bad[:, :, None], torch.zeros_like(v), v)
    a = v.abs()
    grid = torch.tensor(E2M1, dtype=torch.float64)
    dist = (a[..., None] - grid).abs()
    best = dist.min(-1).values
    near = dist == best[..., None]                 # one grid point, or the two sides of a tie
    codes = torch.arange(8)
    even = torch.where(near & (codes % 2 == 0), codes, -1).amax(-1)
    code = torch.where(near.sum(-1) == 2, even, near.int().argmax(-1))
    code = torch.where(a > 6, torch.full_like(code, 7), code)
    code = code + 8 * torch.where(bad[:, :, None], torch.zeros_like(code), torch.signbit(v).long())
    code = code.reshape(R, K).to(torch.uint8)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127)
    scale = torch.zeros(-(-R // 128), -(-K // 128), 32, 4, 4, dtype=torch.uint8)
    r = torch.arange(R)[:, None].expand(R, K // 32)
    k = torch.arange(K // 32)[None, :].expand(R, K // 32)
    scale[r // 128, k // 4, r % 32, r % 128 // 32, k % 4] = byte.to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale


def mx_values(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The values (64 bits) of a 4-bit matrix."""
    q, scale = q.cpu(), scale.cpu()
    R, K = q.shape[0], 2 * q.shape[1]
    grid = torch.tensor(E2M1 + tuple(-g for g in E2M1), dtype=torch.float64)
    v = torch.empty(R, K, dtype=torch.float64)
    v[:, 0::2] = grid[(q & 15).long()]
    v[:, 1::2] = grid[(q >> 4).long()]
    r = torch.arange(R)[:, None].expand(R, K // 32)
    k = torch.arange(K // 32)[None, :].expand(R, K // 32)
    byte = scale[r // 128, k // 4, r % 32, r % 128 // 32, k % 4].double()
    f = torch.where(byte == 255, torch.full_like(byte, float("nan")), torch.exp2(byte - 127))
    return v * f.repeat_interleave(32, 1)


def mx_product(a: torch.Tensor, b: torch.Tensor, dtype: torch.dtype):
    """A B^T of two matrices of 4-bit values: (value, bound)."""
    y = a @ b.T
    e = gamma(a.shape[1]) * (a.abs() @ b.abs().T)
    return y, e + U[dtype] * (y.abs() + e) + TINY[dtype]
