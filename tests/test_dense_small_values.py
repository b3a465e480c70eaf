"""fp16 intermediates of the dense block far below 1: where they are kept in
two parts (up to 64 tokens, for y and the input's gradient), the second holds
what fp16's smallest step leaves of the first."""
from __future__ import annotations

import pytest
import torch

import dense_reference as ref

U = ref.U[torch.float16]
# The rest of a rounding is kept times 2^11: what fp16's smallest step, 2^-24,
# rounds off of it is at most 2^-25 2^-11.
REST = 2.0 ** -36


def _rnd(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device="cuda")


def _forms(x, w13, activation):
    """u, g, act(g), act'(g) in 64 bits with bounds on the kernel's fp32 ones."""
    pre = x @ w13.T
    e = ref.gamma(x.shape[1]) * (x.abs() @ w13.abs().T)
    (up, gate), (e_up, e_gate) = pre.chunk(2, 1), e.chunk(2, 1)
    a, da = ref.act(gate, activation)
    return up, e_up, gate, a, 1.2 * e_gate + ref.ACT * a.abs(), da, 1.2 * e_gate + ref.ACT * (1 + gate.abs())


def _product(left, e_left, right):
    """left @ right of an operand in two parts: value and bound."""
    v = left @ right
    m = e_left @ right.abs()
    e = m + 2 * ref.gamma(left.shape[1]) * (left.abs() @ right.abs() + m)
    return v, e + U * (v.abs() + e) + ref.TINY[torch.float16]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 64])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_small_output_gradients(cuda_device, T, activation):
    """Output gradients of 1e-6, as without a loss scale: du and dg are about
    2^-20, sixteen of fp16's smallest steps; the weights bring dx back up."""
    import ffn_host

    H, inter = 256, 128
    rnd = _rnd(1)
    x = (rnd(T, H) / 16).half()
    w13 = (rnd(2 * inter, H) * (16 * H ** -0.5)).half()
    w2 = (rnd(H, inter) * inter ** -0.5).half()
    dy = (rnd(T, H) * 1e-6).half()
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2, activation)
    dx = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, activation)[0]

    x, w13, w2, dy = (t.double() for t in (x, w13, w2, dy))
    up, e_up, _, a, e_a, da, e_da = _forms(x, w13, activation)
    dh = dy @ w2
    e_dh = ref.gamma(H) * (dy.abs() @ w2.abs())
    d = torch.cat([dh * a, dh * up * da], 1)
    e = torch.cat([e_dh * (a.abs() + e_a) + dh.abs() * e_a,
                   (dh.abs() + e_dh) * (up.abs() + e_up) * (da.abs() + e_da) - (dh * up * da).abs()], 1)
    ref.assert_within(dx, _product(d, e + U * U * (d.abs() + e) + REST, w13), "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 64])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_small_hidden(cuda_device, T, activation):
    """A hidden of about 2^-21 that large weights bring back up."""
    import ffn_host

    H, inter = 256, 128
    rnd = _rnd(2)
    x = (rnd(T, H) * 1e-3).half()
    w13 = (rnd(2 * inter, H) * H ** -0.5).half()
    w2 = (rnd(H, inter) * 16).half()
    y = ffn_host.gated_ffn(x, w13, w2, activation)

    x, w13, w2 = (t.double() for t in (x, w13, w2))
    up, e_up, _, a, e_a, _, _ = _forms(x, w13, activation)
    h = a * up
    e = e_a * up.abs() + a.abs() * e_up + e_a * e_up
    ref.assert_within(y, _product(h, e + U * U * (h.abs() + e) + REST, w2.T), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 64, 130])
@pytest.mark.parametrize("scale", [1e-5, 1e-6])
def test_small_output_gradients_elsewhere(cuda_device, T, scale):
    """Everything else reads du and dg as one fp16 number each: off by half of
    fp16's smallest step, 2^-25, where they are below its normal range."""
    import ffn_host

    rnd = _rnd(3)
    x, w13 = rnd(T, 256).half(), (rnd(256, 256) / 16).half()
    w2, dy = (rnd(256, 128) * 128 ** -0.5).half(), (rnd(T, 256) * scale).half()
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    want = ref.ffn(x, w13, w2, "silu", dy)
    for name, g in zip(("dx", "dw13", "dw2"), ffn_host.gated_ffn_backward(dy, x, w13, w2, saved)):
        ref.assert_within(g, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 64])
def test_large_hidden(cuda_device, T):
    """The other end of the range: a hidden just below fp16's largest number,
    whose rest, times 2^11, still fits."""
    import ffn_host

    x = torch.zeros(T, 64, device="cuda").half()
    x[:, 0] = 1
    w13 = torch.zeros(64, 64, device="cuda").half()
    w13[:32, 0], w13[32:, 0] = 2001, 31.703125       # h = 63437.95: 63424 and a rest of 13.95
    w2 = torch.zeros(64, 32, device="cuda").half()
    w2[:32] = 2.0 ** -6 * torch.eye(32, device="cuda").half()
    gate = w13[32, 0].double()
    want = (2001 * gate / (1 + torch.exp(-gate)) * 2.0 ** -6).half()
    y = ffn_host.gated_ffn(x, w13, w2)
    assert torch.equal(y[:, :32], want.expand(T, 32)) and not y[:, 32:].any()
