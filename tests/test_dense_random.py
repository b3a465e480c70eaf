"""The dense operators at random sizes, types and row distances, against 64
bits within the derived bounds."""
from __future__ import annotations

import math
import random

import pytest
import torch

import dense_reference as ref


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _rows(rng, T, cols, dtype, g):
    """[T, cols] cut from wider rows of NaN, or whole."""
    step = 16 // torch.empty(0, dtype=dtype).element_size()
    left, right = rng.choice([(0, 0), (step, 0), (2 * step, 3 * step)])
    wide = torch.full((T, left + cols + right), float("nan"), device="cuda", dtype=dtype)
    x = wide[:, left:left + cols]
    x.copy_(torch.randn(T, cols, generator=g, device="cuda"))
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_training_step(cuda_device, seed):
    import ffn_host

    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, H, inter = _log(rng, 1, 900), 8 * _log(rng, 1, 160), 8 * _log(rng, 1, 160)
    dtype, activation = rng.choice([torch.bfloat16, torch.float16]), rng.choice(["silu", "gelu_tanh"])
    x, dy = _rows(rng, T, H, dtype, g), _rows(rng, T, H, dtype, g)
    w13 = (torch.randn(2 * inter, H, generator=g, device="cuda") * H ** -0.5).to(dtype)
    w2 = (torch.randn(H, inter, generator=g, device="cuda") * inter ** -0.5).to(dtype)
    needs = [rng.random() < 0.8 for _ in range(3)]
    y, saved = ffn_host.gated_ffn_forward(x, w13, w2, activation)
    want = ref.ffn(x, w13, w2, activation, dy)
    what = f"{T} x {H} x {inter} {dtype} {activation} {needs}"
    ref.assert_within(y, want["y"], what)
    assert torch.equal(y, ffn_host.gated_ffn(x, w13, w2, activation))
    grads = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, activation, needs)
    for name, need, grad in zip(("dx", "dw13", "dw2"), needs, grads):
        assert (grad is not None) == need
        if need:
            ref.assert_within(grad, want[name], f"{name} {what}")
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_4_bit_linear(cuda_device, seed):
    import ffn_host

    rng = random.Random(1000 + seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, K, N = _log(rng, 1, 900), 32 * _log(rng, 1, 60), _log(rng, 1, 1500)
    dtype = rng.choice([torch.bfloat16, torch.float16, torch.float32])
    x = _rows(rng, T, K, dtype, g)
    w = ffn_host.mxfp4_quantize(torch.randn(N, K, generator=g, device="cuda"))
    y = ffn_host.mxfp4_linear(x, *w)
    xq = ffn_host.mxfp4_quantize(x)
    assert torch.equal(y, ffn_host.mxfp4_matmul(*xq, *w, dtype))
    a, b = ref.mx_values(*xq).cuda(), ref.mx_values(*w).cuda()
    ref.assert_within(y, ref.mx_product(a, b, dtype), f"{T} x {K} x {N} {dtype}")
    assert ffn_host.read_status() == 0
