"""Device memory of the dense operators' calls."""
from __future__ import annotations

import pytest
import torch

import dense_reference as ref


@pytest.mark.gpu
@pytest.mark.parametrize("T", [64, 4096])
def test_second_weight_alone_needs_no_scratch(cuda_device, T):
    """The gradient of w2 reads the output's gradient and the saved hidden: no
    [du | dg] is made for it."""
    import ffn_host

    H, inter = 64, 2048
    x, dy = (torch.randn(T, H, device="cuda").bfloat16() for _ in range(2))
    w13, w2 = torch.randn(2 * inter, H, device="cuda").bfloat16(), torch.randn(H, inter, device="cuda").bfloat16()
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)

    def peak(needs):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, needs=needs)
        torch.cuda.synchronize()
        del grads
        return torch.cuda.max_memory_allocated() - before

    # the allocator hands out multiples of 512 bytes
    assert peak((False, False, True)) <= H * inter * 2 + 512
    assert peak((True, False, False)) >= 4 * T * inter


@pytest.mark.gpu
def test_saved_sums_beyond_32_bits(cuda_device):
    """u, g and [du | dg] of more than 2^31 elements: rows at both ends as in a
    call on them alone (over CTA pairs both)."""
    import ffn_host

    T, H, inter, n = ffn_host.MAX_TOKENS, 64, 4128, 300
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    w13, w2, ends = rnd(2 * inter, H), rnd(H, inter) * inter ** -0.5, rnd(2 * n, H)
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    x[:n], x[T - n:] = ends[:n], ends[n:]
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    few, few_saved = ffn_host.gated_ffn_forward(ends, w13, w2)
    for a, b in zip(saved, few_saved):
        # (K of these products is one step: no sums to order differently)
        assert torch.equal(a[:n], b[:n]) and torch.equal(a[T - n:], b[n:]) and not a[n:T - n].any()
    dx = ffn_host.gated_ffn_backward(x, x, w13, w2, saved, needs=(True, False, False))[0]
    want = ref.ffn(ends, w13, w2, "silu", ends)["dx"]
    ref.assert_within(torch.cat([dx[:n], dx[T - n:]]), want, "dx")
    assert not dx[n:T - n].any()
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [4128, 8320])
def test_4_bit_block_beyond_32_bits(cuda_device, inter):
    """The 4-bit block on the most tokens: its fp32 sums (an I that is no
    multiple of 128) or its codes pass 2^31 elements."""
    import ffn_host

    T, H, n = ffn_host.MAX_TOKENS, 96, 300
    g = torch.Generator(device="cuda").manual_seed(2)
    w13 = ffn_host.mxfp4_quantize(torch.randn(2 * inter, H, generator=g, device="cuda"))
    w2 = ffn_host.mxfp4_quantize(torch.randn(H, inter, generator=g, device="cuda"))
    ends = torch.randn(2 * n, H, generator=g, device="cuda").bfloat16()
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    x[:n], x[T - n:] = ends[:n], ends[n:]
    y = ffn_host.mxfp4_gated_ffn(x, *w13, *w2)
    few = ffn_host.mxfp4_gated_ffn(ends, *w13, *w2)
    assert torch.equal(y[:n], few[:n]) and torch.equal(y[T - n:], few[n:]) and not y[n:T - n].any()
    assert ffn_host.read_status() == 0
