"""Device memory of the dense operators' calls."""
from __future__ import annotations

import pytest
import torch


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
