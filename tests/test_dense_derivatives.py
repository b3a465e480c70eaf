"""Derivatives of the dense operators are recorded, or the call is refused:
none is dropped without a word."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwad


def _block(T=8, H=64, inter=32, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (rnd(T, H).to(dtype), (rnd(2 * inter, H) * H ** -0.5).to(dtype), (rnd(H, inter) * inter ** -0.5).to(dtype),
            rnd(T, H).to(dtype))


def _dual(args, n):
    return [fwad.make_dual(t, torch.ones_like(t)) if i == n else t for i, t in enumerate(args)]


@pytest.mark.gpu
@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(cuda_device, grad_mode):
    """Forward-mode tangents, with gradient mode on and off: torch.no_grad()
    stops reverse mode alone."""
    import ffn_host

    x, w13, w2, dy = _block()
    want = ffn_host.gated_ffn(x, w13, w2)
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    q13, q2 = ffn_host.mxfp4_quantize(w13), ffn_host.mxfp4_quantize(w2)
    with fwad.dual_level(), torch.set_grad_enabled(grad_mode):
        for n in range(3):
            with pytest.raises(RuntimeError):
                ffn_host.gated_ffn(*_dual((x, w13, w2), n))
            with pytest.raises(RuntimeError, match="forward-mode"):
                ffn_host.gated_ffn_forward(*_dual((x, w13, w2), n))
        for n in range(6):
            a = _dual((dy, x, w13, w2, *saved), n)
            with pytest.raises(RuntimeError, match="forward-mode"):
                ffn_host.gated_ffn_backward(*a[:4], a[4:])
        dual = _dual((x,), 0)[0]
        with pytest.raises(RuntimeError, match="forward-mode"):
            ffn_host.mxfp4_linear(dual, *q13)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ffn_host.mxfp4_gated_ffn(dual, *q13, *q2)
        # an output with a tangent would keep the tangent of its old values
        with pytest.raises(RuntimeError, match="forward-mode"):
            ffn_host.gated_ffn(x, w13, w2, output=_dual((torch.empty_like(x),), 0)[0])
        with torch.inference_mode():       # stops forward mode too
            assert torch.equal(ffn_host.gated_ffn(dual, w13, w2), want)


@pytest.mark.gpu
def test_4_bit_functions_refuse_gradients(cuda_device):
    """The 4-bit functions record no gradients, so that an input which asks for
    them is refused while gradients are recorded; detached, or where they are
    not recorded, it is taken. Codes are integers and never ask."""
    import ffn_host

    x, w13, w2, _ = _block()
    with torch.no_grad():
        q13, q2 = ffn_host.mxfp4_quantize(w13), ffn_host.mxfp4_quantize(w2)
    leaf = x.clone().requires_grad_()
    calls = (lambda t: ffn_host.mxfp4_linear(t, *q13), lambda t: ffn_host.mxfp4_gated_ffn(t, *q13, *q2))
    for call in calls:
        want = call(x)
        for t in (leaf, leaf * 1):
            with pytest.raises(RuntimeError, match="gradients"):
                call(t)
        with torch.no_grad():
            assert torch.equal(call(leaf), want)
        with torch.inference_mode():
            assert torch.equal(call(leaf), want)
        assert torch.equal(call(leaf.detach()), want)
    for a, b in zip(ffn_host.mxfp4_quantize(torch.nn.Parameter(w13)), q13):
        assert a.dtype == torch.uint8 and not a.requires_grad and torch.equal(a, b)
