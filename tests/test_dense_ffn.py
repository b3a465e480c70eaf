"""The gated feed-forward block and its gradients against the 64-bit form,
element by element within derived bounds; refusals on the CPU."""
from __future__ import annotations

import pytest
import torch

import dense_reference as ref


def _inputs(T, H, inter, dtype, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    x = (rnd(T, H) * torch.exp2(rnd(T, 1))).to(dtype)
    w13 = (rnd(2 * inter, H) * H ** -0.5).to(dtype)
    w2 = (rnd(H, inter) * inter ** -0.5).to(dtype)
    dy = (rnd(T, H) * 0.1).to(dtype)
    return x, w13, w2, dy


# one token to several tiles; sizes that end inside a tile in every direction
# (token tiles of 16, 64 and 256, feature tiles of 64 and 128, 64-wide K
# steps), the smallest sizes, and the split of K over 1 to 8 CTAs and over 1,
# 2 and 4 pairs
SHAPES = [(1, 8, 8), (1, 7168, 2048), (3, 64, 64), (16, 520, 264), (17, 1032, 520), (64, 2048, 136), (65, 4096, 64),
          (127, 72, 1000), (128, 256, 128), (129, 256, 128), (255, 136, 72), (257, 1032, 520), (600, 512, 1048),
          (130, 3200, 264), (256, 7168, 2048), (301, 2056, 1032), (513, 4104, 200)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,inter", SHAPES)
@pytest.mark.parametrize("dtype,activation", [(torch.bfloat16, "silu"), (torch.float16, "gelu_tanh")])
def test_forward(cuda_device, T, H, inter, dtype, activation):
    import ffn_host

    x, w13, w2, _ = _inputs(T, H, inter, dtype)
    y = ffn_host.gated_ffn(x, w13, w2, activation)
    assert y.dtype == dtype
    ref.assert_within(y, ref.ffn(x, w13, w2, activation)["y"], "y")
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,inter", SHAPES)
@pytest.mark.parametrize("dtype,activation", [(torch.bfloat16, "gelu_tanh"), (torch.float16, "silu")])
def test_gradients(cuda_device, T, H, inter, dtype, activation):
    import ffn_host

    x, w13, w2, dy = _inputs(T, H, inter, dtype, seed=1)
    y, saved = ffn_host.gated_ffn_forward(x, w13, w2, activation)
    got = dict(zip(("dx", "dw13", "dw2"), ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, activation)))
    want = ref.ffn(x, w13, w2, activation, dy)
    ref.assert_within(y, want["y"], "y")
    for k, v in got.items():
        ref.assert_within(v, want[k], k)
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_gradients_against_differences(cuda_device, activation):
    """Central differences of the 64-bit block along random directions: each
    gradient's inner product with the direction, within the gradient's own
    bounds summed over the direction (the differences' own error, about
    step^2, is below 1e-6 of the largest terms and added)."""
    import ffn_host

    x, w13, w2, dy = _inputs(9, 136, 72, torch.bfloat16, seed=2)
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2, activation)
    grads = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, activation)
    want = ref.ffn(x, w13, w2, activation, dy)
    args = [t.double() for t in (x, w13, w2)]

    def loss(*a):
        pre = a[0] @ a[1].T
        up, gate = pre.chunk(2, 1)
        return (((ref.act(gate, activation)[0] * up) @ a[2].T) * dy.double()).sum().item()

    gen = torch.Generator(device="cuda").manual_seed(3)
    for n, (name, g) in enumerate(zip(("dx", "dw13", "dw2"), grads)):
        v = torch.randn(args[n].shape, generator=gen, device="cuda", dtype=torch.float64)
        step = 1e-4
        plus = [a + step * v if j == n else a for j, a in enumerate(args)]
        minus = [a - step * v if j == n else a for j, a in enumerate(args)]
        diff = (loss(*plus) - loss(*minus)) / (2 * step)
        bound = (want[name][1] * v.abs()).sum().item() + 1e-6 * (want[name][0].abs() * v.abs()).sum().item()
        assert abs((g.double() * v).sum().item() - diff) <= bound, name


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 300])
def test_rows_apart_and_untouched_neighbours(cuda_device, T):
    """Rows of x and of the output's gradient cut from wider buffers; an
    output inside a larger buffer leaves what is around it alone."""
    import ffn_host

    H, inter = 264, 136
    x, w13, w2, dy = _inputs(T, H, inter, torch.bfloat16, seed=4)
    wide = torch.full((T, H + 40), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 8:8 + H] = x
    xs = wide[:, 8:8 + H]
    wide_dy = torch.full((T, 3 * H), float("nan"), dtype=x.dtype, device="cuda")
    wide_dy[:, H:2 * H] = dy
    buf = torch.full((T + 6, H), 7.0, dtype=x.dtype, device="cuda")
    y = ffn_host.gated_ffn(xs, w13, w2, "silu", output=buf[2:2 + T])
    assert torch.equal(y, ffn_host.gated_ffn(x, w13, w2, "silu"))
    assert (buf[:2] == 7).all() and (buf[2 + T:] == 7).all()
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    plain = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved)
    apart = ffn_host.gated_ffn_backward(wide_dy[:, H:2 * H], xs, w13, w2, saved)
    for a, b in zip(plain, apart):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 200])
def test_rows_do_not_mix(cuda_device, T):
    """A NaN or infinite row spoils its own output row only, and its own row
    of the input's gradient."""
    import ffn_host

    x, w13, w2, dy = _inputs(T, 256, 128, torch.bfloat16, seed=5)
    clean = ffn_host.gated_ffn(x, w13, w2)
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    clean_dx = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved)[0]
    bad = x.clone()
    bad[1, 3] = float("nan")
    bad[T - 1] = float("inf")
    keep = [r for r in range(T) if r not in (1, T - 1)]
    y, saved = ffn_host.gated_ffn_forward(bad, w13, w2)
    dx = ffn_host.gated_ffn_backward(dy, bad, w13, w2, saved)[0]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], clean_dx[keep])
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[T - 1]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 64, 65, 129])
def test_hidden_beyond_half_precision(cuda_device, T):
    """A hidden value beyond fp16 is infinite, with its sign, and so are the
    outputs it enters; nothing turns into NaN."""
    import ffn_host

    x, w13, w2, _ = _inputs(T, 256, 128, torch.float16, seed=6)
    w13[0], w13[128] = 0, 0
    w13[0, 0], w13[128, 0] = -300, 300     # u and g of feature 0
    x[:, 0] = 0
    x[T - 1, 0] = 1                        # h = -300 silu(300) = -90000
    w2[:, 0] = torch.where(w2[:, 0] < 0, -1.0, 1.0)
    y = ffn_host.gated_ffn(x, w13, w2)
    assert torch.equal(y[T - 1], -w2[:, 0] * float("inf"))
    assert torch.isfinite(y[: T - 1]).all()


@pytest.mark.gpu
def test_large_gates(cuda_device):
    """Gates far beyond the exponential's range: act(g) is g or 0, its slope 1
    or 0, and nothing turns into NaN."""
    import ffn_host

    H = inter = 64
    x = torch.eye(H, dtype=torch.bfloat16, device="cuda")
    gates = torch.tensor([3e4, -3e4, 200.0, -200.0, 90.0, -90.0, 1e10, -1e10], device="cuda").repeat(8)
    w13 = torch.cat([torch.ones(inter, H, device="cuda"), gates[:, None].expand(inter, H)]).to(torch.bfloat16)
    w2 = torch.eye(H, dtype=torch.bfloat16, device="cuda")
    dy = torch.ones(H, H, dtype=torch.bfloat16, device="cuda")
    for activation in ("silu", "gelu_tanh"):
        y, saved = ffn_host.gated_ffn_forward(x, w13, w2, activation)
        dx, dw13, dw2 = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, activation)
        want = gates.to(torch.bfloat16).clamp(min=0)
        assert torch.equal(y, want.expand(H, inter))
        assert all(torch.isfinite(t).all() for t in (dx, dw13, dw2))
        assert torch.equal(dw13[inter:], (want > 0).to(torch.bfloat16)[:, None].expand(inter, H))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 64, 300])
def test_repeats_agree_bit_for_bit(cuda_device, T):
    import ffn_host

    x, w13, w2, dy = _inputs(T, 1032, 520, torch.bfloat16, seed=6)
    first = None
    for _ in range(3):
        y, saved = ffn_host.gated_ffn_forward(x, w13, w2)
        now = (y, *saved, *ffn_host.gated_ffn_backward(dy, x, w13, w2, saved))
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


@pytest.mark.gpu
def test_needs(cuda_device):
    import ffn_host

    x, w13, w2, dy = _inputs(70, 256, 128, torch.bfloat16, seed=7)
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    every = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        some = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, needs=needs)
        for n, a, b in zip(needs, some, every):
            assert (a is None) if not n else torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,inter", [(16, 520, 264), (129, 4104, 264), (600, 2056, 1032)])
def test_every_subset_of_gradients(cuda_device, T, H, inter):
    """Which gradients are asked for decides how the products share launches
    and whether K is split: each subset holds the bounds."""
    import ffn_host

    x, w13, w2, dy = _inputs(T, H, inter, torch.bfloat16, seed=9)
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    want = ref.ffn(x, w13, w2, "silu", dy)
    for mask in range(1, 8):
        needs = [bool(mask >> i & 1) for i in range(3)]
        got = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, needs=needs)
        again = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved, needs=needs)
        for name, need, g, h in zip(("dx", "dw13", "dw2"), needs, got, again):
            assert (g is not None) == need
            if need:
                ref.assert_within(g, want[name], name)
                assert torch.equal(g, h)
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
def test_no_tokens(cuda_device):
    import ffn_host

    x, w13, w2, dy = _inputs(0, 64, 32, torch.bfloat16)
    y, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    dx, dw13, dw2 = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved)
    assert y.shape == (0, 64) and dx.shape == (0, 64)
    assert not dw13.any() and not dw2.any() and dw13.shape == w13.shape and dw2.shape == w2.shape


@pytest.mark.gpu
def test_autograd(cuda_device):
    """Through torch's autograd: the gradients of gated_ffn_backward, also for
    an expanded output gradient, accumulated over two uses of the weights."""
    import ffn_host

    x, w13, w2, dy = _inputs(33, 256, 128, torch.bfloat16, seed=8)
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    ffn_host.gated_ffn(*leaves).backward(dy)
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    want = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved)
    for leaf, g in zip(leaves, want):
        assert torch.equal(leaf.grad, g)
    ffn_host.gated_ffn(*leaves).sum().backward()
    ones = ffn_host.gated_ffn_backward(torch.ones_like(dy), x, w13, w2, saved)
    for leaf, g, o in zip(leaves, want, ones):
        assert torch.equal(leaf.grad, g + o)
    frozen = ffn_host.gated_ffn(leaves[0], w13, w2)
    frozen.backward(dy)
    with torch.no_grad():
        assert not ffn_host.gated_ffn(*leaves).requires_grad
    with pytest.raises(RuntimeError, match="output cannot be given"):
        ffn_host.gated_ffn(*leaves, output=torch.empty_like(x))


@pytest.mark.gpu
def test_no_tokens_through_autograd(cuda_device):
    import ffn_host

    leaves = [t.requires_grad_() for t in _inputs(0, 64, 32, torch.bfloat16)[:3]]
    ffn_host.gated_ffn(*leaves).sum().backward()
    assert all(leaf.grad is not None and leaf.grad.shape == leaf.shape and not leaf.grad.any() for leaf in leaves)


@pytest.mark.gpu
def test_lone_row_of_a_wider_matrix(cuda_device):
    """One row has no pitch: any stride of the first dimension will do."""
    import ffn_host

    x, w13, w2, dy = _inputs(9, 72, 40, torch.bfloat16, seed=12)
    wide = torch.zeros(9, 100, dtype=x.dtype, device="cuda")
    wide[:, :72] = x
    row = wide[2:3, :72]                      # 200 bytes between rows
    y, saved = ffn_host.gated_ffn_forward(row, w13, w2)
    want, want_saved = ffn_host.gated_ffn_forward(x[2:3].clone(), w13, w2)
    assert torch.equal(y, want) and y.is_contiguous()
    for a, b in zip(ffn_host.gated_ffn_backward(dy[2:3], row, w13, w2, saved),
                    ffn_host.gated_ffn_backward(dy[2:3], x[2:3].clone(), w13, w2, want_saved)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_device):
    """The most tokens, rows of more than 2^31 elements in all: rows at both
    ends equal those of a call on them alone (the same kernel: over 128 rows),
    and the weights' gradients of a matrix whose other rows are zero equal
    those of its nonzero rows."""
    import ffn_host

    T, H, inter = ffn_host.MAX_TOKENS, 8208, 64
    _, w13, w2, _ = _inputs(1, H, inter, torch.bfloat16, seed=13)
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(14)
    ends = torch.randn(600, H, generator=g, device="cuda").to(torch.bfloat16)
    x[:300] = ends[:300]
    x[T - 300:] = ends[300:]
    y, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    few, few_saved = ffn_host.gated_ffn_forward(ends, w13, w2)
    want = ref.ffn(ends, w13, w2, "silu", ends)
    got = torch.cat([y[:300], y[T - 300:]])
    ref.assert_within(got, want["y"], "y")
    assert not y[300:T - 300].any()
    dx, dw13, dw2 = ffn_host.gated_ffn_backward(x, x, w13, w2, saved)     # dy = x
    ref.assert_within(torch.cat([dx[:300], dx[T - 300:]]), want["dx"], "dx")
    # zero terms add nothing, but the sums' order is another: the bound's
    # gamma(T) covers T / 16 additions, only those of nonzero blocks can round
    ref.assert_within(dw13, want["dw13"], "dw13")
    ref.assert_within(dw2, want["dw2"], "dw2")
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [16, 64])
def test_beside_the_routed_layer(cuda_device, T):
    """A layer's routed experts and its shared expert on the same tokens, the
    shared expert on a side stream, many times over: each as it is alone
    (the routed sums are fp32 atomics, so within the operator's tolerance)."""
    import ffn_host
    import moe_host
    import moe_oracle
    import workloads

    inp = workloads.make_inputs(T, 3, "cuda")
    args = workloads.as_args(inp)
    scale = inp["hidden_states_scale"].t().repeat_interleave(128, 1)
    x = (inp["hidden_states"].float() * scale).to(torch.bfloat16)
    _, w13, w2, _ = _inputs(1, 7168, 2048, torch.bfloat16, seed=15)
    routed, shared = moe_host.run(*args), ffn_host.gated_ffn(x, w13, w2)
    q13, q2 = ffn_host.mxfp4_quantize(w13), ffn_host.mxfp4_quantize(w2)
    four = ffn_host.mxfp4_gated_ffn(x, *q13, *q2)
    ref.assert_within(shared, ref.ffn(x, w13, w2, "silu")["y"], "shared")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        with torch.cuda.stream(side):
            s = ffn_host.gated_ffn(x, w13, w2), ffn_host.mxfp4_gated_ffn(x, *q13, *q2)
        got.append((moe_host.run(*args), *s))
    torch.cuda.synchronize()
    for r, s, f in got:
        assert torch.equal(s, shared) and torch.equal(f, four)
        ok, matched, err, top = moe_oracle.output_close(r, routed, 1e-2, 0.999)
        assert ok, (matched, err, top)
    assert moe_host.read_status(moe_host.get_workspace(T, x.device)) == 0 and ffn_host.read_status() == 0


@pytest.mark.gpu
def test_calls_from_new_threads(cuda_device):
    """Threads that have not used CUDA before, two at once."""
    import threading

    import ffn_host

    x, w13, w2, dy = _inputs(40, 256, 128, torch.bfloat16, seed=9)
    want, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    grads = ffn_host.gated_ffn_backward(dy, x, w13, w2, saved)
    torch.cuda.synchronize()
    got, errors = [], []

    def call():
        try:
            y, s = ffn_host.gated_ffn_forward(x, w13, w2)
            got.append((y, *ffn_host.gated_ffn_backward(dy, x, w13, w2, s)))
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=call) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, (want, *grads)))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [7, 260])
def test_captured_training_step(cuda_device, T):
    """Forward and backward captured into a graph and replayed on new inputs,
    twice captured, the replays interleaved; and the calls on another stream."""
    import ffn_host

    H, inter = 520, 264
    sets = [_inputs(T, H, inter, torch.bfloat16, seed=s) for s in (10, 11)]

    def step(x, w13, w2, dy):
        y, saved = ffn_host.gated_ffn_forward(x, w13, w2)
        return (y, *ffn_host.gated_ffn_backward(dy, x, w13, w2, saved))

    want = [[t.clone() for t in step(*s)] for s in sets]
    graphs = []
    for _ in range(2):
        static = [t.clone() for t in sets[0]]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*static)
        graphs.append((g, static, out))
    for k in (1, 0):
        for n, (g, static, out) in enumerate(graphs):
            for dst, src in zip(static, sets[(k + n) % 2]):
                dst.copy_(src)
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for n, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(k + n) % 2]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s, inp in zip(streams, sets):
            with torch.cuda.stream(s):
                outs.append(step(*inp))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert all(torch.equal(a, b) for a, b in zip(o, want[i % 2]))
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
def test_refusals_on_the_gpu(cuda_device):
    import ffn_host

    x, w13, w2, dy = _inputs(4, 64, 32, torch.bfloat16)
    _, saved = ffn_host.gated_ffn_forward(x, w13, w2)
    bad = [
        ((x.float(), w13, w2), "bfloat16 or float16"),
        ((x.half(), w13, w2), "w13 must be a contiguous"),
        ((x[0], w13, w2), r"\[T"),
        ((x[:, :60], w13[:, :60].contiguous(), w2[:60]), "rows must start on 16 bytes|multiple of 8"),
        ((x.t().contiguous().t(), w13, w2), "contiguous rows"),
        ((x, w13[:63], w2), "2 I"),
        ((x, w13, w2.t()), "w2 must be a contiguous"),
        ((x, w13, w2[:, :24]), "w2 must be a contiguous"),
        ((x.cpu(), w13, w2), "must be CUDA"),
        ((x, w13.cpu(), w2), "must be CUDA"),
        ((x[:1].expand(4, 64), w13, w2), "do not overlap"),
    ]
    for args, message in bad:
        with pytest.raises(RuntimeError, match=message):
            ffn_host.gated_ffn(*args)
    with pytest.raises(RuntimeError, match="activation"):
        ffn_host.gated_ffn(x, w13, w2, "relu")
    with pytest.raises(RuntimeError, match="output must be"):
        ffn_host.gated_ffn(x, w13, w2, output=torch.empty(4, 128, dtype=x.dtype, device="cuda")[:, :64])
    shifted = torch.empty(4 * 64 + 4, dtype=x.dtype, device="cuda")[4:].view(4, 64)
    with pytest.raises(RuntimeError, match="aligned"):
        ffn_host.gated_ffn(x, w13, w2, output=shifted)
    with pytest.raises(RuntimeError, match="rows must start on 16 bytes"):
        ffn_host.gated_ffn(shifted, w13, w2)
    with pytest.raises(RuntimeError, match="grad_output"):
        ffn_host.gated_ffn_backward(dy.float(), x, w13, w2, saved)
    with pytest.raises(RuntimeError, match="saved u and g"):
        ffn_host.gated_ffn_backward(dy, x, w13, w2, (saved[0].bfloat16(), saved[1]))
    with pytest.raises(RuntimeError, match="saved hidden"):
        ffn_host.gated_ffn_backward(dy, x, w13, w2, (saved[0], saved[1][:2]))


@pytest.mark.gpu
def test_output_argument(cuda_device):
    """A given output is returned, its version goes up like that of any tensor
    written in place, and one that overlaps an input or that autograd follows
    is refused; so is forward-mode differentiation."""
    import ffn_host
    import torch.autograd.forward_ad as fwad

    x, w13, w2, _ = _inputs(8, 64, 32, torch.bfloat16, seed=8)
    want = ffn_host.gated_ffn(x, w13, w2)
    out = torch.empty_like(x)
    version = out._version
    assert ffn_host.gated_ffn(x, w13, w2, output=out) is out
    assert torch.equal(out, want) and out._version > version
    with torch.inference_mode():
        inner = torch.empty_like(x)
    assert torch.equal(ffn_host.gated_ffn(x, w13, w2, output=inner), want)

    leaf = torch.empty_like(x).requires_grad_()
    with pytest.raises(RuntimeError, match="output must not require gradients"):
        ffn_host.gated_ffn(x, w13, w2, output=leaf)
    with torch.no_grad():
        ffn_host.gated_ffn(x, w13, w2, output=leaf)
    assert torch.equal(leaf, want)
    buffer = torch.zeros(24, 64, dtype=x.dtype, device="cuda")
    for first in (1, 8, 15):
        with pytest.raises(RuntimeError, match="output must not overlap an input"):
            ffn_host.gated_ffn(buffer[8:16], w13, w2, output=buffer[first:first + 8])
    ffn_host.gated_ffn(buffer[8:16], w13, w2, output=buffer[:8])
    ffn_host.gated_ffn(buffer[8:16], w13, w2, output=buffer[16:])

    q, scale = ffn_host.mxfp4_quantize(w13)
    q2, scale2 = ffn_host.mxfp4_quantize(w2)
    square = torch.zeros(8, 64, dtype=x.dtype, device="cuda")
    for call in (lambda: ffn_host.mxfp4_gated_ffn(square, q, scale, q2, scale2, output=square),
                 lambda: ffn_host.mxfp4_linear(square, q, scale, output=square)):
        with pytest.raises(RuntimeError, match="output must not overlap an input"):
            call()
    raw = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    a = raw[:1024].view(32, 32)
    a_scale = ffn_host.mxfp4_quantize(torch.zeros(32, 64, device="cuda"))[1]
    with pytest.raises(RuntimeError, match="output must not overlap an input"):
        ffn_host.mxfp4_matmul(a, a_scale, a, a_scale, output=raw[512:512 + 2048].view(torch.bfloat16).view(32, 32))

    with fwad.dual_level(), pytest.raises(RuntimeError):
        ffn_host.gated_ffn(fwad.make_dual(x, torch.ones_like(x)), w13, w2)


def test_host_tensors_are_refused():
    import ffn_host

    x, w13, w2, dy = _inputs(2, 64, 32, torch.bfloat16, device="cpu")
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ffn_host.gated_ffn(x, w13, w2)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ffn_host.gated_ffn(x.requires_grad_(), w13, w2)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ffn_host.gated_ffn_backward(dy, x, w13, w2, (torch.zeros(2, 64), torch.zeros(2, 32)))


def test_c_abi_refusals():
    """Bad sizes, codes, pointers and workspaces come back as status codes
    before any device is touched."""
    import ffn_host

    lib = ffn_host._library()
    p = 1 << 20                      # a well-aligned address that nothing dereferences
    big = 1 << 40

    def fwd(x=p, pitch=64, w13=p, w2=p, dtype=0, act=0, T=4, H=64, inter=32, out=p, pre=p, hid=None, ws=p, n=big):
        return lib.moe_b200_gated_ffn(x, pitch, w13, w2, dtype, act, T, H, inter, out, pre, hid, ws, n, None)

    for bad in ({"T": -1}, {"T": 262145}, {"H": 0}, {"H": 60, "pitch": 64}, {"H": 65544, "pitch": 65544},
                {"inter": 0}, {"inter": 12}, {"dtype": 2}, {"dtype": -1}, {"act": 2}, {"pitch": 56}, {"x": None},
                {"w13": None}, {"w2": None}, {"out": None}, {"ws": None}):
        assert fwd(**bad) == 1, bad
    for bad in ({"x": p + 8}, {"pitch": 68}, {"w13": p + 2}, {"w2": p + 8}, {"out": p + 8}, {"pre": p + 16},
                {"hid": p + 8}, {"ws": p + 128}):
        assert fwd(**bad) == 2, bad
    need = lib.moe_b200_gated_ffn_workspace_bytes(4, 64, 32)
    assert need >= 2 * 4 * 32 * 2 and fwd(n=need - 1) == 3
    assert fwd(hid=p, n=need - 1) == 3 and fwd(hid=p, ws=None) == 1   # the second part of up to 64 tokens' hidden
    need = lib.moe_b200_gated_ffn_workspace_bytes(129, 64, 32)
    assert need >= 129 * 32 * 2 and fwd(T=129, n=need - 1) == 3
    assert fwd(T=0, x=None, out=None) == 0

    def bwd(dy=p, gp=64, x=p, xp=64, w13=p, w2=p, pre=p, hid=p, dtype=0, act=0, T=4, H=64, inter=32, gx=p, g13=p, g2=p,
            ws=p, n=big):
        return lib.moe_b200_gated_ffn_backward(dy, gp, x, xp, w13, w2, pre, hid, dtype, act, T, H, inter, gx, g13, g2,
                                               ws, n, None)

    for bad in ({"T": -1}, {"H": 4}, {"inter": 4}, {"dtype": 2}, {"act": -1}, {"gp": 8}, {"xp": 8}, {"dy": None},
                {"x": None}, {"w13": None}, {"w2": None}, {"pre": None}, {"hid": None}, {"ws": None}):
        assert bwd(**bad) == 1, bad
    for bad in ({"dy": p + 8}, {"gp": 68}, {"xp": 68}, {"pre": p + 16}, {"gx": p + 8}, {"g13": p + 8}, {"g2": p + 8},
                {"ws": p + 16}):
        assert bwd(**bad) == 2, bad
    need = lib.moe_b200_gated_ffn_backward_workspace_bytes(4, 64, 32)
    assert need >= 2 * 4 * 64 * 2 and bwd(n=need - 1) == 3
    assert lib.moe_b200_gated_ffn_workspace_bytes(-1, 64, 32) == 0
    assert lib.moe_b200_gated_ffn_backward_workspace_bytes(4, 64, 33) == 0
    assert lib.moe_b200_dense_read_status(None, None) == 1
