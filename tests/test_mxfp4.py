"""4-bit microscaled matrices: the quantiser bit for bit, the product and the
4-bit feed-forward block within derived bounds, and a run of the dense
operators together; refusals on the CPU."""
from __future__ import annotations

import pytest
import torch

import dense_reference as ref

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows(R, K, dtype, seed=0):
    """Rows of unequal magnitude with edge blocks at the front: all zero,
    negative zeros, exact ties, values beyond 6 after scaling, the smallest
    and largest magnitudes of the type, infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    span = 12 if dtype == torch.float16 else 60
    x = torch.randn(R, K, generator=g) * torch.exp2(torch.randint(-span, span // 2, (R, 1), generator=g).float())
    x = x.to(dtype)
    b = x.view(R, K // 32, 32)
    info = torch.finfo(dtype)
    edges = [torch.zeros(32), torch.full((32,), -0.0),
             torch.tensor([0.25, -0.25, 0.75, 1.25, -1.75, 2.5, 3.5, -3.5, 5.0, 4.0] + [0.125] * 22),
             torch.tensor([7.9, 7.0, 6.99, -7.5, 6.0, 5.1, 4.9, 0.2] * 4), torch.full((32,), info.max),
             torch.tensor([info.tiny, -info.smallest_normal] * 16), torch.tensor([info.smallest_normal / 4, 0.0] * 16),
             torch.tensor([float("inf")] + [1.0] * 31), torch.tensor([1.0] * 31 + [float("nan")]),
             torch.tensor([float("-inf"), float("nan")] * 16)]
    flat = b.reshape(-1, 32)
    for i, e in enumerate(edges[: flat.shape[0] if R * K > 32 * len(edges) else 0]):
        flat[i] = e.to(dtype)
    return flat.view(R, K).clone()


@pytest.mark.gpu
@pytest.mark.parametrize("R,K", [(1, 32), (1, 7168), (2, 96), (31, 128), (129, 160), (300, 1056), (53, 4096)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_is_exact(cuda_device, R, K, dtype):
    import ffn_host

    x = _rows(R, K, dtype)
    q, scale = ffn_host.mxfp4_quantize(x.cuda())
    want_q, want_scale = ref.mx_quantize(x)
    assert scale.shape == ffn_host.mxfp4_scale_shape(R, K)
    assert torch.equal(scale.cpu(), want_scale)      # also the zeros in places that do not exist
    assert torch.equal(q.cpu(), want_q)
    for to in TYPES:
        got = ffn_host.mxfp4_dequantize(q, scale, to).cpu()
        assert torch.equal(torch.nan_to_num(got, nan=1.5e30 if to != torch.float16 else 777.0),
                           torch.nan_to_num(ref.mx_values(q, scale).to(to), nan=1.5e30 if to != torch.float16 else 777.0))


@pytest.mark.gpu
def test_quantize_rows_apart(cuda_device):
    import ffn_host

    x = torch.randn(40, 256, device="cuda", dtype=torch.bfloat16)
    for off, cols in ((8, 96), (16, 224), (24, 64)):
        part = x[:, off:off + cols]
        a, b = ffn_host.mxfp4_quantize(part), ffn_host.mxfp4_quantize(part.contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def _matrix(R, K, seed):
    """A random 4-bit matrix on the CPU with exponents spread over 2^-20 .. 2^8."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K // 32, 32, generator=g) * torch.exp2(torch.randint(-18, 7, (R, K // 32, 1), generator=g).float())
    return ref.mx_quantize(x.view(R, K))


# ends inside every tile: 128- and 256-row tiles, 256- and 64-wide K steps
PRODUCTS = [(1, 1, 32), (1, 128, 64), (3, 77, 96), (16, 4096, 256), (17, 300, 288), (65, 129, 544), (128, 256, 2048),
            (129, 128, 160), (256, 255, 512), (300, 513, 1056), (520, 1000, 320)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_product(cuda_device, M, N, K, dtype):
    import ffn_host

    a, b = _matrix(M, K, 1), _matrix(N, K, 2)
    got = ffn_host.mxfp4_matmul(a[0].cuda(), a[1].cuda(), b[0].cuda(), b[1].cuda(), dtype)
    value, bound = ref.mx_product(ref.mx_values(*a), ref.mx_values(*b), dtype)
    # exponents to 2^16 leave fp16's range: compare where the value fits
    keep = (value.abs() + bound < 65000.0) if dtype == torch.float16 else torch.ones_like(value, dtype=torch.bool)
    ref.assert_within(got.cpu()[keep], (value[keep], bound[keep]), "product")
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 200])
def test_nan_blocks_stay_in_their_rows(cuda_device, M):
    import ffn_host

    a, b = _matrix(M, 320, 3), _matrix(150, 320, 4)
    args = [t.cuda() for t in (*a, *b)]
    clean = ffn_host.mxfp4_matmul(*args)
    args[1][0, 2, 1, 0, 1] = 255       # row 1, the last block but one of the ragged tile
    args[3][1, 0, 5, 0, 0] = 255       # row 133 of B
    got = ffn_host.mxfp4_matmul(*args)
    spoilt = torch.zeros(M, 150, dtype=torch.bool, device="cuda")
    spoilt[1] = True
    spoilt[:, 133] = True
    assert torch.isnan(got[spoilt]).all() and torch.equal(got[~spoilt], clean[~spoilt])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20, 65, 128, 130, 400])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear(cuda_device, T, dtype):
    """Equal to quantiser and product called one after the other, within the
    64-bit bounds; rows of x that lie apart; an output inside a buffer."""
    import ffn_host

    N, K = 333, 416
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(T, K + 64, generator=g, device="cuda").to(dtype)
    x = wide[:, 32:32 + K]
    w = ffn_host.mxfp4_quantize(torch.randn(N, K, generator=g, device="cuda"))
    buf = torch.full((T + 2, 336), 3.0, dtype=dtype, device="cuda")
    flat = buf.view(-1)[336:336 + T * N].view(T, N)
    got = ffn_host.mxfp4_linear(x, *w, output=flat)
    xq = ffn_host.mxfp4_quantize(x)
    assert torch.equal(got, ffn_host.mxfp4_matmul(*xq, *w, dtype))
    ref.assert_within(got.cpu(), ref.mx_product(ref.mx_values(*xq), ref.mx_values(*w), dtype), "linear")
    assert (buf.view(-1)[:336] == 3).all() and (buf.view(-1)[336 + T * N:] == 3).all()


def _check_block(x, w13, w2, activation, y, what):
    """The 4-bit block against 64 bits. The hidden is rounded to 4 bits from
    sums that differ in their last bits, so where the 64-bit value lies within
    the fp32 bound of a rounding border (or of a block's power of two) both
    neighbours are right: the bound takes the quantiser at both ends of the
    interval and allows their distance."""
    dt = x.dtype
    xv = ref.mx_values(*ref.mx_quantize(x))
    w13v, w2v = ref.mx_values(*w13), ref.mx_values(*w2)
    inter = w2v.shape[1]
    pre = xv @ w13v.T
    e_pre = ref.gamma(xv.shape[1]) * (xv.abs() @ w13v.abs().T)
    up, gate = pre[:, :inter], pre[:, inter:]
    a = ref.act(gate, activation)[0]
    e_a = 1.2 * e_pre[:, inter:] + ref.ACT * a.abs()
    h = a * up
    e_h = e_a * up.abs() + a.abs() * e_pre[:, :inter] + e_a * e_pre[:, :inter]
    # rounding error of the fp32 value itself, then both ends (each rounding
    # step is monotonic once the exponent is fixed; the exponent is fixed by
    # the largest magnitude, taken at both ends too)
    e_h = e_h + 2.0 ** -23 * h.abs()
    b = h.view(h.shape[0], -1, 32)
    e = e_h.view_as(b)
    ends = []
    for s in (-1, 1):
        top = (b.abs() + s * e).clamp(min=0).amax(2)
        exponent = (torch.frexp(top.clamp(min=1e-300))[1] - 3).clamp(min=-127).double()
        for t in (-1, 0, 1):
            v = ((b + t * e) / torch.exp2(exponent)[:, :, None]).clamp(-6, 6)
            step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
            ends.append(torch.round(v / step) * step * torch.exp2(exponent)[:, :, None])
    ends = torch.stack(ends)
    lo, hi = ends.amin(0).reshape(h.shape), ends.amax(0).reshape(h.shape)
    mid, half = (lo + hi) / 2, (hi - lo) / 2
    assert (half > 0).double().mean() < 0.02        # the borders are rare: the bound is tight almost everywhere
    value, bound = ref.mx_product(mid, w2v, dt)
    spread = half @ w2v.abs().T
    ref.assert_within(y.cpu(), (value, bound + spread * (1 + 2 * ref.U[dt])), what)


# T <= 64 and ragged I: the sums go through memory; T > 64 and whole
# 128-feature tiles: the hidden is brought to 4 bits in the GEMM's epilogue
@pytest.mark.gpu
@pytest.mark.parametrize("T,H,inter", [(1, 256, 128), (16, 544, 288), (64, 256, 256), (65, 544, 288),
                                       (100, 288, 256), (128, 256, 256), (129, 256, 256), (200, 288, 96),
                                       (300, 512, 640)])
@pytest.mark.parametrize("dtype,activation", [(torch.bfloat16, "silu"), (torch.float16, "gelu_tanh")])
def test_block(cuda_device, T, H, inter, dtype, activation):
    import ffn_host

    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(T, H, generator=g, device="cuda").to(dtype)
    w13 = ffn_host.mxfp4_quantize(torch.randn(2 * inter, H, generator=g, device="cuda") * H ** -0.5)
    w2 = ffn_host.mxfp4_quantize(torch.randn(H, inter, generator=g, device="cuda") * inter ** -0.5)
    y = ffn_host.mxfp4_gated_ffn(x, *w13, *w2, activation)
    assert y.dtype == dtype
    _check_block(x, w13, w2, activation, y, "block")
    assert torch.equal(y, ffn_host.mxfp4_gated_ffn(x, *w13, *w2, activation))
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
def test_zero_rows_and_no_rows(cuda_device):
    import ffn_host

    w13 = ffn_host.mxfp4_quantize(torch.randn(256, 128, device="cuda"))
    w2 = ffn_host.mxfp4_quantize(torch.randn(128, 128, device="cuda"))
    for T in (3, 140):
        x = torch.zeros(T, 128, device="cuda", dtype=torch.bfloat16)
        assert not ffn_host.mxfp4_gated_ffn(x, *w13, *w2).any()
        assert not ffn_host.mxfp4_linear(x, *w13).any()
    x = torch.zeros(0, 128, device="cuda", dtype=torch.bfloat16)
    assert ffn_host.mxfp4_gated_ffn(x, *w13, *w2).shape == (0, 128)
    assert ffn_host.mxfp4_linear(x, *w13).shape == (0, 256)
    q, s = ffn_host.mxfp4_quantize(x)
    assert q.shape == (0, 64) and s.numel() == 0 and ffn_host.mxfp4_dequantize(q, s).shape == (0, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 20, 200])
def test_captured_and_on_two_streams(cuda_device, T):
    """Linear and block captured into two graphs each, replayed on new inputs
    in turn, and called on two streams at once."""
    import ffn_host

    H, inter = 544, 256
    g = torch.Generator(device="cuda").manual_seed(8)
    xs = [torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    w13 = ffn_host.mxfp4_quantize(torch.randn(2 * inter, H, generator=g, device="cuda"))
    w2 = ffn_host.mxfp4_quantize(torch.randn(H, inter, generator=g, device="cuda"))

    def both(x):
        return ffn_host.mxfp4_linear(x, *w13), ffn_host.mxfp4_gated_ffn(x, *w13, *w2)

    want = [[t.clone() for t in both(x)] for x in xs]
    graphs = []
    for _ in range(2):
        static = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(static)
        graphs.append((graph, static, out))
    for k in (1, 0):
        for n, (graph, static, _) in enumerate(graphs):
            static.copy_(xs[(k + n) % 2])
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for n, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(k + n) % 2]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(6):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                outs.append(both(x))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2]))
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 300])
def test_weights_written_just_before(cuda_device, T):
    """Weights that a long kernel of the library, or a copy on a joined
    stream, writes right before the call: every kernel of the call sees them,
    eager and captured."""
    import ffn_host

    rows, H, inter = 16384, 1024, 512
    gen = torch.Generator(device="cuda").manual_seed(3)
    big = [torch.randn(rows, H, device="cuda", generator=gen, dtype=torch.bfloat16) for _ in range(2)]
    narrow = [b.view(2 * rows, inter) for b in big]
    x = torch.randn(T, H, device="cuda", generator=gen, dtype=torch.bfloat16)

    def linear(i):
        q, s = ffn_host.mxfp4_quantize(big[i])
        return ffn_host.mxfp4_linear(x, q[-1024:], s[-8:])

    def block4(i):
        q, s = ffn_host.mxfp4_quantize(big[i])
        q2, s2 = ffn_host.mxfp4_quantize(narrow[i])          # the last one written feeds the last GEMM
        return ffn_host.mxfp4_gated_ffn(x, q[-1024:], s[-8:], q2[-1024:], s2[-8:])

    def block16(i):
        w13 = ffn_host.mxfp4_dequantize(*ffn_host.mxfp4_quantize(big[i]))[-1024:]
        w2 = ffn_host.mxfp4_dequantize(*ffn_host.mxfp4_quantize(narrow[i]))[-1024:]
        return ffn_host.gated_ffn(x, w13, w2)

    for call in (linear, block4, block16):
        want = []
        for i in range(2):
            torch.cuda.synchronize()
            want.append(call(i).clone())
        for r in range(6):      # memory of the last round's weights, with the other weights in it
            assert torch.equal(call(r % 2), want[r % 2])

    w13, w2 = big[0][:1024].clone(), narrow[0][:1024].clone()
    source13, source2, side = big[0].clone(), narrow[0].clone(), torch.cuda.Stream()
    full2 = torch.zeros_like(narrow[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            full2.copy_(source2)                             # 34 MB
        w13.copy_(source13[-1024:])
        main.wait_stream(side)
        y = ffn_host.gated_ffn(x, w13, full2[-1024:])
        z = ffn_host.gated_ffn(x, w13, w2)
    for i in (1, 0, 1):
        source13.copy_(big[i]), source2.copy_(narrow[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ffn_host.gated_ffn(x, big[i][-1024:], narrow[i][-1024:]))
        assert torch.equal(z, ffn_host.gated_ffn(x, big[i][-1024:], w2))
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_device):
    """The most rows, more than 2^31 elements in all: rows at both ends."""
    import ffn_host

    T, K, N = ffn_host.MAX_TOKENS, 8224, 8216
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(9)
    ends = torch.randn(400, K, generator=g, device="cuda").to(torch.bfloat16)
    x[:200], x[T - 200:] = ends[:200], ends[200:]
    w = ffn_host.mxfp4_quantize(torch.randn(N, K, generator=g, device="cuda"))
    q, scale = ffn_host.mxfp4_quantize(x)
    few = ffn_host.mxfp4_quantize(ends)
    assert torch.equal(torch.cat([q[:200], q[T - 200:]]), few[0]) and not q[200:T - 200].any()
    back = ffn_host.mxfp4_dequantize(q, scale)
    assert torch.equal(torch.cat([back[:200], back[T - 200:]]), ffn_host.mxfp4_dequantize(*few))
    del back, q, scale
    y = ffn_host.mxfp4_linear(x, *w)
    assert torch.equal(torch.cat([y[:200], y[T - 200:]]), ffn_host.mxfp4_linear(ends, *w))
    assert not y[200:T - 200].any()
    assert ffn_host.read_status() == 0


@pytest.mark.gpu
def test_dense_operators_together(cuda_device):
    """As they are used: two fine-tuning steps of a block, its weights brought
    to 4 bits, then served to a prompt and token by token, from a captured
    graph and on a side stream. Every stage is checked on what went into it."""
    import ffn_host

    T, H, inter = 150, 512, 256
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    target = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    w13 = (torch.randn(2 * inter, H, generator=g, device="cuda") * H ** -0.5).to(torch.bfloat16).requires_grad_()
    w2 = (torch.randn(H, inter, generator=g, device="cuda") * inter ** -0.5).to(torch.bfloat16).requires_grad_()
    for _ in range(2):
        y = ffn_host.gated_ffn(x, w13, w2)
        dy = ((y - target) / T).detach()
        want = ref.ffn(x, w13.detach(), w2.detach(), "silu", dy)
        y.backward(dy)
        ref.assert_within(y.detach(), want["y"], "y")
        ref.assert_within(w13.grad, want["dw13"], "dw13")
        ref.assert_within(w2.grad, want["dw2"], "dw2")
        with torch.no_grad():
            for w in (w13, w2):
                w -= 0.05 * w.grad
                w.grad = None
    with torch.no_grad():
        q13, q2 = ffn_host.mxfp4_quantize(w13), ffn_host.mxfp4_quantize(w2)
    prompt = ffn_host.mxfp4_gated_ffn(x, *q13, *q2)
    _check_block(x, q13, q2, "silu", prompt, "prompt")
    static = x[:1].clone()
    ffn_host.mxfp4_gated_ffn(static, *q13, *q2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token = ffn_host.mxfp4_gated_ffn(static, *q13, *q2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for t in (0, 77, T - 1):
        static.copy_(x[t:t + 1])
        graph.replay()
        with torch.cuda.stream(side):
            lone = ffn_host.mxfp4_gated_ffn(x[t:t + 1], *q13, *q2)
        torch.cuda.synchronize()
        assert torch.equal(token, lone)
        _check_block(x[t:t + 1], q13, q2, "silu", token, "token")
    assert ffn_host.read_status() == 0


def test_reference_quantizer():
    """The 64-bit form itself on values whose result is known by hand."""
    x = torch.zeros(2, 32)
    x[0, :10] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.26])
    x[1, :2] = torch.tensor([1.0, 0.125])
    q, s = ref.mx_quantize(x)
    assert s[0, 0, 0, 0, 0] == 127 and s[0, 0, 1, 0, 0] == 125 and s.sum() == 252
    v = ref.mx_values(q, s)
    assert v[0, :10].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -0.5]
    assert v[1, :2].tolist() == [1.0, 0.125]


def test_host_tensors_are_refused():
    import ffn_host

    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)
    for call in (lambda: ffn_host.mxfp4_quantize(x), lambda: ffn_host.mxfp4_dequantize(q, s),
                 lambda: ffn_host.mxfp4_matmul(q, s, q, s), lambda: ffn_host.mxfp4_linear(x, q, s),
                 lambda: ffn_host.mxfp4_gated_ffn(x, q, s, q, s)):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            call()


@pytest.mark.gpu
def test_refusals_on_the_gpu(cuda_device):
    import ffn_host

    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    q, s = ffn_host.mxfp4_quantize(x)
    for call, message in [
        (lambda: ffn_host.mxfp4_quantize(x[:, :40]), "multiple of 32"),
        (lambda: ffn_host.mxfp4_quantize(x.int()), "bfloat16, float16 or float32"),
        (lambda: ffn_host.mxfp4_quantize(x[:, 4:36]), "start on 16 bytes"),
        (lambda: ffn_host.mxfp4_quantize(x.t()), "contiguous rows"),
        (lambda: ffn_host.mxfp4_dequantize(q, s[:, :, :16]), "scale must be"),
        (lambda: ffn_host.mxfp4_dequantize(q, s, torch.int32), "dtype must be"),
        (lambda: ffn_host.mxfp4_dequantize(q.int(), s), "uint8 codes"),
        (lambda: ffn_host.mxfp4_matmul(q, s, q[:, :16].contiguous(), s), "must have 64 columns"),
        (lambda: ffn_host.mxfp4_matmul(q, s, q[:0], s[:0]), "must have rows"),
        (lambda: ffn_host.mxfp4_matmul(q, s, q, s.cpu()), "must be CUDA"),
        (lambda: ffn_host.mxfp4_matmul(q, s, q, s, output=torch.empty(4, 4, device="cuda")), "output must be"),
        (lambda: ffn_host.mxfp4_linear(x[:, :32], q, s), "must have 32 columns"),
        (lambda: ffn_host.mxfp4_gated_ffn(x, q, s, q, s), "multiple of 32|must have"),
        (lambda: ffn_host.mxfp4_gated_ffn(x, q, s, q, s, "relu"), "activation"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()


def test_c_abi_refusals():
    import ffn_host

    lib = ffn_host._library()
    p, big = 1 << 20, 1 << 40
    assert lib.moe_b200_mxfp4_scale_bytes(129, 160) == 2 * 2 * 512
    assert lib.moe_b200_mxfp4_scale_bytes(129, 33) == 0 and lib.moe_b200_mxfp4_scale_bytes(-1, 32) == 0

    def quantize(x=p, pitch=64, dtype=0, R=4, K=64, q=p, s=p):
        return lib.moe_b200_mxfp4_quantize(x, pitch, dtype, R, K, q, s, None)

    def dequantize(q=p, s=p, R=4, K=64, dtype=0, out=p):
        return lib.moe_b200_mxfp4_dequantize(q, s, R, K, dtype, out, None)

    def matmul(a=p, sa=p, b=p, sb=p, M=4, N=4, K=64, dtype=0, out=p):
        return lib.moe_b200_mxfp4_matmul(a, sa, b, sb, M, N, K, dtype, out, None)

    def linear(x=p, pitch=64, dtype=0, w=p, sw=p, T=4, N=4, K=64, out=p, ws=p, n=big):
        return lib.moe_b200_mxfp4_linear(x, pitch, dtype, w, sw, T, N, K, out, ws, n, None)

    def block(x=p, pitch=64, dtype=0, w13=p, s13=p, w2=p, s2=p, act=0, T=4, H=64, inter=32, out=p, ws=p, n=big):
        return lib.moe_b200_mxfp4_gated_ffn(x, pitch, dtype, w13, s13, w2, s2, act, T, H, inter, out, ws, n, None)

    for call, bads in ((quantize, ({"R": -1}, {"K": 48}, {"K": 0}, {"dtype": 3}, {"pitch": 32}, {"x": None}, {"s": None})),
                       (dequantize, ({"R": -1}, {"K": 16}, {"dtype": -1}, {"q": None}, {"out": None})),
                       (matmul, ({"M": 262145}, {"N": 0}, {"K": 40}, {"dtype": 9}, {"sb": None}, {"out": None})),
                       (linear, ({"T": -2}, {"N": 0}, {"K": 8}, {"dtype": 5}, {"pitch": 0}, {"w": None}, {"ws": None})),
                       (block, ({"T": -2}, {"H": 40}, {"inter": 40}, {"act": 7}, {"dtype": 5}, {"s2": None}, {"ws": None}))):
        for bad in bads:
            assert call(**bad) == 1, (call.__name__, bad)
    for call, bads in ((quantize, ({"x": p + 8}, {"pitch": 68}, {"q": p + 8}, {"s": p + 4})),
                       (dequantize, ({"q": p + 8}, {"s": p + 8}, {"out": p + 8})),
                       (matmul, ({"a": p + 8}, {"sa": p + 8}, {"b": p + 8}, {"sb": p + 8}, {"out": p + 8})),
                       (linear, ({"x": p + 8}, {"pitch": 65}, {"w": p + 8}, {"out": p + 2}, {"ws": p + 16})),
                       (block, ({"x": p + 8}, {"w13": p + 8}, {"s13": p + 8}, {"w2": p + 8}, {"out": p + 8}, {"ws": p + 1}))):
        for bad in bads:
            assert call(**bad) == 2, (call.__name__, bad)
    assert linear(n=lib.moe_b200_mxfp4_linear_workspace_bytes(4, 64) - 1) == 3
    assert block(n=lib.moe_b200_mxfp4_gated_ffn_workspace_bytes(4, 64, 32) - 1) == 3
    for call, empty in ((quantize, {"R": 0}), (dequantize, {"R": 0}), (matmul, {"M": 0}), (linear, {"T": 0}),
                        (block, {"T": 0})):
        assert call(**empty) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("N", [136, 264, 260, 520, 257])
@pytest.mark.parametrize("dtype", TYPES)
def test_product_rows_by_their_alignment(cuda_device, N, dtype):
    """Over CTA pairs, rows of an output that start on 32 bytes, on 16 only, or
    anywhere, and outputs that begin 16 bytes into a larger buffer: the same
    numbers, and what lies around is left."""
    import ffn_host

    M, K = 140, 96
    a, b = _matrix(M, K, 5), _matrix(N, K, 6)
    args = [t.cuda() for t in (*a, *b)]
    value, bound = ref.mx_product(ref.mx_values(*a), ref.mx_values(*b), dtype)
    keep = (value.abs() + bound < 65000.0) if dtype == torch.float16 else torch.ones_like(value, dtype=torch.bool)
    pad = 16 // torch.empty(0, dtype=dtype).element_size()
    for first in (0, pad, 2 * pad):
        buf = torch.full((first + M * N + 3 * pad,), 5.0, dtype=dtype, device="cuda")
        out = buf[first:first + M * N].view(M, N)
        assert ffn_host.mxfp4_matmul(*args, dtype, output=out) is out
        ref.assert_within(out.cpu()[keep], (value[keep], bound[keep]), "product")
        assert (buf[:first] == 5).all() and (buf[first + M * N:] == 5).all()
