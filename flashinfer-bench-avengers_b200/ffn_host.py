"""Host side of the dense operators beside the routed experts: the gated
feed-forward block (the shared expert of a layer) with its gradients, and
4-bit microscaled matrices with the block's 4-bit serving form. Argument
checks, workspaces and the ctypes binding, in the manner of moe_host.

All computation runs in the library's sm_100a kernels; there is no CPU or
framework fallback. The reference implements the routed experts only
(solution/cuda/main.py:31-54) and has no counterpart. Bad arguments raise
RuntimeError before any device work.

Calls run on the current stream of the inputs' device. Scratch comes from
torch's caching allocator call by call, so calls on several streams and
captured graphs never share it.
"""
from __future__ import annotations

import ctypes

import torch

import moe_host

MAX_TOKENS = moe_host.MAX_TOKENS
MAX_DIM = 65536
ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}

_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_INT = ctypes.c_int
_SIZE = ctypes.c_size_t

_check = moe_host._check
_raise_on = moe_host._raise_on

_SIGNATURES = {
    "moe_b200_gated_ffn_workspace_bytes": (_SIZE, [_I64, _I64, _I64]),
    "moe_b200_gated_ffn": (_INT, [_P, _I64, _P, _P, _INT, _INT, _I64, _I64, _I64, _P, _P, _P, _P, _SIZE, _P]),
    "moe_b200_gated_ffn_backward_workspace_bytes": (_SIZE, [_I64, _I64, _I64]),
    "moe_b200_gated_ffn_backward": (_INT, [_P, _I64, _P, _I64, _P, _P, _P, _P, _INT, _INT, _I64, _I64, _I64, _P, _P,
                                           _P, _P, _SIZE, _P]),
    "moe_b200_mxfp4_scale_bytes": (_SIZE, [_I64, _I64]),
    "moe_b200_mxfp4_quantize": (_INT, [_P, _I64, _INT, _I64, _I64, _P, _P, _P]),
    "moe_b200_mxfp4_dequantize": (_INT, [_P, _P, _I64, _I64, _INT, _P, _P]),
    "moe_b200_mxfp4_matmul": (_INT, [_P, _P, _P, _P, _I64, _I64, _I64, _INT, _P, _P]),
    "moe_b200_mxfp4_linear_workspace_bytes": (_SIZE, [_I64, _I64]),
    "moe_b200_mxfp4_linear": (_INT, [_P, _I64, _INT, _P, _P, _I64, _I64, _I64, _P, _P, _SIZE, _P]),
    "moe_b200_mxfp4_gated_ffn_workspace_bytes": (_SIZE, [_I64, _I64, _I64]),
    "moe_b200_mxfp4_gated_ffn": (_INT, [_P, _I64, _INT, _P, _P, _P, _P, _INT, _I64, _I64, _I64, _P, _P, _SIZE, _P]),
    "moe_b200_dense_read_status": (_INT, [ctypes.POINTER(ctypes.c_uint32), _P]),
}

_bound = None


def _library() -> ctypes.CDLL:
    global _bound
    if _bound is None:
        lib = moe_host.load_library()
        for name, (restype, argtypes) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = restype, argtypes
        _bound = lib
    return _bound


# ------------------------------------------------------------------ checks
# Every entry point first tests all its conditions in one expression, a
# microsecond or two; only where one fails does it go through them one by one
# for the message. (Building the messages on every call cost more than the
# launches: 33 us a call of the block at one token, now 17.)
def _check_cuda(name: str, t, dev=None) -> None:
    _check(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    _check(t.is_cuda, f"{name} must be CUDA")
    _check(dev is None or t.device == dev, f"{name} must be on {dev}")


def _check_dim(name: str, d: int, multiple: int) -> None:
    _check(multiple <= d <= MAX_DIM and d % multiple == 0,
           f"{name} must be a multiple of {multiple} from {multiple} to {MAX_DIM}, got {d}")


def _check_rows(name: str, t: torch.Tensor, cols: int | None = None) -> int:
    """Rows that may lie apart, each contiguous; returns their pitch in elements."""
    pitch = _pitch(t)
    if pitch >= 0 and (cols is None or t.size(1) == cols):
        return pitch
    _check(t.dim() == 2 and (cols is None or t.size(1) == cols),
           f"{name} must be [T, {cols if cols is not None else 'K'}]")
    _check(t.size(0) <= MAX_TOKENS, f"{name} has more than {MAX_TOKENS} rows")
    pitch = t.stride(0) if t.size(0) > 1 else t.size(1)
    _check(t.stride(1) == 1 and pitch >= t.size(1), f"{name} must have contiguous rows that do not overlap")
    _check(False, f"{name}'s rows must start on 16 bytes")


def _pitch(t: torch.Tensor) -> int:
    """Elements between the rows of a matrix the kernels can read, else -1:
    rows contiguous, not overlapping, each starting on 16 bytes."""
    stride, shape = t.stride(), t.shape
    if len(shape) != 2:
        return -1
    rows, cols = shape
    pitch = stride[0] if rows > 1 else cols
    if (stride[1] != 1 and cols > 1) or pitch < cols or rows > MAX_TOKENS:
        return -1
    if rows and (t.data_ptr() & 15 or (rows > 1 and pitch * t.element_size() & 15)):
        return -1
    # a lone row has no pitch; its length, a multiple of 16 bytes where the
    # size checks pass, stands in
    return pitch


def _is_dense(t, shape: tuple, dtype: torch.dtype, dev_index: int, align: int = 16) -> bool:
    return (t.dtype is dtype and t.shape == shape and t.get_device() == dev_index and t.is_contiguous()
            and not t.data_ptr() & (align - 1))


def _check_dense(name: str, t, shape: tuple, dtype: torch.dtype, dev, align: int = 16) -> None:
    if isinstance(t, torch.Tensor) and _is_dense(t, shape, dtype, dev.index, align):
        return
    _check_cuda(name, t, dev)
    _check(tuple(t.shape) == shape and t.dtype == dtype and t.is_contiguous(),
           f"{name} must be a contiguous {dtype} tensor of shape {shape}")
    _check(t.numel() == 0 or t.data_ptr() % align == 0, f"{name} must be {align}-byte aligned")


def _activation(name: str) -> int:
    act = ACTIVATIONS.get(name)
    if act is None:
        raise RuntimeError(f"activation must be one of {sorted(ACTIVATIONS)}, got {name!r}")
    return act


def _scratch(nbytes: int, x: torch.Tensor) -> torch.Tensor:
    """Device memory beside x, in elements of x (cheaper to allocate than with
    a type and a device to look up)."""
    return x.new_empty(nbytes // x.element_size() + 1)


def _mx_bytes(rows: int, cols: int) -> int:
    """At least what a 4-bit matrix takes in a workspace, parts 256-byte aligned."""
    return rows * cols // 2 + -(-rows // 128) * -(-cols // 128) * 512 + 1024


def _call(name: str, dev: torch.device, *args) -> None:
    """The library function on the current stream of ``dev``, with ``dev`` the
    current device."""
    idx = dev.index
    fn = getattr(_bound or _library(), name)
    if idx == torch._C._cuda_getDevice():
        code = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    else:
        with torch.cuda.device(idx):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    if code:
        _raise_on(code, name)


# ------------------------------------------------- gated feed-forward block
def _check_ffn(x, w13, w2) -> tuple[int, int, int, int]:
    """(T, H, I, x pitch) of checked inputs."""
    try:
        H, inter = w2.shape
        dtype, idx = x.dtype, x.get_device()
        pitch = _pitch(x)
        if (pitch >= 0 and x.shape[1] == H and idx >= 0 and (dtype is torch.bfloat16 or dtype is torch.float16)
                and not (H | inter) & 7 and 8 <= H <= MAX_DIM and 8 <= inter <= MAX_DIM
                and _is_dense(w13, (2 * inter, H), dtype, idx) and _is_dense(w2, (H, inter), dtype, idx)):
            return x.shape[0], H, inter, pitch
    except (AttributeError, TypeError, ValueError):   # not tensors, or not matrices
        pass
    _check_cuda("x", x)
    _check(x.dtype in (torch.bfloat16, torch.float16), "x must be bfloat16 or float16")
    pitch = _check_rows("x", x)
    T, H = x.shape
    _check_dim("the hidden size", H, 8)
    _check_cuda("w13", w13, x.device)
    _check(w13.dim() == 2 and w13.size(0) % 2 == 0 and w13.size(0) > 0, f"w13 must be [2 I, {H}]")
    inter = w13.size(0) // 2
    _check_dim("the intermediate size", inter, 8)
    _check_dense("w13", w13, (2 * inter, H), x.dtype, x.device)
    _check_dense("w2", w2, (H, inter), x.dtype, x.device)
    return T, H, inter, pitch


def _run_ffn(x, w13, w2, activation, output, save: bool):
    T, H, inter, pitch = _check_ffn(x, w13, w2)
    act = _activation(activation)
    dev = x.device
    if output is not None:
        _check_dense("output", output, (T, H), x.dtype, dev)
    else:   # (the cheaper way where x has the output's layout)
        output = torch.empty_like(x) if pitch == H else x.new_empty((T, H))
    hidden = preact = None
    if save:
        hidden = x.new_empty((T, inter))
        preact = torch.empty((T, 2 * inter), dtype=torch.float32, device=dev)
    if T:
        ws = _scratch((4 if T <= 16 else 2) * T * inter + 1024, x) if T <= 16 or not save else None
        _call("moe_b200_gated_ffn", dev, x.data_ptr(), pitch, w13.data_ptr(), w2.data_ptr(), TYPES[x.dtype], act, T,
              H, inter, output.data_ptr(), preact.data_ptr() if save else None, hidden.data_ptr() if save else None,
              ws.data_ptr() if ws is not None else None, ws.nbytes if ws is not None else 0)
    return output, preact, hidden


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, activation):
        output, preact, hidden = _run_ffn(x, w13, w2, activation, None, True)
        ctx.save_for_backward(x, w13, w2, preact, hidden)
        ctx.activation = activation
        return output

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        x, w13, w2, preact, hidden = ctx.saved_tensors
        needs = ctx.needs_input_grad
        rows_ok = grad_output.stride(1) == 1 and (grad_output.size(0) < 2 or (
            grad_output.stride(0) >= grad_output.size(1) and grad_output.stride(0) % 8 == 0))
        if not rows_ok or grad_output.data_ptr() % 16:   # e.g. the expanded gradient of a sum
            grad_output = grad_output.clone(memory_format=torch.contiguous_format)
        return (*gated_ffn_backward(grad_output, x, w13, w2, (preact, hidden), ctx.activation, needs[:3]), None)


def gated_ffn(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, activation: str = "silu",
              output: torch.Tensor | None = None) -> torch.Tensor:
    """The gated feed-forward block: with [u | g] = x w13^T (w13 [2I, H], up
    rows first, the order of the routed experts' gemm1_weights),
    (act(g) * u) w2^T as [T, H] in x's type (bf16 or fp16). ``activation`` is
    "silu" or "gelu_tanh". Rows of x may lie apart. Differentiable in x, w13
    and w2; ``output`` takes the result of a call without gradients.

    A backward pass that is to be captured into a CUDA graph is best written
    with gated_ffn_forward / gated_ffn_backward: the autograd engine binds
    each leaf to the stream of its first use, the two functions use the
    current stream alone."""
    if torch.is_grad_enabled() and (getattr(x, "requires_grad", False) or getattr(w13, "requires_grad", False)
                                    or getattr(w2, "requires_grad", False)):
        _check(output is None, "output cannot be given where gradients are recorded")
        return _GatedFFN.apply(x, w13, w2, activation)
    return _run_ffn(x, w13, w2, activation, output, False)[0]


def gated_ffn_forward(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, activation: str = "silu"):
    """gated_ffn for training without autograd: (output, saved), ``saved`` for
    gated_ffn_backward: u and g in fp32 [T, 2I], and h [T, I]."""
    output, preact, hidden = _run_ffn(x, w13, w2, activation, None, True)
    return output, (preact, hidden)


def gated_ffn_backward(grad_output: torch.Tensor, x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, saved,
                       activation: str = "silu", needs=(True, True, True)):
    """(grad_x, grad_w13, grad_w2) for ``grad_output`` [T, H], in the inputs'
    type; None where ``needs`` is false. Bit for bit the same on every call."""
    T, H, inter, pitch = _check_ffn(x, w13, w2)
    act = _activation(activation)
    dev = x.device
    _check_cuda("grad_output", grad_output, dev)
    if grad_output.dtype != x.dtype or grad_output.shape != (T, H):
        raise RuntimeError(f"grad_output must be {x.dtype} [{T}, {H}] like the output")
    grad_pitch = _check_rows("grad_output", grad_output, H)
    if not isinstance(saved, (tuple, list)) or len(saved) != 2:
        raise RuntimeError("saved must be the pair that gated_ffn_forward returned")
    preact, hidden = saved
    _check_dense("saved u and g", preact, (T, 2 * inter), torch.float32, dev, 32)
    _check_dense("saved hidden", hidden, (T, inter), x.dtype, dev)
    if len(needs) != 3:
        raise RuntimeError("needs must be three truth values")
    grads = [x.new_empty(shape) if n else None for shape, n in zip(((T, H), (2 * inter, H), (H, inter)), needs)]
    if needs[0] or needs[1] or needs[2]:
        ws = _scratch(4 * T * inter + 1024, x)
        _call("moe_b200_gated_ffn_backward", dev, grad_output.data_ptr(), grad_pitch, x.data_ptr(), pitch,
              w13.data_ptr(), w2.data_ptr(), preact.data_ptr(), hidden.data_ptr(), TYPES[x.dtype], act, T, H, inter,
              *(g.data_ptr() if g is not None else None for g in grads), ws.data_ptr(), ws.nbytes)
    return tuple(grads)


# ------------------------------------------------- 4-bit microscaled matrices
def mxfp4_scale_shape(rows: int, cols: int) -> tuple[int, ...]:
    """Shape of the exponent bytes of a 4-bit matrix [rows, cols]: the byte of
    row r, 32-column block b is at [r // 128, b // 4, r % 32, r % 128 // 32, b % 4]."""
    return (-(-rows // 128), -(-cols // 128), 32, 4, 4)


def _check_values(name: str, x) -> int:
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in TYPES:
        pitch = _pitch(x)
        if pitch >= 0 and not x.shape[1] & 31 and 32 <= x.shape[1] <= MAX_DIM:
            return pitch
    _check_cuda(name, x)
    _check(x.dtype in TYPES, f"{name} must be bfloat16, float16 or float32")
    pitch = _check_rows(name, x)
    _check_dim(f"{name}'s row length", x.size(1), 32)
    return pitch


def _check_mx(name: str, q, scale, dev=None, cols: int | None = None, rows: int | None = None) -> tuple[int, int]:
    """(rows, columns) of a checked 4-bit matrix."""
    try:
        r, half = q.shape
        idx = q.get_device()
        if (idx >= 0 and (dev is None or idx == dev.index) and q.dtype is torch.uint8 and q.is_contiguous()
                and r <= MAX_TOKENS and not half & 15 and 16 <= half <= MAX_DIM // 2
                and (cols is None or 2 * half == cols) and (rows is None or r == rows) and not q.data_ptr() & 15
                and _is_dense(scale, mxfp4_scale_shape(r, 2 * half), torch.uint8, idx)):
            return r, 2 * half
    except (AttributeError, TypeError, ValueError):
        pass
    _check_cuda(name, q, dev)
    _check(q.dtype == torch.uint8 and q.dim() == 2 and q.is_contiguous(),
           f"{name} must be contiguous uint8 codes [R, K / 2]")
    r, k = q.size(0), 2 * q.size(1)
    _check(r <= MAX_TOKENS, f"{name} has more than {MAX_TOKENS} rows")
    _check_dim(f"{name}'s row length", k, 32)
    _check(cols is None or k == cols, f"{name} must have {cols} columns, got {k}")
    _check(rows is None or r == rows, f"{name} must have {rows} rows, got {r}")
    _check(r == 0 or q.data_ptr() % 16 == 0, f"{name} must be 16-byte aligned")
    _check_dense(f"{name}'s scale", scale, mxfp4_scale_shape(r, k), torch.uint8, q.device)
    return r, k


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [R, K] (bf16, fp16 or fp32; K a multiple of 32; rows may lie apart) in
    4 bits: codes uint8 [R, K / 2] and exponent bytes uint8 of
    mxfp4_scale_shape(R, K) (moe_b200_mxfp4_quantize)."""
    pitch = _check_values("x", x)
    R, K = x.shape
    dev = x.device
    q = torch.empty((R, K // 2), dtype=torch.uint8, device=dev)
    scale = q.new_empty(mxfp4_scale_shape(R, K))
    if R:
        _call("moe_b200_mxfp4_quantize", dev, x.data_ptr(), pitch, TYPES[x.dtype], R, K, q.data_ptr(),
              scale.data_ptr())
    return q, scale


def mxfp4_dequantize(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The [R, K] values that a 4-bit matrix stands for, in ``dtype``."""
    R, K = _check_mx("q", q, scale)
    _check_type(dtype)
    dev = q.device
    out = torch.empty((R, K), dtype=dtype, device=dev)
    if R:
        _call("moe_b200_mxfp4_dequantize", dev, q.data_ptr(), scale.data_ptr(), R, K, TYPES[dtype], out.data_ptr())
    return out


def _check_type(dtype) -> None:
    if dtype not in TYPES:
        raise RuntimeError("dtype must be bfloat16, float16 or float32")


def _output(output, shape: tuple, x: torch.Tensor) -> torch.Tensor:
    """``output`` checked, or a new tensor, of x's type."""
    if output is None:
        return x.new_empty(shape)
    _check_dense("output", output, shape, x.dtype, x.device)
    return output


def mxfp4_matmul(a_q: torch.Tensor, a_scale: torch.Tensor, b_q: torch.Tensor, b_scale: torch.Tensor,
                 dtype: torch.dtype = torch.bfloat16, output: torch.Tensor | None = None) -> torch.Tensor:
    """A B^T of two 4-bit matrices [M, K] and [N, K]: fp32 sums, rounded once
    to ``dtype``."""
    M, K = _check_mx("a_q", a_q, a_scale)
    N, _ = _check_mx("b_q", b_q, b_scale, a_q.device, K)
    if N == 0:
        raise RuntimeError("b_q must have rows")
    _check_type(dtype)
    dev = a_q.device
    if output is None:
        output = torch.empty((M, N), dtype=dtype, device=dev)
    else:
        _check_dense("output", output, (M, N), dtype, dev)
    if M:
        _call("moe_b200_mxfp4_matmul", dev, a_q.data_ptr(), a_scale.data_ptr(), b_q.data_ptr(), b_scale.data_ptr(),
              M, N, K, TYPES[dtype], output.data_ptr())
    return output


def mxfp4_linear(x: torch.Tensor, w_q: torch.Tensor, w_scale: torch.Tensor,
                 output: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, K] times a 4-bit weight [N, K]: x is brought to 4 bits inside the
    call, the result [T, N] has x's type."""
    pitch = _check_values("x", x)
    T, K = x.shape
    dev = x.device
    N, _ = _check_mx("w_q", w_q, w_scale, dev, K)
    if N == 0:
        raise RuntimeError("w_q must have rows")
    output = _output(output, (T, N), x)
    if T:
        ws = _scratch(_mx_bytes(T, K), x)
        _call("moe_b200_mxfp4_linear", dev, x.data_ptr(), pitch, TYPES[x.dtype], w_q.data_ptr(), w_scale.data_ptr(),
              T, N, K, output.data_ptr(), ws.data_ptr(), ws.nbytes)
    return output


def mxfp4_gated_ffn(x: torch.Tensor, w13_q: torch.Tensor, w13_scale: torch.Tensor, w2_q: torch.Tensor,
                    w2_scale: torch.Tensor, activation: str = "silu",
                    output: torch.Tensor | None = None) -> torch.Tensor:
    """The gated feed-forward block with 4-bit weights and activations, for
    serving: [u | g] = Q(x) w13^T, Q(act(g) * u) w2^T with Q the quantiser of
    mxfp4_quantize; the result [T, H] has x's type."""
    pitch = _check_values("x", x)
    T, H = x.shape
    dev = x.device
    act = _activation(activation)
    two_i, _ = _check_mx("w13_q", w13_q, w13_scale, dev, H)
    inter = two_i // 2
    if two_i & 63 or not two_i:
        raise RuntimeError(f"w13_q must have 2 I rows, I a multiple of 32; got {two_i}")
    _check_dim("the intermediate size", inter, 32)
    _check_mx("w2_q", w2_q, w2_scale, dev, inter, H)
    output = _output(output, (T, H), x)
    if T:
        ws = _scratch(_mx_bytes(T, H) + _mx_bytes(T, inter) + 8 * T * inter + 1024, x)
        _call("moe_b200_mxfp4_gated_ffn", dev, x.data_ptr(), pitch, TYPES[x.dtype], w13_q.data_ptr(),
              w13_scale.data_ptr(), w2_q.data_ptr(), w2_scale.data_ptr(), act, T, H, inter, output.data_ptr(),
              ws.data_ptr(), ws.nbytes)
    return output


def read_status(device: torch.device | None = None) -> int:
    """Status word of the dense operators on ``device`` since the last read
    (0 = clean); synchronises the current stream and clears the word."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    st = ctypes.c_uint32(0)
    with torch.cuda.device(dev):
        code = _library().moe_b200_dense_read_status(ctypes.byref(st), torch.cuda.current_stream(dev).cuda_stream)
    if code not in (0, 7):
        _raise_on(code, "moe_b200_dense_read_status")
    return int(st.value)
