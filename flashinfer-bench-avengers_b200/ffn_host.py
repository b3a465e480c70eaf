"""Host side of the dense operators beside the routed experts: the gated
feed-forward block (the shared expert of a layer) with its gradients, and
4-bit microscaled matrices with the block's 4-bit serving form.

All computation runs in the library's sm_100a kernels; there is no CPU or
framework fallback. The reference implements the routed experts only
(solution/cuda/main.py:31-54) and has no counterpart. Bad arguments raise
RuntimeError before any device work.

Calls go through a small native binding (csrc/torch_binding.cpp), which tests
their conditions, allocates and launches; where it declines, the checks here
find the argument at fault and say so. They run on the current stream of the
inputs' device. Scratch comes from torch's caching allocator call by call, so
calls on several streams and captured graphs never share it. An ``output`` is
written in place; it may overlap no input.

Gradients are recorded by gated_ffn alone. The 4-bit functions serve: an x that
requires gradients is refused while gradients are recorded (but for the
quantiser, whose codes are integers). No function computes forward-mode
derivatives: a tensor with a tangent is refused while forward mode is on, with
torch.no_grad() too.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import threading

import torch
from torch.autograd import forward_ad

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

# The C ABI, for callers of the library itself and for the binding.
_SIGNATURES = {
    "moe_b200_gated_ffn": (_INT, [_P, _I64, _P, _P, _INT, _INT, _I64, _I64, _I64, _P, _P, _P, _P, _SIZE, _P]),
    "moe_b200_gated_ffn_workspace_bytes": (_SIZE, [_I64, _I64, _I64]),
    "moe_b200_gated_ffn_backward": (_INT, [_P, _I64, _P, _I64, _P, _P, _P, _P, _INT, _INT, _I64, _I64, _I64, _P, _P,
                                           _P, _P, _SIZE, _P]),
    "moe_b200_gated_ffn_backward_workspace_bytes": (_SIZE, [_I64, _I64, _I64]),
    "moe_b200_mxfp4_quantize": (_INT, [_P, _I64, _INT, _I64, _I64, _P, _P, _P]),
    "moe_b200_mxfp4_dequantize": (_INT, [_P, _P, _I64, _I64, _INT, _P, _P]),
    "moe_b200_mxfp4_matmul": (_INT, [_P, _P, _P, _P, _I64, _I64, _I64, _INT, _P, _P]),
    "moe_b200_mxfp4_linear": (_INT, [_P, _I64, _INT, _P, _P, _I64, _I64, _I64, _P, _P, _SIZE, _P]),
    "moe_b200_mxfp4_linear_workspace_bytes": (_SIZE, [_I64, _I64]),
    "moe_b200_mxfp4_gated_ffn": (_INT, [_P, _I64, _INT, _P, _P, _P, _P, _INT, _I64, _I64, _I64, _P, _P, _SIZE, _P]),
    "moe_b200_mxfp4_gated_ffn_workspace_bytes": (_SIZE, [_I64, _I64, _I64]),
    "moe_b200_mxfp4_scale_bytes": (_SIZE, [_I64, _I64]),
    "moe_b200_dense_read_status": (_INT, [ctypes.POINTER(ctypes.c_uint32), _P]),
    "moe_b200_dense_status_address": (_INT, [ctypes.POINTER(_P)]),
}
# Those the binding calls, in the order it takes them (torch_binding.cpp, Library).
_BINDING_CALLS = (
    "moe_b200_gated_ffn", "moe_b200_gated_ffn_workspace_bytes", "moe_b200_gated_ffn_backward",
    "moe_b200_gated_ffn_backward_workspace_bytes", "moe_b200_mxfp4_quantize", "moe_b200_mxfp4_dequantize",
    "moe_b200_mxfp4_matmul", "moe_b200_mxfp4_linear", "moe_b200_mxfp4_linear_workspace_bytes",
    "moe_b200_mxfp4_gated_ffn", "moe_b200_mxfp4_gated_ffn_workspace_bytes")

_library_bound = None
_native = None
_lock = threading.Lock()


def _library() -> ctypes.CDLL:
    """The library with the dense operators' signatures."""
    global _library_bound
    if _library_bound is None:
        lib = moe_host.load_library()
        for name, (restype, argtypes) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = restype, argtypes
        _library_bound = lib
    return _library_bound


def _load():
    """The native binding, built first when it is missing or stale."""
    global _native
    with _lock:
        if _native is None:
            lib = _library()
            path = moe_host._build_module().build_binding()
            loader = importlib.machinery.ExtensionFileLoader("_moe_b200_torch", path)
            module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_moe_b200_torch", loader))
            loader.exec_module(module)
            module.bind(*(ctypes.cast(getattr(lib, name), _P).value for name in _BINDING_CALLS))
            _native = module
    return _native


# ------------------------------------------------- what is wrong with a call
def _check_cuda(name: str, t, dev=None) -> None:
    _check(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    _check(t.is_cuda, f"{name} must be CUDA")
    _check(dev is None or t.device == dev, f"{name} must be on {dev}")


def _check_dim(name: str, d: int, multiple: int) -> None:
    _check(multiple <= d <= MAX_DIM and d % multiple == 0,
           f"{name} must be a multiple of {multiple} from {multiple} to {MAX_DIM}, got {d}")


def _check_rows(name: str, t: torch.Tensor, cols: int | None = None) -> None:
    """Rows that may lie apart, each contiguous and starting on 16 bytes."""
    _check(t.dim() == 2 and (cols is None or t.size(1) == cols),
           f"{name} must be [T, {cols if cols is not None else 'K'}]")
    _check(t.size(0) <= MAX_TOKENS, f"{name} has more than {MAX_TOKENS} rows")
    pitch = t.stride(0) if t.size(0) > 1 else t.size(1)
    _check((t.stride(1) == 1 or t.size(1) < 2) and pitch >= t.size(1),
           f"{name} must have contiguous rows that do not overlap")
    _check(t.size(0) == 0 or (t.data_ptr() % 16 == 0 and (t.size(0) == 1 or pitch * t.element_size() % 16 == 0)),
           f"{name}'s rows must start on 16 bytes")


def _check_dense(name: str, t, shape: tuple, dtype: torch.dtype, dev, align: int = 16) -> None:
    _check_cuda(name, t, dev)
    _check(tuple(t.shape) == shape and t.dtype == dtype and t.is_contiguous(),
           f"{name} must be a contiguous {dtype} tensor of shape {shape}")
    _check(t.data_ptr() % align == 0, f"{name} must be {align}-byte aligned")


def _span(t: torch.Tensor) -> tuple[int, int]:
    elements = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (elements * t.element_size() if t.numel() else 0)


def _check_no_tangents(*tensors: torch.Tensor) -> None:
    for t in tensors:
        _check(forward_ad.unpack_dual(t, level=0).tangent is None,
               "forward-mode derivatives are not computed: a tensor of the call has a tangent")


def _check_serves(x: torch.Tensor) -> None:
    """x carries no derivative that a 4-bit function would drop."""
    _check_no_tangents(x)
    _check(not (torch.is_grad_enabled() and x.requires_grad),
           "x requires gradients, which the 4-bit functions do not record: detach it, or call under torch.no_grad()")


def _check_output(output, shape: tuple, dtype: torch.dtype, dev, *inputs: torch.Tensor) -> None:
    if output is None:
        return
    _check_dense("output", output, shape, dtype, dev)
    _check(not (torch.is_grad_enabled() and output.requires_grad), "output must not require gradients")
    _check_no_tangents(output)
    begin, end = _span(output)
    for t in inputs:
        first, last = _span(t)
        _check(end <= first or last <= begin, "output must not overlap an input")


def _check_ffn(x, w13, w2) -> tuple[int, int, int]:
    """(T, H, I) of checked inputs."""
    _check_cuda("x", x)
    _check(x.dtype in (torch.bfloat16, torch.float16), "x must be bfloat16 or float16")
    _check_rows("x", x)
    T, H = x.shape
    _check_dim("the hidden size", H, 8)
    _check_cuda("w13", w13, x.device)
    _check(w13.dim() == 2 and w13.size(0) % 2 == 0 and w13.size(0) > 0, f"w13 must be [2 I, {H}]")
    inter = w13.size(0) // 2
    _check_dim("the intermediate size", inter, 8)
    _check_dense("w13", w13, (2 * inter, H), x.dtype, x.device)
    _check_dense("w2", w2, (H, inter), x.dtype, x.device)
    return T, H, inter


def _check_values(name: str, x) -> None:
    _check_cuda(name, x)
    _check(x.dtype in TYPES, f"{name} must be bfloat16, float16 or float32")
    _check_rows(name, x)
    _check_dim(f"{name}'s row length", x.size(1), 32)


def _check_mx(name: str, q, scale, dev=None, cols: int | None = None, rows: int | None = None) -> tuple[int, int]:
    """(rows, columns) of a checked 4-bit matrix."""
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


def _answer(name: str, got, explain):
    """What the binding returned, or the exception for it: None is a refused
    call, an integer the library's status."""
    if got is None:
        explain()
        raise RuntimeError(f"{name} refused its arguments")
    if isinstance(got, int):
        _raise_on(got, name)
    return got


def _activation(name: str) -> int:
    act = ACTIVATIONS.get(name)
    if act is None:
        raise RuntimeError(f"activation must be one of {sorted(ACTIVATIONS)}, got {name!r}")
    return act


def _type(dtype) -> int:
    code = TYPES.get(dtype)
    if code is None:
        raise RuntimeError("dtype must be bfloat16, float16 or float32")
    return code


# ------------------------------------------------- gated feed-forward block
class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, activation):
        output, (preact, hidden) = gated_ffn_forward(x, w13, w2, activation)
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
    got = (_native or _load()).gated_ffn(x, w13, w2, _activation(activation), output)
    if got is False:
        _check(output is None, "output cannot be given where gradients are recorded")
        return _GatedFFN.apply(x, w13, w2, activation)
    if isinstance(got, torch.Tensor):
        return got

    def explain():
        T, H, _ = _check_ffn(x, w13, w2)
        _check_no_tangents(x, w13, w2)
        _check_output(output, (T, H), x.dtype, x.device, x, w13, w2)

    return _answer("moe_b200_gated_ffn", got, explain)


def gated_ffn_forward(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, activation: str = "silu"):
    """gated_ffn for training without autograd: (output, saved), ``saved`` for
    gated_ffn_backward: u and g in fp32 [T, 2I], and h [T, I]."""
    got = (_native or _load()).gated_ffn_save(x, w13, w2, _activation(activation))
    if not isinstance(got, tuple):
        def explain():
            _check_ffn(x, w13, w2)
            _check_no_tangents(x, w13, w2)

        got = _answer("moe_b200_gated_ffn", got, explain)
    return got[0], got[1:]


def gated_ffn_backward(grad_output: torch.Tensor, x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, saved,
                       activation: str = "silu", needs=(True, True, True)):
    """(grad_x, grad_w13, grad_w2) for ``grad_output`` [T, H], in the inputs'
    type; None where ``needs`` is false. Bit for bit the same on every call.
    fp16 training wants a loss scale: act(g) and u act'(g) times the hidden's
    gradient are rounded to fp16, where values below 2^-14 lose bits
    (moe_b200_gated_ffn_backward)."""
    if not isinstance(saved, (tuple, list)) or len(saved) != 2:
        raise RuntimeError("saved must be the pair that gated_ffn_forward returned")
    if len(needs) != 3:
        raise RuntimeError("needs must be three truth values")
    got = (_native or _load()).gated_ffn_backward(grad_output, x, w13, w2, saved[0], saved[1],
                                                  _activation(activation), *needs)
    if isinstance(got, tuple):
        return got

    def explain():
        T, H, inter = _check_ffn(x, w13, w2)
        dev = x.device
        _check_cuda("grad_output", grad_output, dev)
        _check(grad_output.dtype == x.dtype and tuple(grad_output.shape) == (T, H),
               f"grad_output must be {x.dtype} [{T}, {H}] like the output")
        _check_rows("grad_output", grad_output, H)
        _check_dense("saved u and g", saved[0], (T, 2 * inter), torch.float32, dev, 32)
        _check_dense("saved hidden", saved[1], (T, inter), x.dtype, dev)
        _check_no_tangents(grad_output, x, w13, w2, *saved)

    return _answer("moe_b200_gated_ffn_backward", got, explain)


# ------------------------------------------------- 4-bit microscaled matrices
def mxfp4_scale_shape(rows: int, cols: int) -> tuple[int, ...]:
    """Shape of the exponent bytes of a 4-bit matrix [rows, cols]: the byte of
    row r, 32-column block b is at [r // 128, b // 4, r % 32, r % 128 // 32, b % 4]."""
    return (-(-rows // 128), -(-cols // 128), 32, 4, 4)


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [R, K] (bf16, fp16 or fp32; K a multiple of 32; rows may lie apart) in
    4 bits: codes uint8 [R, K / 2] and exponent bytes uint8 of
    mxfp4_scale_shape(R, K) (moe_b200_mxfp4_quantize). They are integers, through
    which no gradient passes: x may be a parameter."""
    got = (_native or _load()).mxfp4_quantize(x)
    if isinstance(got, tuple):
        return got
    return _answer("moe_b200_mxfp4_quantize", got, lambda: _check_values("x", x))


def mxfp4_dequantize(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The [R, K] values that a 4-bit matrix stands for, in ``dtype``."""
    got = (_native or _load()).mxfp4_dequantize(q, scale, _type(dtype))
    if isinstance(got, torch.Tensor):
        return got
    return _answer("moe_b200_mxfp4_dequantize", got, lambda: _check_mx("q", q, scale))


def mxfp4_matmul(a_q: torch.Tensor, a_scale: torch.Tensor, b_q: torch.Tensor, b_scale: torch.Tensor,
                 dtype: torch.dtype = torch.bfloat16, output: torch.Tensor | None = None) -> torch.Tensor:
    """A B^T of two 4-bit matrices [M, K] and [N, K]: fp32 sums, rounded once
    to ``dtype``."""
    got = (_native or _load()).mxfp4_matmul(a_q, a_scale, b_q, b_scale, _type(dtype), output)
    if isinstance(got, torch.Tensor):
        return got

    def explain():
        M, K = _check_mx("a_q", a_q, a_scale)
        N, _ = _check_mx("b_q", b_q, b_scale, a_q.device, K)
        _check(N > 0, "b_q must have rows")
        _check_output(output, (M, N), dtype, a_q.device, a_q, a_scale, b_q, b_scale)

    return _answer("moe_b200_mxfp4_matmul", got, explain)


def mxfp4_linear(x: torch.Tensor, w_q: torch.Tensor, w_scale: torch.Tensor,
                 output: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, K] times a 4-bit weight [N, K]: x is brought to 4 bits inside the
    call, the result [T, N] has x's type."""
    got = (_native or _load()).mxfp4_linear(x, w_q, w_scale, output)
    if isinstance(got, torch.Tensor):
        return got

    def explain():
        _check_values("x", x)
        N, _ = _check_mx("w_q", w_q, w_scale, x.device, x.size(1))
        _check(N > 0, "w_q must have rows")
        _check_serves(x)
        _check_output(output, (x.size(0), N), x.dtype, x.device, x, w_q, w_scale)

    return _answer("moe_b200_mxfp4_linear", got, explain)


def mxfp4_gated_ffn(x: torch.Tensor, w13_q: torch.Tensor, w13_scale: torch.Tensor, w2_q: torch.Tensor,
                    w2_scale: torch.Tensor, activation: str = "silu",
                    output: torch.Tensor | None = None) -> torch.Tensor:
    """The gated feed-forward block with 4-bit weights and activations, for
    serving: [u | g] = Q(x) w13^T, Q(act(g) * u) w2^T with Q the quantiser of
    mxfp4_quantize; the result [T, H] has x's type."""
    got = (_native or _load()).mxfp4_gated_ffn(x, w13_q, w13_scale, w2_q, w2_scale, _activation(activation), output)
    if isinstance(got, torch.Tensor):
        return got

    def explain():
        _check_values("x", x)
        T, H = x.shape
        two_i, _ = _check_mx("w13_q", w13_q, w13_scale, x.device, H)
        _check(two_i > 0 and two_i % 64 == 0, f"w13_q must have 2 I rows, I a multiple of 32; got {two_i}")
        _check_mx("w2_q", w2_q, w2_scale, x.device, two_i // 2, H)
        _check_serves(x)
        _check_output(output, (T, H), x.dtype, x.device, x, w13_q, w13_scale, w2_q, w2_scale)

    return _answer("moe_b200_mxfp4_gated_ffn", got, explain)


def read_status(device: torch.device | None = None) -> int:
    """Status word of the dense operators on ``device`` since the last read
    (0 = clean); synchronises the current stream and clears what it returns."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    st = ctypes.c_uint32(0)
    with torch.cuda.device(dev):
        code = _library().moe_b200_dense_read_status(ctypes.byref(st), torch.cuda.current_stream(dev).cuda_stream)
    if code not in (0, 7):
        _raise_on(code, "moe_b200_dense_read_status")
    return int(st.value)
