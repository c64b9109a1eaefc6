"""PyTorch front door: ``torch.ops.aster_b200.gemm_nt`` runs the CUDA GEMM on torch tensors.

The step above the operator surface in the reference is a linalg.matmul front end
(contrib/mlir-air/README.md); for a PyTorch user the equivalent is an operator that takes
CUDA tensors.  The tensors only lend their storage: the op passes ``data_ptr()`` and torch's
current stream to the C ABI (``b200_gemm_run``), there is no copy and no fallback to
``torch.matmul``.

    import aster_b200.torch_op            # registers the op
    c = torch.ops.aster_b200.gemm_nt(a, b, bias, relu=True, out_dtype=torch.bfloat16)
    c = aster_b200.torch_op.gemm_nt_direct(a, b, bias, relu=True)   # same, without the dispatcher

``a`` is ``[M, K]``, ``b`` is ``[N, K]`` (both contiguous, K fastest: ``c = a @ b.T``), dtype
float16, bfloat16 or float8_e4m3fn; ``bias`` is an optional float32 ``[N]``; ``scale_a`` /
``scale_b`` are optional one-element float32 CUDA tensors (per-tensor dequantisation scales).

Block-scaled fp4 (OCP MX: E2M1 elements, one power-of-two scale per 32 of them along K):

    q, s = torch.ops.aster_b200.quantize_mx(x)                # [M, K] -> codes [M, K/2], scales
    c = torch.ops.aster_b200.gemm_mx_nt(q, s, wq, ws, bias, relu=True, out_dtype=torch.bfloat16)
    x2 = torch.ops.aster_b200.dequantize_mx(q, s, torch.bfloat16)

The codes are uint8, two per byte (the lower K index in the low nibble); the scales are one flat
uint8 tensor in the order that the product streams them.  Weights are quantised once, activations
before each product.  Each of the three has a ``..._direct`` twin without the dispatcher's cost.
"""

from __future__ import annotations

import ctypes as C
import threading
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native as nat
from .gemm import GemmPlan

_DTYPES = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float8_e4m3fn: "e4m3"}
_OUT_DTYPES = {torch.float32: "f32", torch.bfloat16: "bf16"}

# (device, M, N, K, dtype_ab, dtype_c, epilogue) -> (plan, workspace tensor or None)
_plans: dict = {}


def _plan_for(device: torch.device, M: int, N: int, K: int, dtype_ab: str, dtype_c: str, epilogue: str):
    key = (device.index, M, N, K, dtype_ab, dtype_c, epilogue)
    hit = _plans.get(key)
    if hit is None:
        plan = GemmPlan(M, N, K, dtype_ab, dtype_c, epilogue=epilogue)
        res = plan.resources()
        ws_bytes = res.workspace_bytes or res.optional_workspace_bytes
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
        hit = _plans[key] = (plan, ws)
    return hit


_run_fn = None


def _gemm_run():
    global _run_fn
    if _run_fn is None:
        _run_fn = nat.lib().b200_gemm_run
    return _run_fn


_raw_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _raw_stream(device: torch.device) -> int:
    """Handle of torch's current stream on ``device`` (0 = the default stream)."""
    if _raw_stream_of is not None:
        return _raw_stream_of(device.index) or None
    return torch.cuda.current_stream(device).cuda_stream or None


_EPILOGUES = {(False, False): "none", (True, True): "bias_relu", (True, False): "bias", (False, True): "relu"}
_ready_devices: set = set()


def gemm_nt_direct(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, relu: bool = False,
                   out_dtype: torch.dtype = torch.float32, scale_a: Optional[torch.Tensor] = None,
                   scale_b: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The operator's implementation as a plain function: same checks and result as
    ``torch.ops.aster_b200.gemm_nt`` without the dispatcher's per-call cost (tens of
    microseconds for a Python custom op), for eager callers with small problems."""
    if not (a.is_cuda and b.is_cuda) or a.device != b.device:
        raise RuntimeError("aster_b200::gemm_nt needs both operands on the same CUDA device (there is no CPU path)")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        raise RuntimeError(f"expected a [M,K] and b [N,K], got {tuple(a.shape)} and {tuple(b.shape)}")
    if a.dtype != b.dtype or a.dtype not in _DTYPES or out_dtype not in _OUT_DTYPES:
        raise RuntimeError(f"unsupported dtypes {a.dtype}, {b.dtype} -> {out_dtype}")
    for name, t in (("bias", bias), ("scale_a", scale_a), ("scale_b", scale_b)):
        if t is not None and (t.dtype != torch.float32 or t.device != a.device):
            raise RuntimeError(f"{name} must be a float32 tensor on the operands' device")
    if not a.is_contiguous():
        a = a.contiguous()
    if not b.is_contiguous():
        b = b.contiguous()
    M, K = a.shape
    N = b.shape[0]
    if bias is not None and bias.numel() != N:
        raise RuntimeError(f"bias has {bias.numel()} elements, expected N={N}")
    device = a.device
    out = torch.empty((M, N), dtype=out_dtype, device=device)

    def launch() -> None:
        if device.index not in _ready_devices:
            nat.init_current()
            _ready_devices.add(device.index)
        plan, ws = _plan_for(device, M, N, K, _DTYPES[a.dtype], _OUT_DTYPES[out_dtype], _EPILOGUES[(bias is not None, relu)])
        # Straight to the entry point with plain integers (its argument types are declared, so
        # ctypes converts them): the wrapper objects of GemmPlan.run cost more host time than a
        # small problem's kernel runs for.
        nat.check(_gemm_run()(
            plan.handle, a.data_ptr(), b.data_ptr(), out.data_ptr(), None if bias is None else bias.contiguous().data_ptr(),
            None if scale_a is None else scale_a.data_ptr(), None if scale_b is None else scale_b.data_ptr(),
            None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), _raw_stream(device)))

    if torch.cuda.current_device() == device.index:  # the C ABI works on the current device, like torch
        launch()
    else:
        with torch.cuda.device(device):
            launch()
    return out


@torch.library.custom_op("aster_b200::gemm_nt", mutates_args=())
def gemm_nt(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, relu: bool = False,
            out_dtype: torch.dtype = torch.float32, scale_a: Optional[torch.Tensor] = None,
            scale_b: Optional[torch.Tensor] = None) -> torch.Tensor:
    return gemm_nt_direct(a, b, bias, relu, out_dtype, scale_a, scale_b)


@gemm_nt.register_fake
def _(a, b, bias=None, relu=False, out_dtype=torch.float32, scale_a=None, scale_b=None):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=out_dtype)


_MX_VALUE_DTYPES = {torch.float32: nat.F32, torch.bfloat16: nat.BF16, torch.float16: nat.F16}
# A block-scaled plan is told its scales before each launch: the two steps of a call belong together
# when several threads share a plan.
_mx_lock = threading.Lock()


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


_prepared_devices: set = set()


def _prepare(device: torch.device) -> None:
    """What the library asks of a device once: not possible while a stream is being captured."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the first call on a device sets the library up there: make it before the stream capture")
    nat.init_current()
    nat.call("b200_head_loss_status", (C.c_uint32 * 4)())  # kernel attributes, address of the status words
    _ready_devices.add(device.index)
    _prepared_devices.add(device.index)


def _call(device: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` with torch's current stream of ``device``, with ``device`` current (the C ABI
    works on the current device, like torch)."""
    if device.index in _prepared_devices and _current_device() == device.index:
        status = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            if device.index not in _prepared_devices:
                _prepare(device)
            status = fn(*args, _raw_stream(device))
    if status != nat.OK:
        nat.check(status)


def _mx_scales_bytes(rows: int, K: int) -> int:
    """What ``b200_mx_scales_bytes`` answers, without the call: 512 bytes per [128 rows][128 of K]."""
    return (rows + 127) // 128 * ((K + 127) // 128) * 512


def _check_mx_operand(name: str, q: torch.Tensor, scales: torch.Tensor) -> None:
    """Packed codes ``[rows, K/2]`` and their scales, in the layout that ``quantize_mx`` returns."""
    if q.is_cuda and q.dtype is torch.uint8 and scales.dtype is torch.uint8 and q.dim() == 2 and scales.dim() == 1 and scales.device == q.device:
        rows, half = q.shape
        if rows >= 1 and half >= 16 and half % 16 == 0 and scales.shape[0] == _mx_scales_bytes(rows, 2 * half):
            return
    for what, t in ((name, q), (f"{name}'s scales", scales)):
        if not t.is_cuda:
            raise RuntimeError(f"{what} must be a CUDA tensor (there is no CPU path)")
        if t.dtype != torch.uint8:
            raise RuntimeError(f"{what} must be uint8, got {t.dtype}")
    if q.dim() != 2 or q.shape[0] < 1 or q.shape[1] < 16 or q.shape[1] % 16:
        raise RuntimeError(f"{name} must be packed codes [rows, K/2] with K a positive multiple of 32, got {tuple(q.shape)}")
    want = _mx_scales_bytes(q.shape[0], 2 * q.shape[1])
    if scales.device != q.device or scales.dim() != 1 or scales.numel() != want:
        raise RuntimeError(f"{name}'s scales must be the {want} packed bytes on {q.device} that quantize_mx returns, got {tuple(scales.shape)} on {scales.device}")


def has_tangent(*tensors: torch.Tensor) -> bool:
    """Does one of them carry a forward-mode tangent?  (Outside of a dual level, where none can, asking each of
    them would cost 0.7 us.)"""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned (a view can start anywhere)."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def quantize_mx_direct(x: torch.Tensor, elem: str = "e2m1") -> tuple[torch.Tensor, torch.Tensor]:
    """``x`` ``[M, K]`` (float32, bfloat16 or float16; K a multiple of 32; rows may be strided) to
    block-scaled fp4: packed codes uint8 ``[M, K/2]`` and the packed scales.  A block of 32 that holds
    a NaN or an infinity reads as 32 NaN afterwards."""
    if torch.compiler.is_compiling():  # a compiler sees the operator, not what is behind it
        return torch.ops.aster_b200.quantize_mx(x, elem)
    return _quantize(x, elem)


def _quantize(x: torch.Tensor, elem: str) -> tuple[torch.Tensor, torch.Tensor]:
    if elem != "e2m1":
        raise RuntimeError(f"quantize_mx makes e2m1 elements, not {elem!r}")
    if not x.is_cuda:
        raise RuntimeError("aster_b200::quantize_mx needs a CUDA tensor (there is no CPU path)")
    if x.dim() != 2 or x.shape[0] < 1 or x.shape[1] < 32 or x.shape[1] % 32:
        raise RuntimeError(f"expected x [M, K] with M >= 1 and K a positive multiple of 32, got {tuple(x.shape)}")
    if x.dtype not in _MX_VALUE_DTYPES:
        raise RuntimeError(f"unsupported dtype {x.dtype}")
    M, K = x.shape
    if x.stride(1) != 1 or (M > 1 and x.stride(0) < K):
        x = x.contiguous()
    q = x.new_empty((M, K // 2), dtype=torch.uint8)
    scales = x.new_empty(_mx_scales_bytes(M, K), dtype=torch.uint8)
    _call(x.device, nat.lib().b200_quantize_mx, x.data_ptr(), _MX_VALUE_DTYPES[x.dtype], M, K, x.stride(0), nat.MXE2M1, q.data_ptr(), scales.data_ptr())
    return q, scales


def dequantize_mx_direct(q: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values ``[M, K]`` that packed codes and scales stand for (exact in float32 and bfloat16)."""
    if torch.compiler.is_compiling():
        return torch.ops.aster_b200.dequantize_mx(q, scales, out_dtype)
    return _dequantize(q, scales, out_dtype)


def _dequantize(q: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    _check_mx_operand("q", q, scales)
    if out_dtype not in _MX_VALUE_DTYPES:
        raise RuntimeError(f"unsupported out_dtype {out_dtype}")
    q, scales = _aligned(q), _aligned(scales)
    M, K = q.shape[0], 2 * q.shape[1]
    out = q.new_empty((M, K), dtype=out_dtype)
    _call(q.device, nat.lib().b200_dequantize_mx, q.data_ptr(), scales.data_ptr(), nat.MXE2M1, M, K, _MX_VALUE_DTYPES[out_dtype], out.data_ptr())
    return out


class _NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, bias, made):
        return made.pop()  # not an input: the result is no view of one and may be changed in place

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("aster_b200::gemm_mx_nt has no backward pass: its bias gets no gradient")


def _without_gradient(out: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """``out`` as part of ``bias``'s graph: a backward pass that reaches it is refused, as the dispatcher's form
    does, where a result without a graph would leave the bias out of it silently."""
    return _NoGradient.apply(bias, [out])


def gemm_mx_nt_direct(a: torch.Tensor, scales_a: torch.Tensor, b: torch.Tensor, scales_b: torch.Tensor, bias: Optional[torch.Tensor] = None,
                      relu: bool = False, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``epilogue(A . B^T)`` of two block-scaled fp4 operands as :func:`quantize_mx_direct` returns
    them: ``a`` ``[M, K/2]``, ``b`` ``[N, K/2]``, optional float32 ``bias`` ``[N]`` and ReLU, fp32
    accumulation, ``[M, N]`` out.  There is no backward pass: one that reaches the bias is refused.  The first
    call of a shape allocates (its plan lives until :func:`clear_plan_cache`): inside a stream capture it is refused."""
    if torch.compiler.is_compiling():
        return torch.ops.aster_b200.gemm_mx_nt(a, scales_a, b, scales_b, bias, relu, out_dtype)
    return _product(a, scales_a, b, scales_b, bias, relu, out_dtype)


def _product(a, scales_a, b, scales_b, bias, relu: bool, out_dtype: torch.dtype) -> torch.Tensor:
    _check_mx_operand("a", a, scales_a)
    _check_mx_operand("b", b, scales_b)
    if a.device != b.device or a.shape[1] != b.shape[1]:
        raise RuntimeError(f"expected a [M, K/2] and b [N, K/2] on one device, got {tuple(a.shape)} on {a.device} and {tuple(b.shape)} on {b.device}")
    if out_dtype not in _OUT_DTYPES:
        raise RuntimeError(f"unsupported out_dtype {out_dtype}")
    M, N, K = a.shape[0], b.shape[0], 2 * a.shape[1]
    if bias is not None and (bias.dtype != torch.float32 or bias.device != a.device or bias.numel() != N):
        raise RuntimeError(f"bias must be {N} float32 values on {a.device}")
    if bias is not None and has_tangent(bias):
        raise RuntimeError("aster_b200::gemm_mx_nt has no forward-mode derivative: bias must not carry a tangent")
    a, scales_a, b, scales_b = _aligned(a), _aligned(scales_a), _aligned(b), _aligned(scales_b)
    bias = None if bias is None else bias.contiguous()
    out = a.new_empty((M, N), dtype=out_dtype)
    _call(a.device, _gemm_mx, a, scales_a, b, scales_b, bias, relu, out)
    return _without_gradient(out, bias) if bias is not None and bias.requires_grad and torch.is_grad_enabled() else out


def _gemm_mx(a, scales_a, b, scales_b, bias, relu, out, stream) -> int:
    M, N = out.shape
    K = 2 * a.shape[1]
    lib = nat.lib()
    with _mx_lock:
        key = (a.device.index, M, N, K, "mxe2m1", _OUT_DTYPES[out.dtype], _EPILOGUES[(bias is not None, relu)])
        hit = _plans.get(key)
        if hit is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"the first product of a shape ({M} x {N} x {K}) allocates: make it before the stream capture")
            hit = _plans[key] = (GemmPlan(*key[1:6], epilogue=key[6]), None)
        handle = hit[0].handle
        status = lib.b200_gemm_plan_set_mx_scales(handle, scales_a.data_ptr(), scales_b.data_ptr())
        if status == nat.OK:
            status = lib.b200_gemm_run(handle, a.data_ptr(), b.data_ptr(), out.data_ptr(), None if bias is None else bias.data_ptr(), None, None, None, 0, stream)
    return status


@torch.library.custom_op("aster_b200::quantize_mx", mutates_args=())
def quantize_mx(x: torch.Tensor, elem: str = "e2m1") -> tuple[torch.Tensor, torch.Tensor]:
    return _quantize(x, elem)


@quantize_mx.register_fake
def _(x, elem="e2m1"):
    M, K = x.shape
    return x.new_empty((M, K // 2), dtype=torch.uint8), x.new_empty((_mx_scales_bytes(M, K),), dtype=torch.uint8)


@torch.library.custom_op("aster_b200::dequantize_mx", mutates_args=())
def dequantize_mx(q: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return _dequantize(q, scales, out_dtype)


@dequantize_mx.register_fake
def _(q, scales, out_dtype=torch.float32):
    return q.new_empty((q.shape[0], 2 * q.shape[1]), dtype=out_dtype)


@torch.library.custom_op("aster_b200::gemm_mx_nt", mutates_args=())
def gemm_mx_nt(a: torch.Tensor, scales_a: torch.Tensor, b: torch.Tensor, scales_b: torch.Tensor, bias: Optional[torch.Tensor] = None,
               relu: bool = False, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return _product(a, scales_a, b, scales_b, bias, relu, out_dtype)


@gemm_mx_nt.register_fake
def _(a, scales_a, b, scales_b, bias=None, relu=False, out_dtype=torch.float32):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=out_dtype)


def clear_plan_cache() -> None:
    """Destroy the plans of all shapes seen so far; not while a captured graph that holds one of their
    products may still be replayed (a launch reports into its plan's status words)."""
    for plan, _ in _plans.values():
        plan.destroy()
    _plans.clear()
