"""Losses of a language model's head on torch tensors, without the logits.

The head's product ``z = x . w^T`` (``x`` ``[tokens, hidden]``, ``w`` ``[vocab, hidden]``, the ``gemm_nt``
layout) is consumed tile by tile where the tensor cores leave it: the forward pass keeps a maximum and
a sum per row, the backward pass computes z again, a range of the vocabulary at a time, and turns it into
both gradients.  Nothing of size ``tokens x vocab`` is ever stored but that range of ``dL/dz`` in 16 bits.

    from aster_b200.head_loss import linear_cross_entropy, linear_distillation

    loss = linear_cross_entropy(x, w, target, label_smoothing=0.1)     # differentiable in x and w
    loss = linear_distillation(x, w, teacher_logits, teacher_ids, temperature=2.0)

``torch.ops.aster_b200.linear_cross_entropy`` / ``linear_distillation`` are the same as operators of the
dispatcher (they return ``(loss, lse, saved)``; ``loss`` is differentiable), which is what a compiler is
shown of the functions.  The tensors only lend their storage to ``b200_head_loss_*``; torch's current stream
is used, there is no CPU path and no fallback.

Precision.  Products, softmax sums and losses are fp32, but not every step rounds as a plain fp32 program's:

* the tensor core's accumulator truncates: logits come out up to (hidden / 16 + 1) * 2^-23 * |x| . |w| off
  (9e-6 rms at hidden = 4096, losses 1.5e-6 relative), and exponentials are the hardware's (2 ulp, 0 below 2^-126);
* ``dL/dz`` is rounded once to the operands' 16 bits before both gradient products, after division by the
  largest row factor: with one label per row the gradients are as near as their own rounding, with a teacher's
  many entries about 1.4 times as far (bf16 0.0024 against 0.0017).  With "none" in float16 a row whose factor
  is below 1e-8 of the largest loses digits of its gradient, below 3e-12 all of them;
* the gradients are products: an ignored row of ``x`` that holds NaN or infinity reaches ``dL/dw`` (0 * NaN),
  and one of ``w`` reaches ``dL/dx``, as in the plain program.

Only the first derivative in reverse mode exists; tangents (``torch.autograd.forward_ad``) are refused.  A stream
capture with gradients is refused while a graph of the same leaves that was made here on the default stream is
alive; a forward pass alone is recorded under ``torch.no_grad()``.
"""

from __future__ import annotations

import ctypes as C
import functools
import weakref
from typing import Optional, Sequence

import torch

from . import _native as nat
from .torch_op import _call, _raw_stream, has_tangent

_DTYPES = {torch.bfloat16: nat.BF16, torch.float16: nat.F16}
_TEACHER_DTYPES = {torch.float32: nat.F32, torch.bfloat16: nat.BF16, torch.float16: nat.F16}
_INDEX_BITS = {torch.int64: 64, torch.int32: 32}
_REDUCTIONS = {"none": nat.REDUCE_NONE, "mean": nat.REDUCE_MEAN, "sum": nat.REDUCE_SUM}
MAX_TOP = 1024  # teacher entries per row


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Two dimensions, the last one contiguous, rows a multiple of 16 bytes apart and aligned (else a copy)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    if t.stride(1) != 1 or (t.shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) < t.shape[1])):
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _check(name: str, x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, reduction: str) -> None:
    if has_tangent(x, w):
        raise RuntimeError(f"aster_b200::{name} has no forward-mode derivative: x and weight must not carry a tangent")
    for what, t in (("x", x), ("weight", w), ("labels", labels)):
        if not t.is_cuda:
            raise RuntimeError(f"aster_b200::{name} needs CUDA tensors, {what} is on {t.device} (there is no CPU path)")
        if t.device != x.device:
            raise RuntimeError(f"{what} is on {t.device}, x on {x.device}")
    if x.dtype not in _DTYPES or w.dtype != x.dtype:
        raise RuntimeError(f"unsupported dtypes {x.dtype}, {w.dtype}: both bfloat16 or both float16")
    if x.dim() < 2 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise RuntimeError(f"expected x [..., hidden] and weight [vocab, hidden], got {tuple(x.shape)} and {tuple(w.shape)}")
    if w.shape[0] < 1 or w.shape[1] < 8 or w.shape[1] % 8:
        raise RuntimeError(f"weight {tuple(w.shape)}: vocab must be at least 1 and hidden a positive multiple of 8")
    if labels.dtype not in _INDEX_BITS:
        raise RuntimeError(f"labels must be int64 or int32, got {labels.dtype}")
    if reduction not in _REDUCTIONS:
        raise RuntimeError(f"unknown reduction {reduction!r}")


def _desc(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, reduction: str) -> nat.HeadDesc:
    d = nat.HeadDesc()
    d.tokens, d.hidden = x.shape
    d.vocab = w.shape[0]
    d.x_stride = x.stride(0) if d.tokens > 1 else d.hidden
    d.w_stride = w.stride(0) if d.vocab > 1 else d.hidden
    d.dtype, d.reduction, d.index_bits = _DTYPES[x.dtype], _REDUCTIONS[reduction], _INDEX_BITS[labels.dtype]
    return d


def _sizes(d: nat.HeadDesc) -> nat.HeadSizes:
    s = nat.HeadSizes()
    nat.call("b200_head_loss_sizes", C.byref(d), C.byref(s))
    return s


@functools.lru_cache(maxsize=256)
def _sizes_of(fields: bytes) -> nat.HeadSizes:
    """The sizes follow from the description alone."""
    return _sizes(nat.HeadDesc.from_buffer_copy(fields))


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _saw(*tensors: torch.Tensor) -> list:
    """What the tensors of a pass have to have in common with those of the other one."""
    return [(t.shape, t.dtype, t.device) for t in tensors]


class _Head:
    """One call's tensors as the C ABI wants them, and its description."""

    def __init__(self, x, w, labels, reduction, *, kind, ignore_index=0, label_smoothing=0.0, temperature=1.0, teacher=None, grad_bytes=0):
        self.x, self.w, self.labels, self.teacher = _rows(x), _rows(w), labels.contiguous(), teacher
        self.device, self.saw = x.device, _saw(self.x, self.w, self.labels)
        self.desc = d = _desc(self.x, self.w, labels, reduction)
        d.kind, d.ignore_index, d.label_smoothing, d.temperature = kind, ignore_index, label_smoothing, temperature
        d.grad_bytes = grad_bytes
        if kind == nat.HEAD_DISTILL:
            d.top, d.dtype_teacher = labels.shape[-1], nat.F32 if teacher is None else _TEACHER_DTYPES[teacher.dtype]
        self.per_row = reduction == "none"

    def without_tensors(self) -> "_Head":
        """The description alone, for the time until the backward pass brings the tensors again."""
        h = _Head.__new__(_Head)
        h.desc, h.per_row, h.device, h.saw = self.desc, self.per_row, self.device, self.saw
        return h

    def with_tensors(self, x, w, labels) -> "_Head":
        """The description with the forward pass's tensors, as they come back from autograd.  Hooks on saved
        tensors may have laid them out anew (an offloaded slice returns contiguous): the strides are theirs."""
        h = self.without_tensors()  # its own object: a graph may be walked from several threads
        h.x, h.w, h.labels, h.teacher = _rows(x), _rows(w), labels.contiguous(), None
        x, w, labels = h.x, h.w, h.labels
        d = self.desc
        saw = _saw(x, w, labels)
        if saw != self.saw:
            raise RuntimeError(f"the saved tensors came back as {saw}; the forward pass had {self.saw}")
        x_stride, w_stride = x.stride(0) if d.tokens > 1 else d.hidden, w.stride(0) if d.vocab > 1 else d.hidden
        if x_stride != d.x_stride or w_stride != d.w_stride:
            h.desc = nat.HeadDesc.from_buffer_copy(d)
            h.desc.x_stride, h.desc.w_stride = x_stride, w_stride
        return h

    def forward(self):
        dev, tokens = self.x.device, self.x.shape[0]
        if tokens == 0:  # nothing to launch
            none = self.x.new_empty(0, dtype=torch.float32)
            loss = none if self.per_row else self.x.new_full((), float("nan") if self.desc.reduction == nat.REDUCE_MEAN else 0.0, dtype=torch.float32)
            return loss, none.clone(), self.x.new_empty(0, dtype=torch.uint8)
        sizes = _sizes_of(bytes(self.desc))
        loss = self.x.new_empty(tokens if self.per_row else (), dtype=torch.float32)
        lse = self.x.new_empty(tokens, dtype=torch.float32)
        saved = self.x.new_empty(sizes.saved, dtype=torch.uint8)
        ws = self.x.new_empty(sizes.forward_workspace, dtype=torch.uint8)
        _call(dev, nat.lib().b200_head_loss_forward, C.byref(self.desc), self.x.data_ptr(), self.w.data_ptr(), self.labels.data_ptr(), _ptr(self.teacher),
              loss.data_ptr(), lse.data_ptr(), saved.data_ptr(), ws.data_ptr(), sizes.forward_workspace)
        return loss, lse, saved

    def backward(self, grad, lse, saved, want_x: bool, want_w: bool):
        dev, tokens = self.x.device, self.x.shape[0]
        dx = torch.empty(self.x.shape, dtype=self.x.dtype, device=dev) if want_x else None
        if tokens == 0:
            return dx, torch.zeros(self.w.shape, dtype=self.w.dtype, device=dev) if want_w else None
        dw = torch.empty(self.w.shape, dtype=self.w.dtype, device=dev) if want_w else None
        if grad.dtype != torch.float32 or not grad.is_contiguous():
            grad = grad.to(torch.float32).contiguous()
        sizes = _sizes_of(bytes(self.desc))
        need = sizes.backward_workspace
        for what, t, dtype, n in (("grad", grad, torch.float32, tokens if self.per_row else 1), ("lse", lse, torch.float32, tokens), ("saved", saved, torch.uint8, sizes.saved)):
            if t.dtype != dtype or t.device != dev or t.numel() != n or not t.is_contiguous():
                raise RuntimeError(f"{what} must be {n} contiguous {dtype} on {dev}, got {tuple(t.shape)} {t.dtype} on {t.device}")
        ws = self.x.new_empty(need, dtype=torch.uint8)
        _call(dev, nat.lib().b200_head_loss_backward, C.byref(self.desc), self.x.data_ptr(), self.w.data_ptr(), self.labels.data_ptr(), lse.data_ptr(),
              saved.data_ptr(), grad.data_ptr(), _ptr(dx), _ptr(dw), ws.data_ptr(), need)
        return dx, dw


def _xent_head(x, w, target, ignore_index, label_smoothing, reduction, grad_bytes=0) -> _Head:
    _check("linear_cross_entropy", x, w, target, reduction)
    if target.shape != x.shape[:-1]:
        raise RuntimeError(f"target {tuple(target.shape)} does not match x {tuple(x.shape)}")
    if not 0.0 <= label_smoothing < 1.0:
        raise RuntimeError(f"label_smoothing={label_smoothing} is outside [0, 1)")
    return _Head(x, w, target, reduction, kind=nat.HEAD_CROSS_ENTROPY, ignore_index=ignore_index, label_smoothing=label_smoothing, grad_bytes=grad_bytes)


def _distill_head(x, w, teacher_logits, teacher_ids, temperature, reduction, grad_bytes=0) -> _Head:
    _check("linear_distillation", x, w, teacher_ids, reduction)
    if teacher_ids.dim() != x.dim() or teacher_ids.shape[:-1] != x.shape[:-1] or not 1 <= teacher_ids.shape[-1] <= MAX_TOP:
        raise RuntimeError(f"teacher_ids {tuple(teacher_ids.shape)} do not match x {tuple(x.shape)} with 1 to {MAX_TOP} entries per row")
    if teacher_logits is not None:
        if teacher_logits.shape != teacher_ids.shape or teacher_logits.device != x.device:
            raise RuntimeError(f"teacher_logits {tuple(teacher_logits.shape)} on {teacher_logits.device} do not match teacher_ids {tuple(teacher_ids.shape)} on {x.device}")
        if teacher_logits.dtype not in _TEACHER_DTYPES:
            raise RuntimeError(f"unsupported teacher_logits dtype {teacher_logits.dtype}")
        teacher_logits = teacher_logits.detach().contiguous()
    if not 2.0 ** -60 <= temperature <= 2.0 ** 60:  # 1 / T and T^2 are fp32 numbers in full
        raise RuntimeError(f"temperature={temperature} is outside [2^-60, 2^60]")
    return _Head(x, w, teacher_ids, reduction, kind=nat.HEAD_DISTILL, temperature=temperature, teacher=teacher_logits, grad_bytes=grad_bytes)


# Graphs of these functions and operators that were made on a default stream, each with its leaves, for as long as they live.
# Autograd keeps one accumulation node per leaf, tied to the stream that was current when it was made, while any
# graph refers to it.  A backward pass that is being captured cannot join the default stream, so a graph left
# over from there would break the capture (and, from the engine's own threads, the process): such a capture is
# refused before it begins.
_default_stream_graphs: dict = {}


def _refuse_capture_beside(*tensors: torch.Tensor) -> None:
    for leaves, _ in list(_default_stream_graphs.values()):
        if any(ref() is t for ref in leaves for t in tensors):
            raise RuntimeError("an autograd graph of the same leaf, made on the default stream, is still alive: a backward pass cannot be captured "
                               "beside it; free that graph (delete its loss) before the capture")


def _note_graph(ctx, x: torch.Tensor, w: torch.Tensor) -> None:
    leaves = tuple(weakref.ref(t) for t in (x, w) if t.requires_grad and t.is_leaf)
    if leaves:
        key = id(ctx)
        _default_stream_graphs[key] = (leaves, weakref.ref(ctx, lambda _: _default_stream_graphs.pop(key, None)))


def _capturing(device: torch.device) -> bool:
    with torch.cuda.device(device):  # of the tensors, which need not be the current one
        return torch.cuda.is_current_stream_capturing()


def _watch_graph(ctx, x: torch.Tensor, w: torch.Tensor) -> None:
    if not _raw_stream(x.device):
        _note_graph(ctx, x, w)
    elif _capturing(x.device):
        _refuse_capture_beside(x, w)


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, head, shape):
        _watch_graph(ctx, x, w)
        loss, lse, saved = head.forward()
        # the tensors come back through save_for_backward: it notices a change in place before the backward pass
        ctx.save_for_backward(x, w, head.labels, lse, saved)
        ctx.head, ctx.shape = head.without_tensors(), x.shape
        return loss.view(shape) if head.per_row else loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, w, labels, lse, saved = ctx.saved_tensors
        dx, dw = ctx.head.with_tensors(x, w, labels).backward(grad, lse, saved, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx if dx is None or dx.dim() == len(ctx.shape) else dx.view(ctx.shape), dw, None, None


def _apply(x: torch.Tensor, w: torch.Tensor, head: _Head, shape) -> torch.Tensor:
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _HeadLoss.apply(x, w, head, shape)
    loss = head.forward()[0]  # nothing to differentiate: no graph
    return loss.view(shape) if head.per_row else loss


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100, label_smoothing: float = 0.0,
                         reduction: str = "mean", grad_bytes: int = 0) -> torch.Tensor:
    """Softmax cross entropy of ``x . weight^T`` against ``target``, as
    ``torch.nn.functional.cross_entropy`` defines it, in fp32, differentiable in ``x`` and ``weight``.

    ``x`` ``[..., hidden]`` and ``weight`` ``[vocab, hidden]`` are both bfloat16 or both float16 (hidden a
    multiple of 8), ``target`` ``[...]`` int64 or int32.  Targets equal to ``ignore_index`` have no loss and
    no gradient; any other target outside the vocabulary makes its loss, and the gradients it enters, NaN.
    "mean" divides by the number of targets that count (NaN without any).  The backward pass keeps at most
    ``max(grad_bytes, 512 * tokens)`` bytes of ``dL/dz`` at a time (``grad_bytes`` 0: 256 MiB); where it works in
    several ranges of the vocabulary or cuts a long axis, fp32 parts of the gradients come on top, up to
    ``32 * 4 * tokens * hidden`` bytes for ``x``'s and 256 MiB for ``w``'s.  The module says what is rounded where."""
    if torch.compiler.is_compiling():  # a compiler sees the operator, not what is behind it
        return torch.ops.aster_b200.linear_cross_entropy(x, weight, target, ignore_index, label_smoothing, reduction, grad_bytes)[0]
    return _apply(x, weight, _xent_head(x, weight, target, ignore_index, label_smoothing, reduction, grad_bytes), target.shape)


def linear_distillation(x: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, *, temperature: float = 1.0,
                        reduction: str = "mean", grad_bytes: int = 0) -> torch.Tensor:
    """Distillation of the head ``x . weight^T`` from a teacher's top logits: per row
    ``T^2 * KL(softmax(teacher_logits / T) || softmax(x . weight^T / T))`` with the teacher's distribution over
    its ``teacher_ids`` alone, in fp32, differentiable in ``x`` and ``weight`` (not in the teacher).

    ``teacher_logits`` (float32, bfloat16 or float16) and ``teacher_ids`` (int64 or int32) are ``[..., top]``, in any
    order, ``top`` at most 1024.  Entries with a negative id or a logit of minus infinity are left out; rows with
    nothing left have no loss and no gradient and do not count for "mean".  An id listed twice counts twice; an
    id beyond the vocabulary, or a logit that is NaN or plus infinity, makes the row NaN.  ``temperature`` is within
    2^-60 .. 2^60; ``grad_bytes`` and rounding as for :func:`linear_cross_entropy`."""
    if torch.compiler.is_compiling():
        return torch.ops.aster_b200.linear_distillation(x, weight, teacher_logits, teacher_ids, temperature, reduction, grad_bytes)[0]
    return _apply(x, weight, _distill_head(x, weight, teacher_logits, teacher_ids, temperature, reduction, grad_bytes), teacher_ids.shape[:-1])


def head_loss_status() -> Sequence[int]:
    """Status words of the calls made so far on the current device (synchronises it); raises
    ``B200Error`` (TIMEOUT) if a bounded device-side wait gave up.  From then until this call, losses
    and gradients on that device are NaN."""
    words = (C.c_uint32 * 4)()
    nat.call("b200_head_loss_status", words)
    return list(words)


# ---- operators of the dispatcher ----
def _fake_outputs(x, reduction, rows_shape, saved):
    loss = x.new_empty(rows_shape if reduction == "none" else (), dtype=torch.float32)
    return loss, x.new_empty((x.numel() // x.shape[-1],), dtype=torch.float32), x.new_empty((saved,), dtype=torch.uint8)


def _align256(n: int) -> int:
    return (n + 255) // 256 * 256


def _wanted(x, weight, dx, dw, want_x: bool, want_w: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """Both gradients of an operator, which cannot return None: an unwanted one is empty."""
    return dx.view(x.shape) if want_x else x.new_empty(0), dw if want_w else weight.new_empty(0)


def _fake_wanted(x, weight, want_x: bool, want_w: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return x.new_empty(x.shape if want_x else 0), weight.new_empty(weight.shape if want_w else 0)


@torch.library.custom_op("aster_b200::linear_cross_entropy", mutates_args=())
def _xent_op(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100, label_smoothing: float = 0.0,
             reduction: str = "mean", grad_bytes: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    head = _xent_head(x, weight, target, ignore_index, label_smoothing, reduction, grad_bytes)
    loss, lse, saved = head.forward()
    return loss.view(target.shape) if head.per_row else loss, lse, saved


@_xent_op.register_fake
def _(x, weight, target, ignore_index=-100, label_smoothing=0.0, reduction="mean", grad_bytes=0):
    return _fake_outputs(x, reduction, target.shape, 256 if x.numel() else 0)


@torch.library.custom_op("aster_b200::linear_cross_entropy_backward", mutates_args=())
def _xent_backward_op(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, lse: torch.Tensor, saved: torch.Tensor,
                      ignore_index: int, label_smoothing: float, reduction: str, want_x: bool = True, want_w: bool = True,
                      grad_bytes: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    dx, dw = _xent_head(x, weight, target, ignore_index, label_smoothing, reduction, grad_bytes).backward(grad, lse, saved, want_x, want_w)
    return _wanted(x, weight, dx, dw, want_x, want_w)


@_xent_backward_op.register_fake
def _(grad, x, weight, target, lse, saved, ignore_index, label_smoothing, reduction, want_x=True, want_w=True, grad_bytes=0):
    return _fake_wanted(x, weight, want_x, want_w)


def _watch_operator(ctx, x: torch.Tensor, w: torch.Tensor) -> None:
    if x.is_cuda and all(type(t) in (torch.Tensor, torch.nn.Parameter) for t in (x, w)):  # not while a compiler traces
        _watch_graph(ctx, x, w)


def _xent_setup(ctx, inputs, output):
    x, weight, target, *ctx.options, ctx.grad_bytes = inputs
    _watch_operator(ctx, x, weight)
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.save_for_backward(x, weight, target, output[1], output[2])


def _xent_autograd(ctx, grad, _lse, _saved):
    want_x, want_w = ctx.needs_input_grad[:2]
    dx, dw = torch.ops.aster_b200.linear_cross_entropy_backward(grad, *ctx.saved_tensors, *ctx.options, want_x, want_w, ctx.grad_bytes)
    return dx if want_x else None, dw if want_w else None, None, None, None, None, None


_xent_op.register_autograd(_xent_autograd, setup_context=_xent_setup)


@torch.library.custom_op("aster_b200::linear_distillation", mutates_args=())
def _distill_op(x: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, temperature: float = 1.0,
                reduction: str = "mean", grad_bytes: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    head = _distill_head(x, weight, teacher_logits, teacher_ids, temperature, reduction, grad_bytes)
    loss, lse, saved = head.forward()
    return loss.view(teacher_ids.shape[:-1]) if head.per_row else loss, lse, saved


@_distill_op.register_fake
def _(x, weight, teacher_logits, teacher_ids, temperature=1.0, reduction="mean", grad_bytes=0):
    rows, top = x.numel() // x.shape[-1], teacher_ids.shape[-1]
    return _fake_outputs(x, reduction, teacher_ids.shape[:-1], 256 + _align256(4 * rows) + 2 * _align256(4 * rows * top) if rows else 0)


@torch.library.custom_op("aster_b200::linear_distillation_backward", mutates_args=())
def _distill_backward_op(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, lse: torch.Tensor, saved: torch.Tensor,
                         temperature: float, reduction: str, want_x: bool = True, want_w: bool = True, grad_bytes: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    dx, dw = _distill_head(x, weight, None, teacher_ids, temperature, reduction, grad_bytes).backward(grad, lse, saved, want_x, want_w)
    return _wanted(x, weight, dx, dw, want_x, want_w)


@_distill_backward_op.register_fake
def _(grad, x, weight, teacher_ids, lse, saved, temperature, reduction, want_x=True, want_w=True, grad_bytes=0):
    return _fake_wanted(x, weight, want_x, want_w)


def _distill_setup(ctx, inputs, output):
    x, weight, _, teacher_ids, *ctx.options, ctx.grad_bytes = inputs
    _watch_operator(ctx, x, weight)
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.save_for_backward(x, weight, teacher_ids, output[1], output[2])


def _distill_autograd(ctx, grad, _lse, _saved):
    want_x, want_w = ctx.needs_input_grad[:2]
    dx, dw = torch.ops.aster_b200.linear_distillation_backward(grad, *ctx.saved_tensors, *ctx.options, want_x, want_w, ctx.grad_bytes)
    return dx if want_x else None, dw if want_w else None, None, None, None, None, None


_distill_op.register_autograd(_distill_autograd, setup_context=_distill_setup)
