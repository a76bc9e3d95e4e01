"""Losses over a large vocabulary at the output layer of a language model, on the padded batches that the other
operators take: cross entropy with token ids, and distillation from a teacher's top logits.

``hidden @ weight.T`` are the logits, which are never kept: the kernels go over the vocabulary in pieces.  Shapes:
``hidden`` ``[N, D]`` or ``[B, L, D]``, ``weight`` ``[V, D]``, both bfloat16 or both float16; ``targets`` and ``valid``
like ``hidden`` without its last dimension, ``teacher_ids`` and ``teacher_logits`` with the teacher's ``K`` entries as
their last.  Any strides, but for the last dimension of ``hidden``, ``weight`` and the teacher's tensors, which is contiguous, so
``hidden[:, :-1]`` with ``tokens[:, 1:]`` and ``valid[:, 1:]`` is the next-token loss of a batch.

A row counts unless ``valid`` is 0 there or its target is negative (the padding of the batches); with a teacher, unless it has
no entry with an id of 0 or more and a logit above ``-inf``.  Rows that do not count have a loss and a gradient of 0, and
what ``hidden`` holds there is not looked at.  ``reduction="mean"`` divides by the rows that count (0 if none does).  Nothing is read back, so
an id of ``V`` or more cannot raise: it makes the loss NaN, as a NaN among the inputs or a logit of
``+inf`` does; a target's logit of ``-inf`` makes it ``+inf``.  Results are the same at every call with the same
inputs; sums are held in 32 bits, those of the losses of rows in 64."""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib as L

_REAL = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_WANT_LOSS, _WANT_GRADS = 1, 2
MAX_TEACHER_ENTRIES = 256
MIN_TEMPERATURE, MAX_TEMPERATURE = 2.0 ** -16, 2.0 ** 16


def _raise(status: int, msg: str) -> None:
    if status == L.E_BADARG:
        raise ValueError(msg)
    raise RuntimeError(msg)


def _rows(t: torch.Tensor, lead: int) -> Tuple[int, int]:
    """Strides of the (outer, inner) row dimensions."""
    return (t.stride(0), t.stride(1)) if lead == 2 else (0, t.stride(0))


def _refuse_tangents(*tensors) -> None:
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the losses over a large vocabulary have no forward-mode derivative")


def _arguments(hidden, weight, ids, logits, valid, temperature, reduction) -> L.VocabLoss:
    device, kd = getattr(hidden, "device", None), logits is not None
    for t in (hidden, weight, ids, logits if kd else ids, ids if valid is None else valid):
        if not isinstance(t, torch.Tensor):
            raise TypeError("hidden, weight, ids, teacher_logits and valid must be tensors")
        if not t.is_cuda:
            raise RuntimeError("supertoken_b200 operators need CUDA tensors; there is no CPU fallback")
        if t.device != device:
            raise ValueError("tensors must be on one device")
    _refuse_tangents(hidden, weight, logits)
    dtype = hidden.dtype
    if (dtype != torch.bfloat16 and dtype != torch.float16) or weight.dtype != dtype:
        raise TypeError("hidden and weight must both be bfloat16 or both be float16")
    if ids.dtype != torch.int32 and ids.dtype != torch.int64:
        raise TypeError("token ids must be int32 or int64")
    if valid is not None and valid.dtype != torch.uint8 and valid.dtype != torch.bool:
        raise TypeError("valid must be uint8 or bool")
    size, wide = hidden.shape, weight.shape
    lead, shape, D = len(size) - 1, size[:-1], size[-1] if size else 0
    if lead not in (1, 2) or len(wide) != 2 or wide[1] != D:
        raise ValueError("hidden must be [N, D] or [B, L, D] and weight [V, D]")
    if wide[0] < 1 or D < 1:
        raise ValueError("weight must have at least one row and one column")
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    if valid is not None and valid.shape != shape:
        raise ValueError("valid must have the shape of hidden without its last dimension")
    step, wide_step = hidden.stride(), weight.stride()
    if D > 1 and (step[-1] != 1 or wide_step[1] != 1):
        raise ValueError("the last dimension of hidden and weight must be contiguous")
    a = L.VocabLoss()
    if not kd:
        if ids.shape != shape:
            raise ValueError("targets must have the shape of hidden without its last dimension")
    else:
        if logits.dtype not in _REAL:
            raise TypeError("teacher_logits must be bfloat16, float16 or float32")
        if ids.dim() != lead + 1 or ids.shape[:-1] != shape or logits.shape != ids.shape:
            raise ValueError("teacher_ids and teacher_logits must have the shape of hidden with K as last dimension")
        a.k = k = ids.size(-1)
        if not 1 <= k <= MAX_TEACHER_ENTRIES:
            raise ValueError(f"a teacher gives 1 to {MAX_TEACHER_ENTRIES} entries per row")
        if k > 1 and (ids.stride(-1) != 1 or logits.stride(-1) != 1):
            raise ValueError("the last dimension of teacher_ids and teacher_logits must be contiguous")
        if not MIN_TEMPERATURE <= temperature <= MAX_TEMPERATURE:
            raise ValueError("temperature must lie between 2^-16 and 2^16")
        a.logits, a.logits_type = logits.data_ptr(), _REAL[logits.dtype]
        a.logits_outer, a.logits_inner = _rows(logits, lead)
    if lead == 2:
        a.outer, a.inner = shape
        a.hidden_outer = step[0]
    else:
        a.outer, a.inner = 1, shape[0]
    a.hidden_inner = step[-2]
    a.vocab, a.dim = wide
    a.type, a.ids_bytes = _REAL[dtype], 4 if ids.dtype == torch.int32 else 8
    a.reduction, a.temperature = _REDUCTIONS[reduction], temperature
    a.hidden, a.weight, a.ids = hidden.data_ptr(), weight.data_ptr(), ids.data_ptr()
    a.weight_stride = wide_step[0]
    a.ids_outer, a.ids_inner = _rows(ids, lead)
    if valid is not None:
        a.valid = valid.data_ptr()
        a.valid_outer, a.valid_inner = _rows(valid, lead)
    return a


def _run(a: L.VocabLoss, device: torch.device) -> None:
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _run(a, device)
    lib, need, err, here = L.load(), ctypes.c_int64(0), ctypes.create_string_buffer(256), ctypes.byref(a)
    st = lib.stbpe_vocab_loss_workspace(here, ctypes.byref(need), err, 256)
    if st == L.OK:
        # torch's allocator knows streams and captures: a graph's workspace is in the graph's own pool
        size = need.value
        space = torch.empty(size + 1024, dtype=torch.uint8, device=device)  # (held until all is launched)
        a.workspace, a.workspace_bytes = (space.data_ptr() + 1023) // 1024 * 1024, size
        st = lib.stbpe_vocab_loss_run(here, torch._C._cuda_getCurrentRawStream(index), err, 256)
    if st != L.OK:
        _raise(st, err.value.decode())


def _loss(a, hidden, reduction, for_backward=False):
    """The loss, and what the gradients need of it again; ``a``: the arguments."""
    loss = hidden.new_empty(hidden.shape[:-1] if reduction == "none" else (), dtype=torch.float32)
    lse2 = hidden.new_empty(max(1, a.outer * a.inner), dtype=torch.float32) if for_backward else None
    a.want, a.loss, a.lse2 = _WANT_LOSS, loss.data_ptr(), lse2.data_ptr() if for_backward else None
    if loss.numel():
        _run(a, hidden.device)
    return loss, lse2


def _grads(a, hidden, weight, reduction, grad_loss, lse2, want_hidden=True, want_weight=True, for_backward=False):
    """(loss or None, grad_hidden or None, grad_weight or None, lse2 or None); without ``lse2`` the loss is made, too."""
    shape, loss = hidden.shape[:-1], None
    if grad_loss is not None:
        if not isinstance(grad_loss, torch.Tensor):
            grad_loss = torch.full((), float(grad_loss), dtype=torch.float32, device=hidden.device)
        _refuse_tangents(grad_loss)
        if grad_loss.device != hidden.device:
            raise ValueError("tensors must be on one device")
        if grad_loss.dtype != torch.float32:
            raise TypeError("grad_loss must be float32")
        if reduction == "none" and grad_loss.shape == shape:
            a.grad_outer, a.grad_inner = _rows(grad_loss, len(shape))
        elif grad_loss.numel() != 1:
            raise ValueError("grad_loss must have one element, or the shape of the loss")
        a.grad_loss = grad_loss.data_ptr()
    gh = hidden.new_empty(hidden.shape) if want_hidden else None
    gw = weight.new_empty(weight.shape) if want_weight else None
    a.want = _WANT_GRADS
    if lse2 is None:
        loss = hidden.new_empty(shape if reduction == "none" else (), dtype=torch.float32)
        if for_backward:
            lse2 = hidden.new_empty(max(1, a.outer * a.inner), dtype=torch.float32)
        # (a tensor without elements has no address, and nothing is written to where it would be)
        a.want, a.loss = _WANT_LOSS | _WANT_GRADS, loss.data_ptr() or weight.data_ptr()
    a.lse2 = lse2.data_ptr() if lse2 is not None else None
    a.grad_hidden = gh.data_ptr() or None if want_hidden else None
    a.grad_weight = gw.data_ptr() if want_weight else None
    if loss is not None or a.grad_hidden or a.grad_weight:
        _run(a, hidden.device)
    return loss, gh, gw, lse2


class _VocabLoss(torch.autograd.Function):
    """One loss for a batch in bfloat16 makes its gradients with it, three products instead of the four of a loss and a later
    backward pass, which only multiplies them: exact for 1 and other powers of two, for other numbers one more rounding of the
    result.  Where what comes down differs from row to row, in float16 (a loss scale has to come before the gradients' rounding)
    and for a second backward pass, the gradients are made from the saved sums."""

    @staticmethod
    def forward(ctx, hidden, weight, ids, logits, valid, a, temperature, reduction):
        ctx.how, ctx.grads = (temperature, reduction), None
        if hidden.dtype == torch.bfloat16 and reduction != "none":
            wanted = ctx.needs_input_grad
            loss, gh, gw, lse2 = _grads(a, hidden, weight, reduction, None, None, wanted[0], wanted[1], for_backward=True)
            ctx.grads = gh, gw
        else:
            loss, lse2 = _loss(a, hidden, reduction, for_backward=True)
        ctx.save_for_backward(hidden, weight, ids, logits, valid, lse2)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        _refuse_capture(grad_loss.device)
        _refuse_tangents(grad_loss)
        if ctx.grads is not None:
            (gh, gw), ctx.grads = ctx.grads, None  # they are given away: a second pass makes its own
            _scale(gh, gw, grad_loss)
        else:
            hidden, weight, ids, logits, valid, lse2 = ctx.saved_tensors
            temperature, reduction = ctx.how
            a = _arguments(hidden, weight, ids, logits, valid, temperature, reduction)
            _, gh, gw, _ = _grads(a, hidden, weight, reduction, grad_loss, lse2, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return gh, gw, None, None, None, None, None, None


def _scale(gh: Optional[torch.Tensor], gw: Optional[torch.Tensor], by: torch.Tensor) -> None:
    index = by.device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _scale(gh, gw, by)
    st = L.load().stbpe_scale_gradients(gh.data_ptr() if gh is not None else None, gh.numel() if gh is not None else 0,
                                        gw.data_ptr() if gw is not None else None, gw.numel() if gw is not None else 0,
                                        by.data_ptr(), torch._C._cuda_getCurrentRawStream(index))
    if st != L.OK:
        _raise(st, f"stbpe_scale_gradients failed with status {st}")


def _refuse_capture(device: torch.device) -> None:
    """torch adds a leaf's gradient on the stream that the leaf was first used on.  A captured backward pass reaches out
    of its capture there when an eager graph of the same leaf is alive, which torch answers by ending the process."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _refuse_capture(device)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a loss with autograd cannot be captured: capture the call that returns the gradients "
                           "(vocab_cross_entropy_grads, vocab_distillation_grads)")


def _differentiable(hidden, weight, ids, logits, valid, temperature, reduction):
    a = _arguments(hidden, weight, ids, logits, valid, temperature, reduction)
    if logits is not None and logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("teacher_logits get no gradient: detach them")
    if (hidden.requires_grad or weight.requires_grad) and torch.is_grad_enabled():
        _refuse_capture(hidden.device)
        return _VocabLoss.apply(hidden, weight, ids, logits, valid, a, temperature, reduction)
    return _loss(a, hidden, reduction)[0]


def vocab_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                        valid: Optional[torch.Tensor] = None, *, reduction: str = "mean") -> torch.Tensor:
    """``-log softmax(hidden @ weight.T)[targets]`` in float32: a scalar, or one per row with ``reduction="none"``.
    Differentiable in ``hidden`` and ``weight``, once and in reverse mode.  A reduced loss in bfloat16 makes its gradients at once, so score under
    ``torch.no_grad()``; without gradients wanted the call can be captured into a graph."""
    return _differentiable(hidden, weight, targets, None, valid, 1.0, reduction)


def vocab_cross_entropy_grads(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                              valid: Optional[torch.Tensor] = None, grad_loss=None, *, reduction: str = "mean"
                              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss, grad_hidden, grad_weight)`` in one call without autograd, which can be captured into a graph.  The
    gradients are contiguous, in the inputs' type, and times ``grad_loss``: a number, a float32 tensor of one element (a loss
    scale), or with ``reduction="none"`` one of the loss's shape.  In float16 all rows' dlogits are held at one scale, the largest
    ``|grad_loss|``'s: rows with a millionth of it still have their gradient in full, those with less lose it bit by bit."""
    return _grads(_arguments(hidden, weight, targets, None, valid, 1.0, reduction), hidden, weight, reduction, grad_loss, None)[:3]


def vocab_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor,
                       teacher_logits: torch.Tensor, valid: Optional[torch.Tensor] = None, *, temperature: float = 1.0,
                       reduction: str = "mean") -> torch.Tensor:
    """``T^2 KL(p || softmax(hidden @ weight.T / T))`` with ``p = softmax(teacher_logits / T)`` over the teacher's up to 256
    entries of a row (in any order; an id below 0 is no entry, the same id twice counts twice); ``T`` between 2^-16 and 2^16.  The
    teacher's logits are constants: those that require a gradient are refused.  Gradients and captures as with
    ``vocab_cross_entropy``."""
    if teacher_logits is None:
        raise TypeError("teacher_logits must be a tensor")
    return _differentiable(hidden, weight, teacher_ids, teacher_logits, valid, float(temperature), reduction)


def vocab_distillation_grads(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor,
                             teacher_logits: torch.Tensor, valid: Optional[torch.Tensor] = None, grad_loss=None, *,
                             temperature: float = 1.0, reduction: str = "mean"
                             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss, grad_hidden, grad_weight)`` of ``vocab_distillation``, as ``vocab_cross_entropy_grads`` gives them."""
    if teacher_logits is None:
        raise TypeError("teacher_logits must be a tensor")
    a = _arguments(hidden, weight, teacher_ids, teacher_logits, valid, float(temperature), reduction)
    return _grads(a, hidden, weight, reduction, grad_loss, None)[:3]
