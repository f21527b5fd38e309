"""Losses of a language model's head through the HIP library, as torch
autograd functions (pto_linear_cross_entropy, pto_linear_distillation).

With a mean or sum the forward call also returns the gradients of hidden and
weight, so the backward only multiplies them by the gradient of the loss (in
place, and not at all where that is 1). They are handed out once; a second
backward through a retained graph computes them again. With one loss per row
the forward keeps the normalisers and the targets' logits, and the backward computes the
gradients under the rows' own.
"""

from __future__ import annotations

import contextlib
import functools

import torch
from torch.autograd.function import once_differentiable

from . import reference
from .reference import OpsArgumentError

_DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 2}
_REDUCTION_CODE = {"none": 0, "mean": 1, "sum": 2}
MAX_TEACHER = 1024


def _ptr(t):
    return None if t is None else t.data_ptr()


def _on(device):
    """The tensors' GPU as the current one; a switch costs more than the rest of a small call's host work."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _rows_readable(t):
    """t as the library reads a matrix: contiguous rows at a pitch."""
    return t if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(lib, *sizes):
    return lib.pto_linear_loss_workspace_bytes(*sizes)


class _Call:
    """One loss: its constants, and the C call that computes parts of it."""

    def __init__(self, backend, what, dtype, labels, k, options, reduction):
        self.backend, self.what, self.labels, self.k = backend, what, labels, k
        self.code = _DTYPE_CODE.get(dtype)
        self.options, self.reduction = options, _REDUCTION_CODE[reduction]

    def __call__(self, h, w, loss=None, norm=None, z=None, dh=None, dw=None, grad_rows=None):
        be, lib = self.backend, self.backend._lib
        code, (rows, d), vocab = self.code, h.shape, w.shape[0]
        ldh = h.stride(0) if rows > 1 else d
        ldw = w.stride(0) if vocab > 1 else d
        ce = self.what == "linear_cross_entropy"
        sizes = (code, rows, d, vocab) if ce else (code, rows, d, vocab, self.k)
        with _on(h.device):
            nbytes = _workspace_bytes(lib, code, rows, d, vocab, self.k, ldw, self.options[1] if ce else 0.0, int(not ce),
                                      int(grad_rows is not None), int(dh is not None), int(dw is not None),
                                      be.LOSS_CHUNK_BYTES)
            ws = be._workspace(nbytes, h.device)
            rc = (lib.pto_linear_cross_entropy if ce else lib.pto_linear_distillation)(
                _ptr(h), ldh, _ptr(w), ldw, *map(_ptr, self.labels), *sizes, *self.options, self.reduction,
                _ptr(grad_rows), _ptr(loss), _ptr(norm), _ptr(z), _ptr(dh), _ptr(dw), be.LOSS_CHUNK_BYTES, _ptr(ws),
                nbytes, be._stream(h.device))
        be._check(rc, self.what)

    def gradients(self, h, w, needs, **more):
        dh = torch.empty(h.shape, dtype=h.dtype, device=h.device) if needs[0] else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if needs[1] else None
        self(h, w, dh=dh, dw=dw, **more)
        return dh, dw


def _readable(h, w):
    h, w = _rows_readable(h), _rows_readable(w)
    return h, w.clone(memory_format=torch.contiguous_format) if w.data_ptr() % 16 else w


def _score(call, h, w):
    h, w = _readable(h, w)
    loss = torch.empty(() if call.reduction else h.shape[0], dtype=torch.float32, device=h.device)
    call(h, w, loss=loss)
    return loss


class _LinearLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, call, needs):
        ctx.call, ctx.needs, ctx.grads = call, needs, None
        h, w = _readable(h, w)
        if call.reduction:
            loss = torch.empty((), dtype=torch.float32, device=h.device)
            ctx.grads = call.gradients(h, w, needs, loss=loss)
            ctx.save_for_backward(h, w)
            return loss
        loss = torch.empty(h.shape[0], dtype=torch.float32, device=h.device)
        norm = torch.empty(2 * h.shape[0], dtype=torch.float32, device=h.device)
        z = torch.empty(h.shape[0] * call.k, dtype=torch.float32, device=h.device)
        call(h, w, loss=loss, norm=norm, z=z)
        ctx.save_for_backward(h, w, norm, z)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        call, be = ctx.call, ctx.call.backend
        grad = grad.to(torch.float32).contiguous()
        if not call.reduction:
            h, w, norm, z = ctx.saved_tensors
            if h.shape[0] == 0:
                return (*(torch.zeros_like(t) if n else None for t, n in zip((h, w), ctx.needs)), None, None)
            dh, dw = call.gradients(h, w, ctx.needs, norm=norm, z=z, grad_rows=grad)
            return dh, dw, None, None
        grads, ctx.grads = ctx.grads, None
        if grads is None:
            h, w = ctx.saved_tensors
            grads = call.gradients(h, w, ctx.needs, loss=torch.empty_like(grad))
        dh, dw = grads
        with _on(grad.device):
            rc = be._lib.pto_scale_pair(_ptr(dh), 0 if dh is None else dh.numel(), _ptr(dw),
                                        0 if dw is None else dw.numel(), call.code, _ptr(grad),
                                        be._stream(grad.device))
        be._check(rc, call.what)
        return dh, dw, None, None


def _apply(call, hidden, weight, shape):
    if call.code is None:
        raise OpsArgumentError(f"{call.what}: float32 and bfloat16 on the GPU, got {hidden.dtype}")
    on = torch.is_grad_enabled()
    needs = (on and hidden.requires_grad, on and weight.requires_grad)
    h = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    loss = _LinearLoss.apply(h, weight, call, needs) if any(needs) else _score(call, h.detach(), weight.detach())
    return loss if call.reduction else loss.reshape(shape)


def _autocast(hidden, weight):
    if torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        return hidden.to(to), weight.to(to)
    return hidden, weight


def cross_entropy(backend, hidden, weight, targets, ignore_index, label_smoothing, z_loss, reduction):
    hidden, weight = _autocast(hidden, weight)
    reference.check_cross_entropy(hidden, weight, targets, label_smoothing, z_loss, reduction)
    labels = (targets.reshape(-1).to(torch.int64).contiguous(),)
    call = _Call(backend, "linear_cross_entropy", hidden.dtype, labels, 1, (ignore_index, label_smoothing, z_loss), reduction)
    return _apply(call, hidden, weight, targets.shape)


def distillation(backend, hidden, weight, teacher_logits, teacher_index, temperature, reduction):
    hidden, weight = _autocast(hidden, weight)
    reference.check_distillation(hidden, weight, teacher_logits, teacher_index, temperature, reduction)
    k = teacher_index.shape[-1]
    if k > MAX_TEACHER:
        raise OpsArgumentError(f"linear_distillation: at most {MAX_TEACHER} teacher entries per row, got {k}")
    labels = (teacher_logits.detach().reshape(-1).to(torch.float32).contiguous(),
              teacher_index.reshape(-1).to(torch.int64).contiguous())
    call = _Call(backend, "linear_distillation", hidden.dtype, labels, k, (temperature,), reduction)
    return _apply(call, hidden, weight, teacher_index.shape[:-1])
