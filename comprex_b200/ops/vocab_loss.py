"""``linear_cross_entropy``: the loss of a language model's last layer and its gradients, without the logits in memory
(csrc/vocab_loss.cu).

    s = hidden weight^T        loss_r = log sum_v exp(s_rv) - s_r,target(r)

The [rows, vocab] logits of a training step are the largest tensor of the model (GPT-2 medium, 8192 tokens: 0.8 GB in
bf16, as much again for their gradient).  Here neither is stored: the forward call keeps one number per row, the
backward call computes the logits once more, a piece of the vocabulary at a time.
"""
from __future__ import annotations

import ctypes as C

import torch

from .. import _lib
from .._lib import ComprexError
from .linear import on_device, rows_of, stride_of, workspace


def _descriptor(hm, wm, tm, ignore_index, reduction, lse, count):
    d = _lib.VocabLoss()
    d.rows, d.vocab, d.dim = hm.size(0), wm.size(0), wm.size(1)
    d.h, d.ldh, d.w, d.ldw, d.targets = hm.data_ptr(), stride_of(hm), wm.data_ptr(), stride_of(wm), tm.data_ptr()
    d.ignore_index, d.lse, d.count = ignore_index, lse.data_ptr(), count.data_ptr()
    d.dtype, d.reduction = _lib.dtype_code(hm.dtype), _lib.REDUCTIONS[reduction]
    return d


def _forward(hidden, weight, targets, ignore_index, reduction):
    hm, wm, tm = rows_of(hidden, weight.size(1)), rows_of(weight, weight.size(1)), targets.reshape(-1).contiguous()
    rows, new = hm.size(0), dict(dtype=torch.float32, device=hidden.device)
    loss = torch.empty(targets.shape if reduction == "none" else (), **new)
    lse, count = torch.empty(rows, **new), torch.empty(1, **new)
    if rows == 0:
        return (loss if reduction == "none" else loss.fill_(0.0 if reduction == "sum" else float("nan"))), lse, count, tm
    d = _descriptor(hm, wm, tm, ignore_index, reduction, lse, count)
    d.loss = loss.data_ptr()
    lib = _lib.load()
    with on_device(hidden):
        ws = workspace(d, lib.cx_vocab_loss_workspace_bytes, hidden.device, 0)
        _lib.check(lib.cx_vocab_loss_forward(_lib.dev_code(hidden), C.byref(d), _lib.stream_ptr(hidden.device)), "cx_vocab_loss_forward")
        del ws
    return loss, lse, count, tm


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        loss, lse, count, tm = _forward(hidden, weight, targets, ignore_index, reduction)
        ctx.settings = ignore_index, reduction
        ctx.save_for_backward(hidden, weight, tm, lse, count)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, tm, lse, count = ctx.saved_tensors
        need = ctx.needs_input_grad
        dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if need[0] else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if need[1] else None
        if tm.numel() == 0:
            return dh, None if dw is None else dw.zero_(), None, None, None
        hm, wm = rows_of(hidden, weight.size(1)), rows_of(weight, weight.size(1))
        d = _descriptor(hm, wm, tm, *ctx.settings, lse, count)
        gm = grad.to(torch.float32)
        if gm.dim() > 1:
            gm = gm.reshape(-1)
        d.grad, d.grad_stride = gm.data_ptr(), gm.stride(0) if gm.dim() else 0
        if dh is not None:
            d.dh = dh.data_ptr()
        if dw is not None:
            d.dw = dw.data_ptr()
        lib = _lib.load()
        with on_device(hidden):
            ws = workspace(d, lib.cx_vocab_loss_workspace_bytes, hidden.device, 1)
            _lib.check(lib.cx_vocab_loss_backward(_lib.dev_code(hidden), C.byref(d), _lib.stream_ptr(hidden.device)), "cx_vocab_loss_backward")
            del ws
        return dh, dw, None, None, None


def linear_cross_entropy(hidden, weight, targets, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of ``hidden @ weight.T`` against ``targets``, as ``torch.nn.functional.cross_entropy`` of
    those logits in 32 bits, with gradients for ``hidden`` and ``weight``.

    ``hidden`` [..., dim] and ``weight`` [vocab, dim]: float32, bfloat16 or float16, of one type and on one device;
    ``targets`` [...]: int64.  Rows whose target is ``ignore_index`` have loss 0 and no gradient; the mean is over the
    others, and NaN (with zero gradients) where there are none.  A target outside the vocabulary makes its row's loss
    and gradients NaN.  The loss is float32: a scalar, or with ``reduction="none"`` of the shape of ``targets``."""
    if reduction not in _lib.REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    for name, t in (("hidden", hidden), ("weight", weight), ("targets", targets)):
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise ComprexError(f"{name} must be a strided tensor")
        if t.device != hidden.device:
            raise ComprexError(f"{name} is on {t.device}, hidden on {hidden.device}")
    if hidden.device.type not in ("cuda", "cpu"):
        raise ComprexError(f"tensors on {hidden.device} are not supported")
    if weight.dtype != hidden.dtype:
        raise ComprexError(f"weight is {weight.dtype}, hidden {hidden.dtype}: one type is needed")
    _lib.dtype_code(hidden.dtype)
    if targets.dtype != torch.int64:
        raise ComprexError(f"targets must be int64, not {targets.dtype}")
    if weight.dim() != 2 or weight.numel() == 0 or hidden.dim() < 1 or hidden.size(-1) != weight.size(1):
        raise ComprexError(f"hidden {tuple(hidden.shape)} does not fit weight {tuple(weight.shape)}")
    if targets.shape != hidden.shape[:-1]:
        raise ComprexError(f"targets {tuple(targets.shape)} do not fit hidden {tuple(hidden.shape)}")
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _VocabLoss.apply(hidden, weight, targets, int(ignore_index), reduction)
    return _forward(hidden, weight, targets, int(ignore_index), reduction)[0]
