"""``linear``: a product with bias, activation and residual in its epilogue, and its gradients (csrc/linear.cu).

    y = act(x w^T + b) + r        du = dy act'(u)    dx = du w    dw = du^T x    db = sum of du    dr = dy

One kernel forward; backward one pass that makes ``du`` and ``db`` and the two products.  Sums are held in 32 bits; a
training step keeps ``u`` (in the operands' type) where there is an activation.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from .. import _lib
from .._lib import ComprexError


def on_device(t: torch.Tensor):
    """Context in which launches go to the device of ``t``."""
    if t.is_cuda and t.device.index != torch.cuda.current_device():
        return torch.cuda.device(t.device)
    return contextlib.nullcontext()


def rows_of(t: torch.Tensor, cols: int) -> torch.Tensor:
    """``t`` as a matrix of rows of ``cols`` consecutive elements that do not overlap: a view where that can be."""
    m = t.reshape(-1, cols)
    if m.size(0) > 1 and m.stride(0) < cols or cols > 1 and m.stride(1) != 1:
        m = m.contiguous()
    return m


def stride_of(m: torch.Tensor) -> int:
    return m.stride(0) if m.size(0) > 1 else m.size(1)


def workspace(d, query, device: torch.device, backward: int):
    """Scratch of one call, of the current stream, in the descriptor ``d``; the caller keeps it until the launches are out."""
    d.ws_bytes = query(_lib.DEV_CUDA, C.byref(d), backward) if device.type == "cuda" else 0
    if not d.ws_bytes:
        return None
    ws = torch.empty(d.ws_bytes, dtype=torch.uint8, device=device)
    d.workspace = ws.data_ptr()
    return ws


def _check(x, weight, bias, activation, residual):
    for name, t in (("x", x), ("weight", weight), ("bias", bias), ("residual", residual)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise ComprexError(f"{name} must be a strided tensor")
        if t.dtype != x.dtype or t.device != x.device:
            raise ComprexError(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}: one type and device are needed")
    _lib.dtype_code(x.dtype)
    if x.device.type not in ("cuda", "cpu"):
        raise ComprexError(f"tensors on {x.device} are not supported")
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(a for a in _lib.ACTIVATIONS if a)} or None")
    if weight.dim() != 2 or x.dim() < 1 or x.size(-1) != weight.size(1) or weight.numel() == 0:
        raise ComprexError(f"x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ComprexError(f"bias {tuple(bias.shape)} does not fit weight {tuple(weight.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], weight.size(0)):
        raise ComprexError(f"residual {tuple(residual.shape)} does not have the result's shape")


def _forward(x, weight, bias, activation, residual, keep_pre):
    outer, inner = weight.shape
    y = torch.empty((*x.shape[:-1], outer), dtype=x.dtype, device=x.device)
    pre = torch.empty_like(y) if keep_pre else None
    if y.numel() == 0:
        return y, pre
    d = _lib.Linear()
    xm, wm = rows_of(x, inner), rows_of(weight, inner)
    rm = None if residual is None else rows_of(residual, outer)
    bias = None if bias is None else bias.contiguous()
    d.rows, d.inner, d.outer = xm.size(0), inner, outer
    d.x, d.ldx, d.w, d.ldw, d.y = xm.data_ptr(), stride_of(xm), wm.data_ptr(), stride_of(wm), y.data_ptr()
    if bias is not None:
        d.bias = bias.data_ptr()
    if rm is not None:
        d.residual, d.ldr = rm.data_ptr(), stride_of(rm)
    if pre is not None:
        d.pre = pre.data_ptr()
    d.dtype, d.act = _lib.dtype_code(x.dtype), _lib.ACTIVATIONS[activation]
    lib = _lib.load()
    with on_device(x):
        ws = workspace(d, lib.cx_linear_workspace_bytes, x.device, 0)
        _lib.check(lib.cx_linear_forward(_lib.dev_code(x), C.byref(d), _lib.stream_ptr(x.device)), "cx_linear_forward")
        del ws
    return y, pre


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        y, pre = _forward(x, weight, bias, activation, residual, activation is not None)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, pre)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        outer, inner = weight.shape
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        dw = torch.empty(weight.shape, dtype=x.dtype, device=x.device) if need[1] else None
        db = torch.empty(outer, dtype=x.dtype, device=x.device) if need[2] else None
        if grad.numel() == 0:
            return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_(), None, grad if need[4] else None
        if dx is not None or dw is not None or db is not None:
            d = _lib.Linear()
            gm, xm, wm = rows_of(grad, outer), rows_of(x, inner), rows_of(weight, inner)
            d.rows, d.inner, d.outer = gm.size(0), inner, outer
            d.x, d.ldx, d.w, d.ldw = xm.data_ptr(), stride_of(xm), wm.data_ptr(), stride_of(wm)
            d.grad, d.ldg = gm.data_ptr(), stride_of(gm)
            if pre is not None:
                d.pre = pre.data_ptr()
            for name, t in (("dx", dx), ("dw", dw), ("dbias", db)):
                if t is not None:
                    setattr(d, name, t.data_ptr())
            d.dtype, d.act = _lib.dtype_code(x.dtype), _lib.ACTIVATIONS[ctx.activation]
            lib = _lib.load()
            with on_device(x):
                ws = workspace(d, lib.cx_linear_workspace_bytes, x.device, 1)
                _lib.check(lib.cx_linear_backward(_lib.dev_code(x), C.byref(d), _lib.stream_ptr(x.device)), "cx_linear_backward")
                del ws
        return dx, dw, db, None, grad if need[4] else None


def linear(x, weight, bias=None, *, activation=None, residual=None):
    """``activation(x @ weight.T + bias) + residual``.

    ``x`` [..., inner], ``weight`` [outer, inner], ``bias`` [outer], ``residual`` [..., outer]: float32, bfloat16 or
    float16, all of one type and on one device (CUDA, or the host).  Rows may lie apart in memory; other orders are
    copied.  ``activation``: None, ``"relu"``, ``"gelu"``, ``"gelu_tanh"`` or ``"silu"``.  Gradients reach ``x``,
    ``weight``, ``bias`` and ``residual``."""
    _check(x, weight, bias, activation, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _Linear.apply(x, weight, bias, activation, residual)
    return _forward(x, weight, bias, activation, residual, False)[0]
