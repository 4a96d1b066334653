"""``linear``: a product with bias, activation and residual in its epilogue, and its gradients (csrc/linear.cu).

    y = act(x w^T + b) + r        du = dy act'(u)    dx = du w    dw = du^T x    db = sum of du    dr = dy

One kernel forward; backward one pass that makes ``du`` and ``db`` and the two products.  Sums are held in 32 bits; a
training step keeps ``u`` (in the operands' type) where there is an activation.
"""
from __future__ import annotations

from .. import _lib


def linear(x, weight, bias=None, *, activation=None, residual=None):
    """``activation(x @ weight.T + bias) + residual``.

    ``x`` [..., inner], ``weight`` [outer, inner], ``bias`` [outer], ``residual`` [..., outer]: float32, bfloat16 or
    float16, all of one type and on one device (CUDA, or the host).  Rows may lie apart in memory; other orders are
    copied.  ``activation``: None, ``"relu"``, ``"gelu"``, ``"gelu_tanh"`` or ``"silu"``.  Gradients reach ``x``,
    ``weight``, ``bias`` and ``residual``, once: they cannot be differentiated again.  Under ``torch.autocast`` the operands
    are cast as torch's own product casts them, and a residual of another type is added to the result.  Products of 16-bit
    operands run on the tensor cores, of float32 on the CUDA cores; the host's are plain loops, for ranks without a GPU and for
    tests."""
    try:
        act = _lib.ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {sorted(a for a in _lib.ACTIVATIONS if a)} or None") from None
    return _lib.host().linear(x, weight, bias, act, residual)
