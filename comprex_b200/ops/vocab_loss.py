"""``linear_cross_entropy``: the loss of a language model's last layer and its gradients, without the logits in memory
(csrc/vocab_loss.cu).

    s = hidden weight^T        loss_r = log sum_v exp(s_rv) - s_r,target(r)

The [rows, vocab] logits of a training step are the largest tensor of the model (GPT-2 medium, 8192 tokens: 0.8 GB in
bf16, as much again for their gradient).  Here neither is stored: the forward call keeps one number per row, the
backward call computes the logits once more, a piece of the vocabulary at a time.
"""
from __future__ import annotations

from .. import _lib


def linear_cross_entropy(hidden, weight, targets, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of ``hidden @ weight.T`` against ``targets``, as ``torch.nn.functional.cross_entropy`` of
    those logits in 32 bits, with gradients for ``hidden`` and ``weight`` (which cannot be differentiated again).

    ``hidden`` [..., dim] and ``weight`` [vocab, dim]: float32, bfloat16 or float16, of one type and on one device;
    ``targets`` [...]: int64.  Rows whose target is ``ignore_index`` have loss 0 and no gradient; the mean is over the
    others, and NaN (with zero gradients) where there are none.  A target outside the vocabulary makes its row's loss
    and gradients NaN.  Under ``torch.autocast`` the product is in autocast's type.  The loss is float32: a scalar, or with ``reduction="none"`` of the shape of ``targets``."""
    try:
        code = _lib.REDUCTIONS[reduction]
    except (KeyError, TypeError):
        raise ValueError("reduction must be 'none', 'sum' or 'mean'") from None
    return _lib.host().vocab_loss(hidden, weight, targets, int(ignore_index), code)
