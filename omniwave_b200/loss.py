"""Loss of a classifier that learns from a teacher's top logits and from labels.

The reference trains on labels alone (``F.cross_entropy``,
omniweave/training/engine.py:193-210).  A student that is distilled adds the
divergence from a teacher of which only the largest logits of each sample are
kept, as they are when a large teacher's answers are stored.  ``distill_loss`` takes
both terms from one pass over the logits, and their gradient from another
(``ow_distill_fwd``, ``ow_distill_bwd``); ``train.TrainStep`` calls it when it is
given a teacher's logits.
"""

from __future__ import annotations

from torch import Tensor

from omniwave_b200 import _lib

__all__ = ["distill_loss"]


def distill_loss(logits: Tensor, top_logits: Tensor, top_classes: Tensor, labels: Tensor | None = None, *,
                 temperature: float = 1.0, weight: float = 0.5, reduction: str = "mean") -> Tensor:
    """``weight * T^2 KL(p || softmax(logits / T)) + (1 - weight) * cross_entropy(logits, labels)``.

    ``logits`` is ``[..., V]`` in float32, bfloat16 or float16.  ``top_logits``
    ``[..., K]`` (any of these types, K at most 1024) are the teacher's logits of
    the classes ``top_classes`` ``[..., K]`` (int32 or int64), and ``p`` is the softmax
    of ``top_logits / T`` over them; ``T`` is ``temperature``.  A negative class is
    padding; an entry of -inf has probability 0; a class named twice counts twice.
    A row with no entry above -inf has no first term, a row with a negative label
    (such as -100), or without ``labels``, no second.  A class or label that is not
    below V makes its row's loss and gradient NaN.

    ``reduction`` ``"mean"`` takes each term's mean over the rows that have it (0 if
    none has), ``"sum"`` the sum over rows, ``"none"`` gives ``[...]``.  The result is
    float32; the gradient, of ``logits`` alone, has their type.  Bad shapes and values
    raise ``ValueError``, what the kernels do not take ``RuntimeError``.  The backward
    cannot be differentiated again, and forward-mode differentiation is refused.
    """
    how = _lib.REDUCTIONS.get(reduction)
    if how is None:
        raise ValueError(f"reduction must be one of {sorted(_lib.REDUCTIONS)}, got {reduction!r}")
    return _lib.host().distill_loss(logits, top_logits, top_classes, labels, temperature, weight, how)
