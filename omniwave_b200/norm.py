"""RMSNorm before and after a block, with the block's gate, residual scale and residual add.

The reference's block normalises its input only: ``x + s * gamma * f(rms(x) w)``
(omniweave/models/block.py:80-108, fused by ``ops.block_forward``).  A block that
is normalised on both sides adds ``s * gate * rms(delta) * w_post`` instead, and
the next block starts with ``rms(h) * w_next``; ``norm_residual`` does both in one
pass over ``x`` and ``delta``, and ``rms_norm`` is the norm in front of the first
block.  Forward and backward are CUDA kernels (``ow_norm_fwd``, ``ow_norm_bwd``);
argument checks and the autograd node are native too (``csrc/host/ow_host.cpp``).

All arithmetic is f32, whatever the tensors' types; each output is rounded once.
"""

from __future__ import annotations

import torch
from torch import Tensor

from omniwave_b200 import _lib
from omniwave_b200.ops import RMS_EPS

__all__ = ["norm_residual", "norm_supported", "rms_norm"]


def norm_supported(x: Tensor, *others: Tensor | None) -> tuple[bool, str | None]:
    """``(is_supported, reason_if_not)`` for tensors of ``rms_norm`` and ``norm_residual``."""
    return _lib.host().norm_supported(x, list(others))


def rms_norm(x: Tensor, weight: Tensor, *, eps: float = RMS_EPS, out_dtype: torch.dtype | None = None) -> Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last dimension.

    ``x`` is ``[..., C]`` in float32, bfloat16 or float16, ``weight`` ``[C]``.  The
    result is in ``out_dtype``: by default the autocast type where autocast is
    on, else x's.  Bad shapes raise ``ValueError``, what the kernels do not take
    ``RuntimeError``.  The backward cannot be differentiated again, and forward-mode
    differentiation is refused.
    """
    return _lib.host().rms_norm(x, weight, eps, out_dtype)


def norm_residual(x: Tensor, delta: Tensor, weight: Tensor, gate: Tensor | None = None, *,
                  sample_scale: Tensor | None = None, next_weight: Tensor | None = None,
                  eps: float = RMS_EPS, out_dtype: torch.dtype | None = None):
    """``h = x + sample_scale[b] * gate * rms(delta) * weight``, and the next block's ``rms(h) * next_weight``.

    ``x`` and ``delta`` are ``[B, ..., C]`` (each float32, bfloat16 or float16;
    ``h`` has x's type), ``weight`` and ``next_weight`` ``[C]``, ``gate`` ``[C]``,
    or ``[B, C]`` with one for each sample.  ``sample_scale`` ``[B]`` is the
    drop-path scale (``ops.drop_path_scale``); it takes no gradient.  Returns
    ``h``, or ``(h, n)`` with ``next_weight``; ``n`` is taken from the unrounded
    ``h`` and is in ``out_dtype``.  Types and errors as for ``rms_norm``.
    """
    out = _lib.host().norm_residual(x, delta, weight, gate, sample_scale, next_weight, eps, out_dtype)
    return out[0] if next_weight is None else tuple(out)
