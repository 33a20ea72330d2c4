"""Linear layer with bias, activation and residual in its epilogue, on the B200 tensor cores.

The backbone's own projections are bias-free and fused with their
rearrangement (``s2d``), its head with the pool (``head``); this is the general
``nn.Linear`` next to them: ``y = act(x W^T + b) + residual`` as one kernel, its
backward as GEMMs that read their operands where they lie, and a kernel for the
few rows of a serving step (``csrc/ow_linear.cu``; argument checks and the
autograd node in ``csrc/host/ow_host.cpp``).

The products are taken in 16 bits with f32 accumulation (autocast bf16/f16, or
a 16-bit model), as the rest of the cuda backend does; bias, activation and
residual are applied in f32 and ``y`` is rounded once.  gelu's own error is under a
third of that rounding, for small results too.
"""

from __future__ import annotations

from torch import Tensor

from omniwave_b200 import _lib

__all__ = ["linear", "linear_supported"]


def linear_supported(x: Tensor, weight: Tensor, bias: Tensor | None = None,
                     residual: Tensor | None = None) -> tuple[bool, str | None]:
    """``(is_supported, reason_if_not)`` for tensors of ``linear``."""
    return _lib.host().linear_supported(x, weight, bias, residual)


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str = "none",
           residual: Tensor | None = None) -> Tensor:
    """``act(x @ weight.T + bias) + residual``.

    ``x`` is ``[..., K]``, ``weight`` ``[N, K]`` (as ``nn.Linear`` holds it), ``bias``
    ``[N]``, ``residual`` ``[..., N]``; ``activation`` is ``"none"``, ``"relu"``,
    ``"silu"`` or ``"gelu"`` (by erf).  The result is in the compute type:
    autocast's where it is on, and then x, weight and residual are cast to it
    (an f32 weight gets an f32 gradient); else x's, which must be 16-bit, and
    weight and residual must have it too.  Bad shapes raise ``ValueError``, what
    the kernels do not take ``RuntimeError``.  The backward holds the
    pre-activation in the compute type; it cannot be differentiated again, and
    forward-mode differentiation is refused.
    """
    act = _lib.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(_lib.ACTIVATIONS)}, got {activation!r}")
    return _lib.host().linear(x, weight, bias, act, residual)
