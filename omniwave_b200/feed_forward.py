"""Gated feed-forward block on the B200 tensor cores.

``y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual``: the block that mixes
channels between BiGEMM blocks where a model has one (the operator's own channel
mix, omniweave/ops/reference.py:155-162, is gated the same way, within groups of
channels).  Both projections, the activation and the product are one kernel, the
projection back with its residual is ``linear.linear``'s; a serving step's few rows
read each weight once (``csrc/ow_ffn.cu``; argument checks and the autograd node in
``csrc/host/ow_host.cpp``).

As in ``linear``, products are taken in 16 bits with f32 accumulation; bias,
activation, product and residual are f32.  The gated product is rounded to the
compute type before the projection back, ``y`` once.
"""

from __future__ import annotations

from torch import Tensor

from omniwave_b200 import _lib

__all__ = ["gated_feed_forward", "gated_feed_forward_supported"]


def gated_feed_forward_supported(x: Tensor, gate_weight: Tensor, up_weight: Tensor, down_weight: Tensor, *,
                                 gate_bias: Tensor | None = None, up_bias: Tensor | None = None,
                                 down_bias: Tensor | None = None,
                                 residual: Tensor | None = None) -> tuple[bool, str | None]:
    """``(is_supported, reason_if_not)`` for tensors of ``gated_feed_forward``."""
    return _lib.host().gated_feed_forward_supported(x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias,
                                                    residual)


def gated_feed_forward(x: Tensor, gate_weight: Tensor, up_weight: Tensor, down_weight: Tensor, *,
                       gate_bias: Tensor | None = None, up_bias: Tensor | None = None,
                       down_bias: Tensor | None = None, activation: str = "silu",
                       residual: Tensor | None = None) -> Tensor:
    """``(act(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias)) @ down_weight.T + down_bias + residual``.

    ``x`` is ``[..., K]``, ``gate_weight`` and ``up_weight`` ``[F, K]``, ``down_weight``
    ``[N, F]`` (as ``nn.Linear`` holds them; the halves of a packed ``[2F, K]`` weight
    serve as they are), the biases ``[F]``, ``[F]`` and ``[N]``, ``residual``
    ``[..., N]``; ``activation`` is ``"silu"``, ``"gelu"`` (by erf), ``"relu"`` or
    ``"none"``.  Types, errors and derivatives as for ``linear.linear``.  The backward
    holds the gated product, the activation and its slope times the other projection,
    each ``[..., F]`` in the compute type; in float16 the last two end at its largest
    value, 65504.
    """
    act = _lib.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(_lib.ACTIVATIONS)}, got {activation!r}")
    return _lib.host().gated_feed_forward(x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias, act, residual)
