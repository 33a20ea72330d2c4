"""OmniWeave block: RMSNorm -> BiGEMM -> residual, fused on the B200 kernels.

Same constructor, parameter names, shapes and initialisation order as the
reference ``OmniWeaveBlock`` (omniweave/models/block.py:15-108), so state
dicts interchange and a seeded construction draws the same weights.  With
``backend="cuda"`` (or ``"auto"`` on a supported GPU) ``forward`` is one
fused call: the tile loads apply RMSNorm, the tile stores add the residual.

With ``post_norm=True`` the block normalises the operator's output as well,
``x + s * gamma * rms(bigemm(rms(x) w)) w_post``, and ``forward_blocks`` runs a
row of such blocks with each residual add and the next block's norm in one pass.
"""

from __future__ import annotations

import math
from collections.abc import Iterable

import torch
import torch.nn as nn
from torch import Tensor
from torch.nn.modules import module as _module

from omniwave_b200.norm import norm_residual, rms_norm
from omniwave_b200.ops import (bigemm_delta_cuda, block_forward, cuda_is_supported, drop_path_scale,
                               select_backend)
from omniwave_b200.routing import RoutePlan, build_route_plan


class OmniWeaveBlock(nn.Module):
    """One OmniWeave block returning ``x + delta``."""

    def __init__(
        self,
        height: int,
        width: int,
        dim: int,
        channel_tile: int,
        route: str,
        radix_level: int,
        expansion: int = 2,
        layer_scale_init: float = 1e-5,
        spatial_tile: int = 16,
        backend: str = "cuda",
        drop_path_rate: float = 0.0,
        post_norm: bool = False,
    ) -> None:
        super().__init__()
        if not 0.0 <= drop_path_rate < 1.0:
            raise ValueError("drop_path_rate must be in [0, 1)")
        self.height = height
        self.width = width
        self.dim = dim
        self.backend = backend
        self.drop_path_rate = drop_path_rate
        g = spatial_tile
        d = channel_tile
        rd = d * expansion
        q_c = math.ceil(dim / d)
        self.plan: RoutePlan = build_route_plan(height, width, dim, g, d, route, radix_level)
        # Creation and init order follow block.py:54-78 exactly.
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.a_u = nn.Parameter(torch.empty(g, g))
        self.a_v = nn.Parameter(torch.empty(g, g))
        self.a_o = nn.Parameter(torch.empty(g, g))
        self.b_u = nn.Parameter(torch.empty(q_c, d, rd))
        self.b_v = nn.Parameter(torch.empty(q_c, d, rd))
        self.b_o = nn.Parameter(torch.empty(q_c, rd, d))
        self.gamma = nn.Parameter(torch.full((dim,), layer_scale_init))
        self._init_weights()
        self.post_norm = post_norm
        if post_norm:  # not in the reference: its blocks hold no such parameter
            self.post_norm_weight = nn.Parameter(torch.ones(dim))
            # the gate goes on behind the norm, so the operator's own scale is 1
            self.register_buffer("_unit", torch.ones(dim), persistent=False)

    def _init_weights(self) -> None:
        nn.init.orthogonal_(self.a_u)
        nn.init.orthogonal_(self.a_v)
        nn.init.eye_(self.a_o)
        nn.init.xavier_uniform_(self.b_u)
        nn.init.xavier_uniform_(self.b_v)
        nn.init.xavier_uniform_(self.b_o)

    def _check_backend(self, x: Tensor) -> None:
        chosen, _ = select_backend(x, self.backend, lambda t: cuda_is_supported(t, self.plan, self.b_u))
        if chosen != "cuda":
            raise RuntimeError(
                f"OmniWeaveBlock backend {self.backend!r} resolved to {chosen!r}; "
                f"omniwave_b200 runs blocks only on the cuda backend"
            )

    def forward(self, x: Tensor) -> Tensor:
        """``x``: ``[B, H, W, C]`` -> ``[B, H, W, C]``."""
        if self.post_norm:
            return _forward_post_norm([self], x)
        self._check_backend(x)
        return block_forward(
            x, self.plan, self.norm_weight, self.a_u, self.a_v, self.a_o,
            self.b_u, self.b_v, self.b_o, self.gamma,
            drop_path_scale(x, self.gamma, self.drop_path_rate, self.training),
        )


def _plain_call(blk: nn.Module) -> bool:
    """Whether calling ``blk`` is ``OmniWeaveBlock.forward`` and nothing else: no hook, wrapper or override sees the call."""
    hooks = (blk._forward_hooks, blk._forward_pre_hooks, blk._backward_hooks, blk._backward_pre_hooks,
             _module._global_forward_hooks, _module._global_forward_pre_hooks, _module._global_backward_hooks,
             _module._global_backward_pre_hooks)
    return (type(blk).forward is OmniWeaveBlock.forward and type(blk).__call__ is nn.Module.__call__
            and "forward" not in vars(blk) and blk._compiled_call_impl is None and not any(hooks))


def forward_blocks(blocks: Iterable[nn.Module], x: Tensor) -> Tensor:
    """Run blocks one after another, ``x`` ``[B, H, W, C]`` -> ``[B, H, W, C]``.

    Between two post-norm blocks the first one's norm, gate and residual add
    and the second one's pre-norm are one kernel.  The residual stream keeps
    x's type there; the operator runs in the compute type (autocast's, or x's).
    Plain blocks, other modules (a wrapper around a block among them) and
    blocks with hooks or a ``forward`` of their own are called as they are.
    """
    run: list[OmniWeaveBlock] = []  # post-norm blocks to run together
    for blk in blocks:
        if isinstance(blk, OmniWeaveBlock) and blk.post_norm and _plain_call(blk):
            run.append(blk)
            continue
        x = blk(_forward_post_norm(run, x))
        run = []
    return _forward_post_norm(run, x)


def _forward_post_norm(blocks: list[OmniWeaveBlock], x: Tensor) -> Tensor:
    n = None  # the pre-norm of x, where the block before has taken it
    for i, blk in enumerate(blocks):
        blk._check_backend(x)
        if n is None:
            n = rms_norm(x, blk.norm_weight)
        delta = bigemm_delta_cuda(x=n, plan=blk.plan, a_u=blk.a_u, a_v=blk.a_v, a_o=blk.a_o,
                                  b_u=blk.b_u, b_v=blk.b_v, b_o=blk.b_o, gamma=blk._unit)
        nxt = blocks[i + 1] if i + 1 < len(blocks) else None
        out = norm_residual(x, delta, blk.post_norm_weight, blk.gamma,
                            sample_scale=drop_path_scale(x, blk.gamma, blk.drop_path_rate, blk.training),
                            next_weight=None if nxt is None else nxt.norm_weight)
        x, n = (out, None) if nxt is None else out
    return x
