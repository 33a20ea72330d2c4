"""Linear layer with bias, activation and residual in its epilogue, on the B200 tensor cores.

The backbone's own projections are bias-free and fused with their
rearrangement (``s2d``), its head with the pool (``head``); this is the general
``nn.Linear`` next to them: ``y = act(x W^T + b) + residual`` as one kernel, its
backward as GEMMs that read their operands where they lie, and a kernel for the
few rows of a serving step.

The products are taken in 16 bits with f32 accumulation (autocast bf16/f16, or
a 16-bit model), as the rest of the cuda backend does; bias, activation and
residual are applied in f32 and ``y`` is rounded once.
"""

from __future__ import annotations

import torch
from torch import Tensor

from omniwave_b200 import _lib
from omniwave_b200.ops import _device_ok

__all__ = ["linear", "linear_supported"]

_C16 = (torch.bfloat16, torch.float16)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _compute(x: Tensor) -> torch.dtype:
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype


def linear_supported(x: Tensor, weight: Tensor, bias: Tensor | None = None,
                     residual: Tensor | None = None) -> tuple[bool, str | None]:
    """``(is_supported, reason_if_not)`` for tensors of ``linear``."""
    if not x.is_cuda:
        return False, "CUDA is unavailable"
    compute = _compute(x)
    if compute not in _C16:
        return False, f"compute dtype {compute} is not 16-bit"
    for t in (x, weight, bias, residual):
        if t is None:
            continue
        if t.dtype not in _FLOATS:
            return False, f"unsupported dtype {t.dtype}"
        if t.device != x.device:
            return False, f"tensors on {x.device} and {t.device}"
    if not torch.is_autocast_enabled("cuda") and any(t is not None and t.dtype != compute for t in (weight, residual)):
        return False, f"weight and residual must be {compute} without autocast"
    return _device_ok(x.device)


def _rows(t: Tensor) -> Tensor:
    """``t`` as a matrix whose rows lie densely, copied only if they do not."""
    t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _ld(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _args(x, weight, bias, residual, act) -> _lib.Linear:
    m, k = x.shape
    n = weight.shape[0]
    a = _lib.Linear(m, k, n, _lib.DTYPE_CODE[weight.dtype], _lib.ACTIVATIONS[act], x.data_ptr(), _ld(x),
                    weight.data_ptr(), _ld(weight))
    if bias is not None:
        a.bias, a.bias_dtype = bias.data_ptr(), _lib.DTYPE_CODE[bias.dtype]
    if residual is not None:
        a.residual, a.ldr = residual.data_ptr(), _ld(residual)
    return a


def _run(call, what: str, a: _lib.Linear, g, device) -> None:
    lib = _lib.load()
    with torch.cuda.device(device):  # the library launches on the current device
        size = lib.ow_linear_workspace_size(a, g)
        if size == 0:
            _lib.check(1, "ow_linear_workspace_size")
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
        stream = _lib.stream_handle(device)
        _lib.check(call(lib)(a, stream) if g is None else call(lib)(a, g, stream), what)
        del ws


def _forward(x, weight, bias, residual, act, keep):
    """``y`` and, when ``keep`` and the backward needs it, z, from matrices of the compute type."""
    m, n = x.shape[0], weight.shape[0]
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    z = None
    if keep and act != "none":
        z = torch.empty((m, -(-n // 8) * 8), dtype=x.dtype, device=x.device)
    if y.numel():
        a = _args(x, weight, bias, residual, act)
        a.out, a.z = y.data_ptr(), _lib.ptr(z)
        _run(lambda lib: lib.ow_linear_fwd, "ow_linear_fwd", a, None, x.device)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, compute):
        xm, wm = _rows(x.to(compute)), _rows(weight.to(compute))
        rm = None if residual is None else _rows(residual.to(compute))
        y, z = _forward(xm, wm, bias, rm, act, True)
        ctx.save_for_backward(xm, wm, bias, z)
        ctx.act = act
        ctx.shapes = (x.shape, x.dtype, weight.dtype, None if residual is None else (residual.shape, residual.dtype))
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, z = ctx.saved_tensors
        x_shape, x_dtype, w_dtype, res = ctx.shapes
        need = ctx.needs_input_grad
        dr = dy.to(res[1]) if res is not None and need[3] else None
        if not any(need[:3]):
            return None, None, None, dr, None, None
        g = dy.to(x.dtype).reshape(-1, weight.shape[0]).contiguous()
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
        dw = torch.empty(weight.shape, dtype=torch.float32 if w_dtype == torch.float32 else x.dtype,
                         device=x.device) if need[1] else None
        db = torch.empty_like(bias) if bias is not None and need[2] else None
        if g.numel() == 0:
            dw, db = (None if t is None else t.zero_() for t in (dw, db))
        else:
            a = _args(x, weight, bias, None, ctx.act)
            a.z = _lib.ptr(z)
            grads = _lib.LinearGrads(g.data_ptr(), _lib.ptr(dx), _lib.ptr(dw),
                                     0 if dw is None else _lib.DTYPE_CODE[dw.dtype], _lib.ptr(db))
            _run(lambda lib: lib.ow_linear_bwd, "ow_linear_bwd", a, grads, x.device)
        return (None if dx is None else dx.to(x_dtype).view(x_shape), None if dw is None else dw.to(w_dtype), db, dr,
                None, None)


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str = "none",
           residual: Tensor | None = None) -> Tensor:
    """``act(x @ weight.T + bias) + residual``.

    ``x`` is ``[..., K]``, ``weight`` ``[N, K]`` (as ``nn.Linear`` holds it), ``bias``
    ``[N]``, ``residual`` ``[..., N]``; ``activation`` is ``"none"``, ``"relu"``,
    ``"silu"`` or ``"gelu"`` (by erf).  The result is in the compute type:
    autocast's where it is on, and then x, weight and residual are cast to it
    (an f32 weight gets an f32 gradient); else x's, which must be 16-bit, and
    weight and residual must have it too.  Raises ``RuntimeError`` for what the
    kernels do not take.
    """
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_lib.ACTIVATIONS)}, got {activation!r}")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight must be [N, K], got {tuple(weight.shape)}")
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x must be [..., {k}], got {tuple(x.shape)}")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], n):
        raise ValueError(f"residual must be {(*x.shape[:-1], n)}, got {tuple(residual.shape)}")
    ok, why = linear_supported(x, weight, bias, residual)
    if not ok:
        raise RuntimeError(f"linear not supported: {why}")
    compute = _compute(x)
    if bias is not None:
        bias = bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _Linear.apply(x, weight, bias, residual, activation, compute)
    r = None if residual is None else _rows(residual.detach().to(compute))
    y, _ = _forward(_rows(x.detach().to(compute)), _rows(weight.detach().to(compute)),
                    None if bias is None else bias.detach(), r, activation, False)
    return y.view(*x.shape[:-1], n)
