"""RMSNorm before and after a block, with the block's gate, residual scale and residual add.

The reference's block normalises its input only: ``x + s * gamma * f(rms(x) w)``
(omniweave/models/block.py:80-108, fused by ``ops.block_forward``).  A block that
is normalised on both sides adds ``s * gate * rms(delta) * w_post`` instead, and
the next block starts with ``rms(h) * w_next``; ``norm_residual`` does both in one
pass over ``x`` and ``delta``, and ``rms_norm`` is the norm in front of the first
block.  Forward and backward are CUDA kernels (``ow_norm_fwd``, ``ow_norm_bwd``).

All arithmetic is f32, whatever the tensors' types; each output is rounded once.
"""

from __future__ import annotations

import torch
from torch import Tensor

from omniwave_b200 import _lib
from omniwave_b200.ops import RMS_EPS, _device_ok

__all__ = ["norm_residual", "norm_supported", "rms_norm"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def norm_supported(x: Tensor, *others: Tensor | None) -> tuple[bool, str | None]:
    """``(is_supported, reason_if_not)`` for tensors of ``rms_norm`` and ``norm_residual``."""
    if not x.is_cuda:
        return False, "CUDA is unavailable"
    for t in (x, *others):
        if t is None:
            continue
        if t.dtype not in _DTYPES:
            return False, f"unsupported dtype {t.dtype}"
        if t.device != x.device:
            return False, f"tensors on {x.device} and {t.device}"
    return _device_ok(x.device)


def _require(x: Tensor, *others: Tensor | None) -> None:
    ok, why = norm_supported(x, *others)
    if not ok:
        raise RuntimeError(f"norm not supported: {why}")


def _out_dtype(x: Tensor, out_dtype: torch.dtype | None) -> torch.dtype:
    if out_dtype is None:
        out_dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
    if out_dtype not in _DTYPES:
        raise RuntimeError(f"norm not supported: unsupported dtype {out_dtype}")
    return out_dtype


def _vector(name: str, w: Tensor, c: int) -> None:
    if w.shape != (c,):
        raise ValueError(f"{name} must be [{c}], got {tuple(w.shape)}")


def _args(x, delta, post, gate, scale, next_w, eps, n_dtype) -> _lib.Norm:
    """The C arguments but for the outputs, from contiguous tensors."""
    code = _lib.DTYPE_CODE
    c = x.shape[-1]
    b = x.shape[0] if x.dim() > 1 else 1
    a = _lib.Norm(b, x.numel() // max(1, b * c), c, x.data_ptr(), code[x.dtype])
    if delta is not None:
        a.delta, a.delta_dtype = delta.data_ptr(), code[delta.dtype]
        a.post_w, a.post_dtype = post.data_ptr(), code[post.dtype]
        if gate is not None:
            a.gate, a.gate_dtype = gate.data_ptr(), code[gate.dtype]
            a.gate_rows = 1 if gate.dim() == 1 else b
        if scale is not None:
            a.sample_scale = scale.data_ptr()
    if next_w is not None:
        a.next_w, a.next_dtype, a.n_dtype = next_w.data_ptr(), code[next_w.dtype], code[n_dtype]
    a.eps = eps
    return a


def _forward(x, delta, post, gate, scale, next_w, eps, n_dtype, keep):
    """(h or None, n or None, rstd of delta, rstd of h); the last two when ``keep``."""
    dev = x.device
    h = n = rd = rh = None
    if delta is not None:
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
    if next_w is not None:
        n = torch.empty(x.shape, dtype=n_dtype, device=dev)
    if x.numel():
        a = _args(x, delta, post, gate, scale, next_w, eps, n_dtype)
        if keep:
            rows = x.numel() // x.shape[-1]
            stats = torch.empty((2, rows), dtype=torch.float32, device=dev)
            rd, rh = stats[0], stats[1]
            a.rstd_delta, a.rstd_h = rd.data_ptr(), rh.data_ptr()
        a.h, a.n = _lib.ptr(h), _lib.ptr(n)
        with torch.cuda.device(dev):  # the library launches on the current device
            _lib.check(_lib.load().ow_norm_fwd(a, _lib.stream_handle(dev)), "ow_norm_fwd")
    return h, n, rd, rh


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, post, gate, scale, next_w, eps, n_dtype):
        h, n, rd, rh = _forward(x, delta, post, gate, scale, next_w, eps, n_dtype, True)
        ctx.save_for_backward(x, delta, post, gate, scale, next_w, rd, rh)
        ctx.eps, ctx.n_dtype = eps, n_dtype
        ctx.set_materialize_grads(False)
        if delta is None:
            return n
        return h if next_w is None else (h, n)

    @staticmethod
    def backward(ctx, *grads):
        x, delta, post, gate, scale, next_w, rd, rh = ctx.saved_tensors
        if delta is None:
            dh, dn = None, grads[0]
        else:
            dh, dn = grads[0], grads[1] if next_w is not None else None
        if dh is None and dn is None:
            return (None,) * 8
        dev = x.device
        dx = torch.empty_like(x)
        dd = None if delta is None else torch.empty_like(delta)
        dpost, dgate = (None if t is None else torch.empty_like(t) for t in (post, gate))
        used_next = next_w if dn is not None else None
        dnext = None if next_w is None else torch.empty_like(next_w) if dn is not None else torch.zeros_like(next_w)
        if x.numel() == 0:
            for t in (dpost, dgate, dnext):
                if t is not None:
                    t.zero_()
        else:
            dh, dn = (None if g is None else g.contiguous() for g in (dh, dn))
            a = _args(x, delta, post, gate, scale, used_next, ctx.eps, ctx.n_dtype)
            a.rstd_delta, a.rstd_h = rd.data_ptr(), rh.data_ptr()
            lib = _lib.load()
            with torch.cuda.device(dev):
                size = lib.ow_norm_bwd_workspace_size(a)
                ws = torch.empty(size, dtype=torch.uint8, device=dev)
                a.workspace, a.workspace_bytes = ws.data_ptr(), size
                g = _lib.NormGrads(_lib.ptr(dh), _lib.ptr(dn), dx.data_ptr(), _lib.ptr(dd), _lib.ptr(dpost),
                                   _lib.ptr(dgate), _lib.ptr(dnext if dn is not None else None))
                _lib.check(lib.ow_norm_bwd(a, g, _lib.stream_handle(dev)), "ow_norm_bwd")
            del ws
        return dx, dd, dpost, dgate, None, dnext, None, None


def _call(x, delta, post, gate, scale, next_w, eps, n_dtype):
    ts = [x, delta, post, gate, next_w]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        x, delta, post, gate, next_w = (None if t is None else t.contiguous() for t in ts)
        return _Norm.apply(x, delta, post, gate, scale, next_w, eps, n_dtype)
    x, delta, post, gate, next_w = (None if t is None else t.detach().contiguous() for t in ts)
    h, n, _, _ = _forward(x, delta, post, gate, scale, next_w, eps, n_dtype, False)
    return n if delta is None else h if next_w is None else (h, n)


def rms_norm(x: Tensor, weight: Tensor, *, eps: float = RMS_EPS, out_dtype: torch.dtype | None = None) -> Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last dimension.

    ``x`` is ``[..., C]`` in float32, bfloat16 or float16.  The result is in
    ``out_dtype``: by default the autocast type where autocast is on, else x's.
    Raises ``RuntimeError`` for what the kernels do not take.
    """
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., C], got {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    _vector("weight", weight, x.shape[-1])
    _require(x, weight)
    return _call(x, None, None, None, None, weight, float(eps), _out_dtype(x, out_dtype))


def norm_residual(x: Tensor, delta: Tensor, weight: Tensor, gate: Tensor | None = None, *,
                  sample_scale: Tensor | None = None, next_weight: Tensor | None = None,
                  eps: float = RMS_EPS, out_dtype: torch.dtype | None = None):
    """``h = x + sample_scale[b] * gate * rms(delta) * weight``, and the next block's ``rms(h) * next_weight``.

    ``x`` and ``delta`` are ``[B, ..., C]`` (each float32, bfloat16 or float16;
    ``h`` has x's type), ``weight`` and ``next_weight`` ``[C]``, ``gate`` ``[C]``,
    or ``[B, C]`` with one for each sample.  ``sample_scale`` ``[B]`` is the
    drop-path scale (``ops.drop_path_scale``); it takes no gradient.  Returns
    ``h``, or ``(h, n)`` with ``next_weight``; ``n`` is taken from the unrounded
    ``h`` and is in ``out_dtype`` (see ``rms_norm``).
    """
    if x.dim() < 2 or x.shape[-1] == 0:
        raise ValueError(f"x must be [B, ..., C], got {tuple(x.shape)}")
    if delta.shape != x.shape:
        raise ValueError(f"delta must be {tuple(x.shape)}, got {tuple(delta.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    b, c = x.shape[0], x.shape[-1]
    _vector("weight", weight, c)
    if next_weight is not None:
        _vector("next_weight", next_weight, c)
    if gate is not None and gate.shape not in ((c,), (b, c)):
        raise ValueError(f"gate must be [{c}] or [{b}, {c}], got {tuple(gate.shape)}")
    _require(x, delta, weight, gate, next_weight)
    if sample_scale is not None:
        if sample_scale.shape != (b,):
            raise ValueError(f"sample_scale must be [{b}], got {tuple(sample_scale.shape)}")
        if sample_scale.requires_grad:
            raise ValueError("sample_scale takes no gradient")
        if sample_scale.device != x.device:
            raise RuntimeError(f"norm not supported: tensors on {x.device} and {sample_scale.device}")
        sample_scale = sample_scale.to(torch.float32).contiguous()
    return _call(x, delta, weight, gate, sample_scale, next_weight, float(eps), _out_dtype(x, out_dtype))
