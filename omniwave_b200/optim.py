"""AdamW over many tensors at once on the B200 kernels, moments in 32 or 8 bits.

``AdamW`` takes the place of the ``torch.optim.AdamW`` of the reference's
training engine (omniweave/training/engine.py:411) together with what that
engine does to the gradients in front of it: the finite check of every
gradient (:229-240) and ``clip_grad_norm_`` (:243-244).  A step is one kernel
over all tensors of a parameter group, and one more that takes the norm when
the gradients are clipped or checked; nothing waits for the GPU.

    p <- p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

Everything is computed in f32 and a parameter is rounded once to its own
dtype (f32, bf16 or f16).  ``state_bits=8`` holds the moments as e4m3 with one
f32 scale for 256 elements, rounded stochastically by a hash of the
element's place and the step, so a run repeats bit for bit.

The state lives in flat buffers (``AdamW.buffers``); ``state[p]`` holds views of
them in ``p``'s shape under the names ``torch.optim.AdamW`` uses, so its
checkpoints load here (and, with 32 bits, this one's load there), those of 16-bit
parameters too, whose moments torch holds in the parameter's type.
"""

from __future__ import annotations

import copy
import ctypes
from typing import Any

import torch
from torch import Tensor

from omniwave_b200 import _lib

__all__ = ["AdamW", "adamw_supported"]

BLOCK = _lib.ADAMW_BLOCK
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
# of a checkpoint's groups: what says which parameters they are and how they are held, and choices of torch's own code
_NOT_LOADED = ("params", "param_names", "state_bits", "amsgrad", "maximize", "foreach", "capturable", "differentiable",
               "fused", "decoupled_weight_decay")


def _dense(p: Tensor) -> bool:
    """Whether ``p`` covers a run of memory with each element in a place of its own."""
    at = 1
    for stride, size in sorted((st, sz) for sz, st in zip(p.shape, p.stride()) if sz != 1):
        if stride != at:
            return False
        at *= size
    return True


def adamw_supported(p: Tensor) -> tuple[bool, str | None]:
    """``(is_supported, reason_if_not)`` for a parameter of ``AdamW``."""
    if p.device.type != "cuda":
        return False, "CUDA is unavailable"
    if p.layout != torch.strided or p.is_complex() or p.dtype not in _DTYPES:
        return False, f"unsupported dtype or layout {p.dtype}, {p.layout}"
    if not _dense(p):
        return False, "the parameter's elements do not lie densely in memory"
    try:
        lib = _lib.load()
    except _lib.NativeLibraryError as exc:
        return False, str(exc)
    if not lib.ow_device_supported(p.device.index):
        return False, f"device {p.device.index} is not sm_100 (B200-class)"
    return True, None


class _Bucket:
    """The parameters of one group that share a dtype, and their flat state."""

    def __init__(self, group: dict[str, Any], params: list[Tensor], bits: int) -> None:
        self.group, self.params, self.bits = group, params, bits
        dev = self.device = params[0].device
        self.dtype = params[0].dtype
        slots, total = [0], 0
        for p in params:
            total += -(-p.numel() // BLOCK) * BLOCK
            slots.append(total)
        self.slots = slots
        blocks = total // BLOCK
        self._slots = (ctypes.c_int64 * len(slots))(*slots)
        # one record for each block: its tensor, its place in the tensor, its elements in use
        numel = torch.tensor([p.numel() for p in params])
        first = torch.tensor(slots[:-1]) // BLOCK
        counts = torch.tensor(slots[1:]) // BLOCK - first
        tensor = torch.repeat_interleave(torch.arange(len(params)), counts)
        place = torch.arange(blocks) - first[tensor]
        used = (numel[tensor] - place * BLOCK).clamp(max=BLOCK)
        self.blocks = torch.stack([tensor, place, used, torch.zeros_like(used)], 1).to(torch.int32).to(dev)
        self.control = torch.zeros(_lib.ADAMW_CONTROL_BYTES, dtype=torch.uint8, device=dev)
        state = torch.float32 if bits == 32 else torch.float8_e4m3fn
        self.held: dict[str, Tensor] = {
            "step": torch.zeros(len(params), dtype=torch.float32, device=dev),
            "exp_avg": torch.zeros(total, dtype=torch.float32 if bits == 32 else torch.uint8, device=dev).view(state),
            "exp_avg_sq": torch.zeros(total, dtype=torch.float32 if bits == 32 else torch.uint8, device=dev).view(state),
        }
        if bits == 8:
            self.held["exp_avg_scale"] = torch.zeros(blocks, dtype=torch.float32, device=dev)
            self.held["exp_avg_sq_scale"] = torch.zeros(blocks, dtype=torch.float32, device=dev)
        h = self.held
        n = len(params)
        self._p, self._g = (ctypes.c_void_p * n)(), (ctypes.c_void_p * n)()
        self.args = _lib.AdamW(
            n, _lib.DTYPE_CODE[self.dtype], ctypes.addressof(self._p), ctypes.addressof(self._g),
            ctypes.addressof(self._slots), self.blocks.data_ptr(), self.control.data_ptr(), bits, h["exp_avg"].data_ptr(),
            h["exp_avg_sq"].data_ptr(), _lib.ptr(h.get("exp_avg_scale")), _lib.ptr(h.get("exp_avg_sq_scale")),
            h["step"].data_ptr())
        self.native = _lib.host().Bucket(params, ctypes.addressof(self.args), ctypes.addressof(self._p),
                                         ctypes.addressof(self._g))

    def views(self, i: int) -> dict[str, Tensor]:
        """Parameter i's share of the state, in its shape."""
        p, o, h = self.params[i], self.slots[i], self.held
        out = {"step": h["step"][i]}
        for k in ("exp_avg", "exp_avg_sq"):
            out[k] = torch.as_strided(h[k], p.shape, p.stride(), o)
        if self.bits == 8:
            for k in ("exp_avg_scale", "exp_avg_sq_scale"):
                out[k] = h[k][o // BLOCK:self.slots[i + 1] // BLOCK]
        return out


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay over all parameters at once.

    ``lr`` is a number, or a float32 tensor of one element on the parameters'
    device, which the kernel reads when it runs (so a captured step follows a
    schedule).  ``state_bits`` is 32 or 8 (also as a parameter group's own
    option); 8 needs a positive ``eps``.  ``max_norm`` clips the gradients by their global norm, as
    ``clip_grad_norm_`` does but without writing them; ``skip_nonfinite`` leaves
    parameters and state untouched in a step whose gradients hold an inf or a
    NaN.  With either, ``grad_norm`` is the norm of the last step, on the
    device.  ``step(found_inf=...)`` takes a float32 device flag: nonzero calls
    the step off, and ``skip_nonfinite`` sets it.

    Parameters are float32, bfloat16 or float16 on one B200, dense in memory;
    others raise ``RuntimeError``.  A parameter without a gradient takes no step.
    """

    def __init__(self, params, lr: float | Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 max_norm: float | None = None, skip_nonfinite: bool = False) -> None:
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        self.max_norm = max_norm
        self.skip_nonfinite = bool(skip_nonfinite)
        self._buckets: list[_Bucket] = []
        self._partials: Tensor | None = None
        self._replaced: list[Tensor | None] = []
        self.grad_norm: Tensor | None = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    # ------------------------------------------------------------ construction
    @staticmethod
    def _check_hyper(group: dict[str, Any], device: torch.device) -> None:
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32 or lr.device != device:
                raise ValueError("a tensor lr must be one float32 on the parameters' device")
        elif not lr >= 0.0:
            raise ValueError(f"invalid learning rate: {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be in [0, 1), got {group['betas']}")
        if not group["eps"] >= 0.0:
            raise ValueError(f"invalid eps: {group['eps']}")
        if not group["weight_decay"] >= 0.0:
            raise ValueError(f"invalid weight_decay: {group['weight_decay']}")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {group['state_bits']}")
        if group["state_bits"] == 8 and not ctypes.c_float(group["eps"]).value > 0.0:
            raise ValueError(f"8-bit moments need a positive eps (both may be held as 0), got {group['eps']}")

    def add_param_group(self, param_group: dict[str, Any]) -> None:
        super().add_param_group(param_group)
        try:
            self._add_buckets(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    def _add_buckets(self, group: dict[str, Any]) -> None:
        params = group["params"]
        if not params:
            return
        if len({id(p) for p in params}) != len(params):
            raise ValueError("a parameter appears more than once in a group")
        for p in params:
            ok, why = adamw_supported(p)
            if not ok:
                raise RuntimeError(f"AdamW not supported: {why}")
        device = self._buckets[0].device if self._buckets else params[0].device
        if any(p.device != device for p in params):
            raise ValueError("all parameters must be on one device")
        self._check_hyper(group, device)
        by_dtype: dict[torch.dtype, list[Tensor]] = {}
        for p in params:
            if p.numel():
                by_dtype.setdefault(p.dtype, []).append(p)
        made = [_Bucket(group, ps, group["state_bits"]) for ps in by_dtype.values()]  # all of them, or none
        self._buckets += made
        for b in made:
            for i, p in enumerate(b.params):
                self.state[p] = b.views(i)
        self._norm_buffers()

    def _norm_buffers(self) -> None:
        if self._buckets and (self.max_norm is not None or self.skip_nonfinite):
            dev = self._buckets[0].device
            need = sum(b.native.partials for b in self._buckets)
            if self._partials is None or self._partials.numel() < need:
                # a step that was captured before writes to the sums of its day for as long as it is replayed
                self._replaced.append(self._partials)
                self._partials = torch.empty(need, dtype=torch.float64, device=dev)
            if self.grad_norm is None:
                self.grad_norm = torch.zeros((), dtype=torch.float32, device=dev)

    @property
    def buffers(self) -> list[dict[str, Tensor]]:
        """The flat state, a dict for each parameter group and dtype: ``step``, ``exp_avg``,
        ``exp_avg_sq`` (each tensor from the next multiple of 256 slots on) and, with 8 bits,
        ``exp_avg_scale`` and ``exp_avg_sq_scale`` (one for 256 slots)."""
        return [b.held for b in self._buckets]

    # ------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None, *, found_inf: Tensor | None = None):
        """One step on the gradients at hand; nothing waits for the GPU."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if not self._buckets:
            return loss
        norm = self.max_norm is not None or self.skip_nonfinite
        if norm and self._partials is None:  # asked for since the parameters were added
            self._norm_buffers()
        hyper = [(g["lr"], g["betas"], g["eps"], g["weight_decay"]) for g in (b.group for b in self._buckets)]
        _lib.host().adamw_step([b.native for b in self._buckets], hyper, found_inf, self._partials if norm else None,
                               self.grad_norm, self.max_norm or 0.0, self.skip_nonfinite)
        return loss

    # ------------------------------------------------------------ checkpoints
    @torch.no_grad()
    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        """Copy a checkpoint's values into the state, which must be held in as many bits.

        A parameter that the checkpoint has no state for starts anew, as with torch's.
        A checkpoint of another rule (``maximize``, ``amsgrad``, decay that is not
        decoupled) raises ``ValueError``, and nothing is changed.
        """
        state_dict = state_dict.copy()
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        groups, saved = self.param_groups, state_dict["param_groups"]
        if len(groups) != len(saved):
            raise ValueError("loaded state dict has a different number of parameter groups")
        if any(len(g["params"]) != len(s["params"]) for g, s in zip(groups, saved)):
            raise ValueError("loaded state dict contains a parameter group that doesn't match the size of optimizer's group")
        for s in saved:
            for rule in ("maximize", "amsgrad"):
                if s.get(rule):
                    raise ValueError(f"loaded state is of an optimizer with {rule}, which this one does not do")
            if not s.get("decoupled_weight_decay", True) and s.get("weight_decay"):
                raise ValueError("loaded state is of an optimizer whose weight decay is not decoupled from the gradient")
        moves = []
        for g, s in zip(groups, saved):
            for p, key in zip(g["params"], s["params"]):
                mine, theirs = self.state.get(p, {}), state_dict["state"].get(key, {})
                if not mine:
                    continue
                if theirs and set(theirs) != set(mine):
                    raise ValueError(f"loaded state holds {sorted(theirs)}, this optimizer {sorted(mine)}: "
                                     f"state_bits differ, or it is another optimizer's")
                for k, t in mine.items():
                    v = theirs.get(k)
                    if v is None:
                        moves.append((t, None))
                        continue
                    v = torch.as_tensor(v)
                    # 32-bit moments take any of torch's (it holds a 16-bit parameter's in 16 bits); codes are codes
                    wide = k in ("exp_avg", "exp_avg_sq") and t.dtype == torch.float32
                    fits = k == "step" or v.dtype == t.dtype or (wide and v.dtype in (*_DTYPES, torch.float64))
                    if v.shape != t.shape or not fits:
                        raise ValueError(f"loaded {k} is {v.dtype} {tuple(v.shape)}, expected {t.dtype} {tuple(t.shape)}")
                    moves.append((t, v))
        for t, v in moves:
            if t.dtype == torch.float8_e4m3fn:
                t, v = t.view(torch.uint8), None if v is None else v.view(torch.uint8)
            t.zero_() if v is None else t.copy_(v)
        for g, s in zip(groups, saved):
            new = {k: copy.deepcopy(v) for k, v in s.items() if k not in _NOT_LOADED}  # a scheduler's entries too
            lr = new.pop("lr", g["lr"])
            if isinstance(g["lr"], Tensor) and g["params"]:
                g["lr"].copy_(torch.as_tensor(lr))  # a captured step reads this tensor
            else:
                g["lr"] = float(lr) if isinstance(lr, Tensor) else lr
            g.update({k: tuple(v) if k == "betas" else v for k, v in new.items()})
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def __getstate__(self) -> dict[str, Any]:
        return {**super().__getstate__(), "max_norm": self.max_norm, "skip_nonfinite": self.skip_nonfinite}

    @torch.no_grad()
    def __setstate__(self, state: dict[str, Any]) -> None:
        """Rebuild the flat buffers around the values of a copied or unpickled optimizer."""
        super().__setstate__(state)
        old, self.state = self.state, type(self.state)(dict)
        self._buckets, self._partials, self._replaced, self.grad_norm = [], None, [], None
        for g in self.param_groups:
            self._add_buckets(g)
        for p, mine in self.state.items():
            for k, t in mine.items():
                v = old[p][k]
                if t.dtype == torch.float8_e4m3fn:
                    t, v = t.view(torch.uint8), v.view(torch.uint8)
                t.copy_(v)
