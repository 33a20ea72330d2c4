"""Distillation loss (host side, no GPU): argument checks, and the training step that calls it."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_b200 import _lib, loss
from omniwave_b200.train import TrainStep


def _call(**over):
    a = dict(logits=torch.zeros(4, 10), top_logits=torch.zeros(4, 3), top_classes=torch.zeros(4, 3, dtype=torch.int64),
             labels=torch.zeros(4, dtype=torch.int64))
    kw = {k: over.pop(k) for k in list(over) if k in ("temperature", "weight", "reduction")}
    a.update(over)
    return loss.distill_loss(*a.values(), **kw)


def test_refuses_host_tensors():
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        _call()


@pytest.mark.parametrize("over,match", [
    (dict(logits=torch.zeros(())), "logits must be"),
    (dict(logits=torch.zeros(4, 0)), "logits must be"),
    (dict(top_logits=torch.zeros(3, 3)), "top_logits must be"),
    (dict(top_logits=torch.zeros(4)), "top_logits must be"),
    (dict(top_logits=torch.zeros(4, 0)), "top_logits must be"),
    (dict(top_classes=torch.zeros(4, 2, dtype=torch.int64)), "top_classes must be"),
    (dict(top_classes=torch.zeros(4, 3)), "int32 or int64"),
    (dict(top_classes=torch.zeros(4, 3, dtype=torch.int16)), "int32 or int64"),
    (dict(labels=torch.zeros(3, dtype=torch.int64)), "labels must be"),
    (dict(labels=torch.zeros(4, 1, dtype=torch.int64)), "labels must be"),
    (dict(labels=torch.zeros(4)), "int32 or int64"),
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
    (dict(weight=-0.1), "weight"),
    (dict(weight=1.5), "weight"),
    (dict(weight=float("nan")), "weight"),
    (dict(reduction="batchmean"), "reduction"),
    (dict(top_logits=torch.zeros(4, 3, requires_grad=True)), "no gradient"),
    (dict(logits=torch.zeros(4, 1).expand(4, 2 ** 32 + 1)), "too many classes"),
])
def test_refuses_shapes_and_values(over, match):
    with pytest.raises(ValueError, match=match):
        _call(**over)


@pytest.mark.parametrize("which", ["logits", "top_logits"])
def test_refuses_forward_mode(which):
    import torch.autograd.forward_ad as fw

    with fw.dual_level():
        t = torch.zeros(4, 10 if which == "logits" else 3)
        with pytest.raises(RuntimeError, match="forward-mode"):
            _call(**{which: fw.make_dual(t, torch.ones_like(t))})


def _args(**over):
    a = _lib.Distill(100, 64, 8, 16, 2, 64, 16, 3, 16, 4, 16, 8, 2.0, 0.5, 1, 16, 16, 16, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


BAD = [
    (dict(rows=-1), 1, "bad shape"),
    (dict(classes=0), 1, "bad shape"),
    (dict(top=0), 1, "bad shape"),
    (dict(top=1025), 2, "at most"),
    (dict(ld=63), 1, "row stride"),
    (dict(dtype=1), 2, "float32"),
    (dict(top_dtype=1), 2, "float32"),
    (dict(class_bytes=2), 1, "integers"),
    (dict(label_bytes=1), 1, "integers"),
    (dict(temperature=0.0), 1, "temperature"),
    (dict(weight=2.0), 1, "weight"),
    (dict(reduction=3), 1, "reduction"),
    (dict(logits=None), 1, "pointer is NULL"),
    (dict(top_logits=None), 1, "pointer is NULL"),
    (dict(top_classes=None), 1, "pointer is NULL"),
    (dict(stats=None), 1, "pointer is NULL"),
    (dict(factors=None), 1, "pointer is NULL"),
    (dict(logits=17), 1, "not aligned"),
    (dict(top_logits=17), 1, "not aligned"),
    (dict(top_classes=18), 1, "not aligned"),
    (dict(labels=20), 1, "not aligned"),
    (dict(stats=18), 1, "not aligned"),
]


@pytest.mark.parametrize("over,status,msg", BAD + [(dict(loss=None), 1, "pointer is NULL"), ({}, 4, "workspace")])
def test_c_forward_refuses_before_any_cuda_call(over, status, msg):
    lib = _lib.load()
    assert lib.ow_distill_fwd(ctypes.byref(_args(**over)), None) == status
    assert msg in lib.ow_last_error().decode()


@pytest.mark.parametrize("over,grads,status,msg", [(o, {}, s, m) for o, s, m in BAD] + [
    ({}, dict(dloss=None), 1, "pointer is NULL"),
    ({}, dict(dlogits=None), 1, "pointer is NULL"),
    ({}, dict(dloss=18), 1, "not aligned"),
    ({}, dict(dlogits=17), 1, "not aligned"),
])
def test_c_backward_refuses_before_any_cuda_call(over, grads, status, msg):
    lib = _lib.load()
    g = _lib.DistillGrads(16, 16)
    for k, v in grads.items():
        setattr(g, k, v)
    assert lib.ow_distill_bwd(ctypes.byref(_args(**over)), ctypes.byref(g), None) == status
    assert msg in lib.ow_last_error().decode()


def test_no_rows_is_no_work():
    lib = _lib.load()
    assert lib.ow_distill_fwd(ctypes.byref(_args(rows=0, logits=None)), None) == 0
    assert lib.ow_distill_workspace_size(ctypes.byref(_args(dtype=1))) == 0


def test_training_step_without_a_teacher_is_as_before_and_with_one_needs_the_gpu():
    torch.manual_seed(0)
    model = torch.nn.Linear(6, 5)
    step = TrainStep(model, distill_weight=0.7, distill_temperature=2.0)
    x, y = torch.randn(4, 6), torch.tensor([0, 1, 2, 3])
    want = torch.nn.functional.cross_entropy(model(x), y)
    assert torch.equal(step.step(x, y), want.detach())
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        step.step(x, y, teacher=(torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64)))
    with pytest.raises(ValueError, match="distill_weight"):
        TrainStep(model, distill_weight=1.5)
    with pytest.raises(ValueError, match="distill_temperature"):
        TrainStep(model, distill_temperature=0.0)
