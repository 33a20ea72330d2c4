"""AdamW over many tensors (host side, no GPU): argument checks of the optimizer and of its C entry points."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_b200 import _lib, optim
from omniwave_b200.train import TrainStep


def test_refuses_host_parameters():
    p = torch.nn.Parameter(torch.zeros(4))
    assert optim.adamw_supported(p) == (False, "CUDA is unavailable")
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        optim.AdamW([p])
    with pytest.raises(ValueError, match="max_norm"):
        optim.AdamW([p], max_norm=0.0)


@pytest.mark.parametrize("kw,match", [
    (dict(lr=-1.0), "learning rate"),
    (dict(betas=(1.0, 0.9)), "betas"),
    (dict(betas=(0.9, -0.1)), "betas"),
    (dict(eps=-1e-8), "eps"),
    (dict(weight_decay=-0.1), "weight_decay"),
    (dict(state_bits=16), "state_bits"),
    (dict(lr=torch.zeros(2)), "tensor lr"),
    (dict(lr=torch.zeros((), dtype=torch.float64)), "tensor lr"),
])
def test_refuses_hyperparameters(kw, match):
    group = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, state_bits=32) | kw
    with pytest.raises(ValueError, match=match):
        optim.AdamW._check_hyper(group, torch.device("cpu"))


@pytest.mark.parametrize("make,dense", [
    (lambda: torch.zeros(3, 4), True),
    (lambda: torch.zeros(3, 4).t(), True),
    (lambda: torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last), True),
    (lambda: torch.zeros(()), True),
    (lambda: torch.zeros(5, 1, 2), True),
    (lambda: torch.zeros(3, 4)[:, :2], False),
    (lambda: torch.zeros(4)[::2], False),
    (lambda: torch.zeros(1).expand(3), False),
])
def test_dense_parameters_are_told_from_others(make, dense):
    assert optim._dense(make()) is dense


def test_train_step_refuses_unknown_optimizers():
    m = torch.nn.Linear(2, 2)
    with pytest.raises(ValueError, match="optimizer"):
        TrainStep(m, optimizer="sgd")
    with pytest.raises(ValueError, match="state_bits"):
        TrainStep(m, state_bits=8)
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        TrainStep(m, optimizer="fused")


def _args(**over):
    keep = [(ctypes.c_void_p * 2)(16, 16), (ctypes.c_void_p * 2)(16, None), (ctypes.c_int64 * 3)(0, 256, 1024)]
    a = _lib.AdamW(2, 0, *[ctypes.addressof(k) for k in keep], 16, 16, 32, 16, 16, None, None, 16,
                   1e-3, 0.9, 0.999, 1e-8, 0.0, None, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a, keep


@pytest.mark.parametrize("over,status,msg", [
    (dict(tensors=0), 1, "tensors must be positive"),
    (dict(params=None), 1, "NULL"),
    (dict(dev_blocks=None), 1, "device table"),
    (dict(control=None), 1, "device table"),
    (dict(dtype=1), 2, "float32, bfloat16 or float16"),
    (dict(state_bits=4), 1, "state_bits"),
    (dict(exp_avg=None), 1, "state pointer"),
    (dict(state_bits=8), 1, "need their scales"),
    (dict(beta1=1.0), 1, "betas"),
])
def test_c_entry_refuses_before_any_cuda_call(over, status, msg):
    lib = _lib.load()
    a, keep = _args(**over)
    assert lib.ow_adamw_step(a, None) == status
    assert msg in lib.ow_last_error().decode()
    del keep


def test_c_entry_checks_slots_and_partials():
    lib = _lib.load()
    a, keep = _args()
    keep[2][1] = 100  # not a multiple of the block
    assert lib.ow_adamw_step(a, None) == 1 and "multiple of 256" in lib.ow_last_error().decode()
    keep[2][1] = 1024  # the second tensor has no slot
    assert lib.ow_adamw_step(a, None) == 1
    keep[2][1] = 256
    need = lib.ow_grad_norm_partials(a)
    assert need >= 1
    opt = _lib.GradNorm(16, 0, need - 1, 1, 1.0, 0, None, None)
    assert lib.ow_grad_norm(a, opt, None) == 1 and "partial sums" in lib.ow_last_error().decode()
    opt = _lib.GradNorm(None, 0, need, 1, 1.0, 0, None, None)
    assert lib.ow_grad_norm(a, opt, None) == 1
    assert lib.ow_grad_norm_partials(None) == 0


@pytest.mark.parametrize("over", [
    dict(dev_blocks=24), dict(control=18), dict(exp_avg=24), dict(exp_avg_sq=20), dict(dev_steps=18), dict(lr_ptr=18),
    dict(found=18), dict(state_bits=8, exp_avg=18, exp_avg_scale=16, exp_avg_sq_scale=16),
    dict(state_bits=8, exp_avg_scale=18, exp_avg_sq_scale=16),
])
def test_c_entry_refuses_pointers_off_their_alignment(over):
    lib = _lib.load()
    a, keep = _args(**over)
    assert lib.ow_adamw_step(a, None) == 1
    assert "not aligned" in lib.ow_last_error().decode()
    a, keep = _args()
    for which in (0, 1):
        keep[which][0] = 18  # f32
        assert lib.ow_adamw_step(a, None) == 1 and "tensor 0 is not aligned" in lib.ow_last_error().decode()
        keep[which][0] = 16
    for bad in (dict(partials=20), dict(norm=18), dict(found=18)):
        opt = _lib.GradNorm(16, 0, 1000, 1, 1.0, 0, None, None)
        for k, v in bad.items():
            setattr(opt, k, v)
        assert lib.ow_grad_norm(a, opt, None) == 1 and "not aligned" in lib.ow_last_error().decode()


def test_8bit_moments_need_a_positive_eps():
    """Both moments may be held as 0, where a step is 0 / eps."""
    group = dict(lr=1e-3, betas=(0.9, 0.999), eps=0.0, weight_decay=0.0, state_bits=32)
    optim.AdamW._check_hyper(group, torch.device("cpu"))
    lib = _lib.load()
    for eps in (0.0, 1e-60):  # 0 in f32
        with pytest.raises(ValueError, match="positive eps"):
            optim.AdamW._check_hyper(group | dict(state_bits=8, eps=eps), torch.device("cpu"))
        a, keep = _args(state_bits=8, exp_avg_scale=16, exp_avg_sq_scale=16, eps=eps)
        assert lib.ow_adamw_step(a, None) == 1 and "positive eps" in lib.ow_last_error().decode()
        del keep
