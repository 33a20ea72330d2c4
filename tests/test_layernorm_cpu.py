"""Layer norm (host side, no GPU): argument checks of the function and of the C entry points."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_b200 import _lib, norm


def test_refuses_host_tensors():
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        norm.layer_norm(torch.zeros(2, 8), torch.zeros(8), torch.zeros(8))


@pytest.mark.parametrize("call,match", [
    (lambda x, w: norm.layer_norm(torch.zeros(()), w), "x must be"),
    (lambda x, w: norm.layer_norm(torch.zeros(2, 0), w), "x must be"),
    (lambda x, w: norm.layer_norm(x, w[:4]), "weight must be"),
    (lambda x, w: norm.layer_norm(x, w, w[:4]), "bias must be"),
    (lambda x, w: norm.layer_norm(x, w[None]), "weight must be"),
    (lambda x, w: norm.layer_norm(x, w, eps=-1.0), "eps"),
    (lambda x, w: norm.layer_norm(torch.zeros(1, 1).expand(1, 2 ** 32 + 8), w), "too many channels"),
])
def test_refuses_shapes(call, match):
    with pytest.raises(ValueError, match=match):
        call(torch.zeros(2, 8), torch.zeros(8))


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
def test_refuses_forward_mode(which):
    import torch.autograd.forward_ad as fw

    t = {"x": torch.zeros(2, 8), "weight": torch.zeros(8), "bias": torch.zeros(8)}
    with fw.dual_level():
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            norm.layer_norm(t["x"], t["weight"], t["bias"])


def _args(**over):
    a = _lib.LayerNorm(100, 64, 16, 2, 16, 0, 16, 0, 1e-5, 16, 2, 16, 16, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status,msg", [
    (dict(rows=-1), 1, "bad shape"),
    (dict(channels=0), 1, "bad shape"),
    (dict(channels=1 << 30), 1, "bad shape"),
    (dict(x_dtype=1), 2, "float32"),
    (dict(weight_dtype=7), 2, "float32"),
    (dict(bias_dtype=1), 2, "float32"),
    (dict(n_dtype=1), 2, "float32"),
    (dict(eps=-1.0), 1, "eps"),
    (dict(x=None), 1, "pointer is NULL"),
    (dict(weight=None), 1, "pointer is NULL"),
    (dict(n=None), 1, "pointer is NULL"),
    (dict(mean=None), 1, "pointer is NULL"),
    (dict(x=17), 1, "not aligned"),
    (dict(weight=18), 1, "not aligned"),
    (dict(bias=18), 1, "not aligned"),
    (dict(n=17), 1, "not aligned"),
    (dict(rstd=18), 1, "not aligned"),
])
def test_c_forward_refuses_before_any_cuda_call(over, status, msg):
    lib = _lib.load()
    assert lib.ow_layernorm_fwd(ctypes.byref(_args(**over)), None) == status
    assert msg in lib.ow_last_error().decode()


@pytest.mark.parametrize("over,grads,status,msg", [
    (dict(rows=0), {}, 1, "no rows"),
    (dict(rstd=None), {}, 1, "pointer is NULL"),
    ({}, dict(dn=None), 1, "pointer is NULL"),
    ({}, dict(dn=17), 1, "not aligned"),
    ({}, dict(dx=17), 1, "not aligned"),
    ({}, dict(dweight=18), 1, "not aligned"),
    ({}, dict(dbias=18), 1, "not aligned"),
    (dict(bias=None, bias_dtype=9), {}, 1, "bias_dtype"),
    ({}, {}, 4, "workspace"),
])
def test_c_backward_refuses_before_any_cuda_call(over, grads, status, msg):
    lib = _lib.load()
    g = _lib.LayerNormGrads(16, 16, 16, 16)
    for k, v in grads.items():
        setattr(g, k, v)
    assert lib.ow_layernorm_bwd(ctypes.byref(_args(**over)), ctypes.byref(g), None) == status
    assert msg in lib.ow_last_error().decode()


def test_no_rows_is_no_work():
    lib = _lib.load()
    assert lib.ow_layernorm_fwd(ctypes.byref(_args(rows=0, x=None, n=None)), None) == 0
    assert lib.ow_layernorm_bwd_workspace_size(ctypes.byref(_args(x_dtype=1))) == 0
    assert lib.ow_layernorm_bwd_workspace_size(ctypes.byref(_args(rows=0))) > 0
