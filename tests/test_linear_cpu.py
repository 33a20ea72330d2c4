"""Linear with its epilogue (host side, no GPU): argument checks of the function and of the C entry points."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_b200 import _lib, linear


def test_refuses_host_tensors():
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    assert linear.linear_supported(x, w) == (False, "CUDA is unavailable")
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        linear.linear(x, w)


@pytest.mark.parametrize("call,match", [
    (lambda x, w: linear.linear(x, w, activation="tanh"), "activation"),
    (lambda x, w: linear.linear(x, w[0]), "weight must be"),
    (lambda x, w: linear.linear(x, torch.zeros(0, 8)), "weight must be"),
    (lambda x, w: linear.linear(x[:, :3], w), "x must be"),
    (lambda x, w: linear.linear(x, w, torch.zeros(8)), "bias must be"),
    (lambda x, w: linear.linear(x, w, residual=torch.zeros(2, 8)), "residual must be"),
])
def test_refuses_shapes(call, match):
    with pytest.raises(ValueError, match=match):
        call(torch.zeros(2, 8), torch.zeros(4, 8))


def _args(**over):
    a = _lib.Linear(100, 64, 40, 2, 1, 16, 64, 16, 64, 16, 0, 16, 40, 16, 16, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status,msg", [
    (dict(rows=-1), 1, "bad shape"),
    (dict(in_features=0), 1, "bad shape"),
    (dict(rows=1 << 31), 1, "too large"),
    (dict(dtype=0), 2, "bfloat16 or float16"),
    (dict(activation=4), 1, "unknown activation"),
    (dict(ldx=63), 1, "row stride"),
    (dict(ldw=63), 1, "row stride"),
    (dict(ldr=39), 1, "row stride"),
    (dict(bias_dtype=1), 1, "bias must be"),
    (dict(x=None), 1, "pointer is NULL"),
    (dict(weight=None), 1, "pointer is NULL"),
    (dict(out=None), 1, "pointer is NULL"),
    (dict(x=17), 1, "not aligned"),
    (dict(z=18), 1, "not aligned"),
    (dict(), 4, "workspace"),
])
def test_c_forward_refuses_before_any_cuda_call(over, status, msg):
    lib = _lib.load()
    assert lib.ow_linear_fwd(ctypes.byref(_args(**over)), None) == status
    assert msg in lib.ow_last_error().decode()


@pytest.mark.parametrize("over,grads,status,msg", [
    (dict(rows=0), {}, 1, "no rows"),
    (dict(z=None), {}, 1, "pointer is NULL"),
    (dict(x=None), {}, 1, "pointer is NULL"),
    (dict(weight=None), {}, 1, "pointer is NULL"),
    (dict(), dict(dout=None), 1, "pointer is NULL"),
    (dict(), dict(dweight_dtype=3), 2, "dweight must be"),
    (dict(), {}, 4, "workspace"),
])
def test_c_backward_refuses_before_any_cuda_call(over, grads, status, msg):
    lib = _lib.load()
    g = _lib.LinearGrads(16, 16, 16, 2, 16)
    for k, v in grads.items():
        setattr(g, k, v)
    assert lib.ow_linear_bwd(ctypes.byref(_args(**over)), ctypes.byref(g), None) == status
    assert msg in lib.ow_last_error().decode()


def test_workspace_covers_padded_operands():
    lib = _lib.load()
    plain = lib.ow_linear_workspace_size(_args(), None)
    odd = lib.ow_linear_workspace_size(_args(in_features=63, ldx=63, ldw=63), None)
    assert odd >= plain + 100 * 64 * 2 + 40 * 64 * 2  # x and weight in rows of 64
    assert lib.ow_linear_workspace_size(_args(rows=0), None) > 0
    assert lib.ow_linear_workspace_size(_args(dtype=0), None) == 0
    g = _lib.LinearGrads(16, 16, 16, 2, 16)
    assert lib.ow_linear_workspace_size(_args(), g) >= 100 * 40 * 2  # dz


@pytest.mark.parametrize("over,grads", [
    (dict(bias=17), None), (dict(z=8), {}), (dict(x=17), {}), ({}, dict(dout=17)), ({}, dict(dx=17)), ({}, dict(dweight=17)),
    ({}, dict(dweight=18, dweight_dtype=0)), ({}, dict(dbias=17)),
])
def test_c_entries_refuse_pointers_off_their_alignment(over, grads):
    lib = _lib.load()
    if grads is None:
        status = lib.ow_linear_fwd(ctypes.byref(_args(**over)), None)
    else:
        g = _lib.LinearGrads(16, 16, 16, 2, 16)
        for k, v in grads.items():
            setattr(g, k, v)
        status = lib.ow_linear_bwd(ctypes.byref(_args(**over)), ctypes.byref(g), None)
    assert status == 1 and "not aligned" in lib.ow_last_error().decode()


def test_refuses_features_that_their_field_does_not_hold():
    k = 2 ** 32 + 8  # 8 in 32 bits
    with pytest.raises(ValueError, match="too large"):
        linear.linear(torch.zeros(1, 1).expand(1, k), torch.zeros(1, 1).expand(2, k))
    with pytest.raises(ValueError, match="too large"):
        linear.linear(torch.zeros(1, 8), torch.zeros(1, 8).expand(k, 8))


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
def test_refuses_forward_mode(which):
    """A tangent would be dropped: there is no formula for it here."""
    import torch.autograd.forward_ad as fw

    t = {"x": torch.zeros(2, 8), "weight": torch.zeros(4, 8), "bias": torch.zeros(4), "residual": torch.zeros(2, 4)}
    with fw.dual_level():
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear.linear(t["x"], t["weight"], t["bias"], residual=t["residual"])
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            linear.linear(t["x"], t["weight"], t["bias"], residual=t["residual"])


@pytest.mark.parametrize("n", [4095, 4089])
def test_backward_workspace_has_no_copies_that_are_not_made(n):
    """dz is made in rows that TMA reads, so an odd width asks for no more than the next multiple of 8 does."""
    lib = _lib.load()
    g = _lib.LinearGrads(16, 16, 16, 2, 16)
    kw = dict(rows=32768, in_features=4096, activation=3, ldx=4096, ldw=4096, residual=None)
    even = lib.ow_linear_workspace_size(_args(out_features=4096, **kw), g)
    odd = lib.ow_linear_workspace_size(_args(out_features=n, **kw), g)
    assert 32768 * 4096 * 2 <= odd <= even + 4096
    # without an activation dy itself is read: where its rows are no 16-byte units it is copied once, as dz
    plain = lib.ow_linear_workspace_size(_args(out_features=n, **(kw | dict(activation=0))), g)
    assert plain == odd
