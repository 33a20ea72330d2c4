"""Gated feed-forward block (host side, no GPU): argument checks of the function and of the C entry points."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_b200 import _lib, feed_forward

BF = torch.bfloat16


def _call(**over):
    a = dict(x=torch.zeros(2, 8), gate_weight=torch.zeros(4, 8), up_weight=torch.zeros(4, 8), down_weight=torch.zeros(6, 4))
    kw = {k: over.pop(k) for k in list(over) if k not in a}
    a.update(over)
    return feed_forward.gated_feed_forward(*a.values(), **kw)


def test_refuses_host_tensors():
    t = [torch.zeros(2, 8, dtype=BF), torch.zeros(4, 8, dtype=BF), torch.zeros(4, 8, dtype=BF), torch.zeros(6, 4, dtype=BF)]
    assert feed_forward.gated_feed_forward_supported(*t) == (False, "CUDA is unavailable")
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        feed_forward.gated_feed_forward(*t)


@pytest.mark.parametrize("over,match", [
    (dict(activation="tanh"), "activation"),
    (dict(gate_weight=torch.zeros(8)), "gate_weight must be"),
    (dict(gate_weight=torch.zeros(0, 8)), "gate_weight must be"),
    (dict(up_weight=torch.zeros(5, 8)), "up_weight must be"),
    (dict(up_weight=torch.zeros(4, 7)), "up_weight must be"),
    (dict(down_weight=torch.zeros(6, 5)), "down_weight must be"),
    (dict(down_weight=torch.zeros(0, 4)), "down_weight must be"),
    (dict(x=torch.zeros(2, 7)), "x must be"),
    (dict(x=torch.zeros(())), "x must be"),
    (dict(gate_bias=torch.zeros(6)), "gate_bias must be"),
    (dict(up_bias=torch.zeros(1, 4)), "up_bias must be"),
    (dict(down_bias=torch.zeros(4)), "down_bias must be"),
    (dict(residual=torch.zeros(2, 8)), "residual must be"),
    (dict(down_weight=torch.zeros(1, 4).expand(2 ** 32 + 8, 4)), "too large"),
])
def test_refuses_shapes(over, match):
    with pytest.raises(ValueError, match=match):
        _call(**over)


@pytest.mark.parametrize("which", ["x", "gate_weight", "up_weight", "down_weight", "gate_bias", "up_bias", "down_bias", "residual"])
def test_refuses_forward_mode(which):
    import torch.autograd.forward_ad as fw

    t = dict(x=torch.zeros(2, 8), gate_weight=torch.zeros(4, 8), up_weight=torch.zeros(4, 8), down_weight=torch.zeros(6, 4),
             gate_bias=torch.zeros(4), up_bias=torch.zeros(4), down_bias=torch.zeros(6), residual=torch.zeros(2, 6))
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            _call(**{which: fw.make_dual(t[which], torch.ones_like(t[which]))})


def _args(**over):
    a = _lib.Ffn(100, 64, 40, 48, 2, 2, 16, 64, 16, 64, 16, 64, 16, 40, 16, 0, 16, 0, 16, 0, 16, 48, 16, 16, 16, 16, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


BAD = [
    (dict(rows=-1), 1, "bad shape"),
    (dict(in_features=0), 1, "bad shape"),
    (dict(hidden=0), 1, "bad shape"),
    (dict(out_features=0), 1, "bad shape"),
    (dict(rows=1 << 31), 1, "too large"),
    (dict(dtype=0), 2, "bfloat16 or float16"),
    (dict(activation=4), 1, "unknown activation"),
    (dict(ldx=63), 1, "row stride"),
    (dict(ldg=63), 1, "row stride"),
    (dict(ldu=63), 1, "row stride"),
    (dict(ldd=39), 1, "row stride"),
    (dict(ldr=47), 1, "row stride"),
    (dict(gate_bias_dtype=1), 1, "bias must be"),
    (dict(up_bias_dtype=1), 1, "bias must be"),
    (dict(down_bias_dtype=1), 1, "bias must be"),
    (dict(act=None), 1, "both or neither"),
    (dict(x=17), 1, "not aligned"),
    (dict(up_weight=17), 1, "not aligned"),
    (dict(h=18), 1, "not aligned"),
    (dict(slope=18), 1, "not aligned"),
    (dict(gate_bias=18), 1, "not aligned"),
]


@pytest.mark.parametrize("over,status,msg", BAD + [(dict(**{k: None}), 1, "pointer is NULL") for k in
                                                   ("x", "gate_weight", "up_weight", "down_weight", "h", "out")] + [({}, 4, "workspace")])
def test_c_forward_refuses_before_any_cuda_call(over, status, msg):
    lib = _lib.load()
    assert lib.ow_ffn_fwd(ctypes.byref(_args(**over)), None) == status
    assert msg in lib.ow_last_error().decode()


@pytest.mark.parametrize("over,grads,status,msg", [(o, {}, s, m) for o, s, m in BAD] + [
    (dict(rows=0), {}, 1, "no rows"),
    (dict(act=None, slope=None), {}, 1, "pointer is NULL"),
    (dict(x=None), {}, 1, "pointer is NULL"),
    (dict(h=None), {}, 1, "pointer is NULL"),
    (dict(down_weight=None), {}, 1, "pointer is NULL"),
    ({}, dict(dout=None), 1, "pointer is NULL"),
    ({}, dict(dup_weight=None), 1, "asked for alike"),
    ({}, dict(dgate_dtype=0), 1, "asked for alike"),
    ({}, dict(ddown_dtype=3), 2, "of dtype or float32"),
    ({}, dict(dx=17), 1, "not aligned"),
    ({}, dict(dgate_bias=18), 1, "not aligned"),
    ({}, {}, 4, "workspace"),
])
def test_c_backward_refuses_before_any_cuda_call(over, grads, status, msg):
    lib = _lib.load()
    g = _lib.FfnGrads(16, 16, 16, 2, 16, 2, 16, 2, 16, 16, 16)
    for k, v in grads.items():
        setattr(g, k, v)
    assert lib.ow_ffn_bwd(ctypes.byref(_args(**over)), ctypes.byref(g), None) == status
    assert msg in lib.ow_last_error().decode()


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.ow_ffn_workspace_size(_args(dtype=0), None) == 0
    assert lib.ow_ffn_workspace_size(_args(rows=0), None) > 0
    plain = lib.ow_ffn_workspace_size(_args(), None)
    odd = lib.ow_ffn_workspace_size(_args(in_features=63, ldx=63, ldg=63, ldu=63), None)
    assert odd >= plain + 100 * 64 * 2 + 2 * 40 * 64 * 2  # x and both weights in rows of 64
    g = _lib.FfnGrads(16, 16, 16, 2, 16, 2, 16, 2, 16, 16, 16)
    assert lib.ow_ffn_workspace_size(_args(), g) >= 2 * 100 * 40 * 2  # dg and du
