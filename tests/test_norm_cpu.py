"""Norms with gate and residual (host side, no GPU): argument checks of the functions and of the C entry points."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_b200 import _lib, norm
from omniwave_b200.block import OmniWeaveBlock


def test_refuses_host_tensors():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    assert norm.norm_supported(x, w) == (False, "CUDA is unavailable")
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        norm.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        norm.norm_residual(x, x, w)


@pytest.mark.parametrize("call,match", [
    (lambda x, w: norm.rms_norm(x, torch.ones(7)), r"weight must be \[8\]"),
    (lambda x, w: norm.rms_norm(torch.zeros(3, 0), torch.ones(0)), r"x must be"),
    (lambda x, w: norm.rms_norm(x, w, eps=-1.0), "eps"),
    (lambda x, w: norm.norm_residual(x[0, 0], x[0, 0], w), r"x must be \[B"),
    (lambda x, w: norm.norm_residual(x, x[:1], w), "delta must be"),
    (lambda x, w: norm.norm_residual(x, x, w[:5]), "weight must be"),
    (lambda x, w: norm.norm_residual(x, x, w, w[:1]), "gate must be"),
    (lambda x, w: norm.norm_residual(x, x, w, torch.ones(3, 8)), "gate must be"),
    (lambda x, w: norm.norm_residual(x, x, w, next_weight=torch.ones(2, 8)), "next_weight must be"),
])
def test_refuses_shapes(call, match):
    with pytest.raises(ValueError, match=match):
        call(torch.zeros(2, 3, 8), torch.ones(8))


def _args(**over):
    a = _lib.Norm(4, 49, 70, 16, 0, 16, 2, 16, 0, 16, 0, 1, None, 16, 0, 1e-6, 16, 16, 0, 16, 16, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status,msg", [
    (dict(channels=0), 1, "bad shape"),
    (dict(tokens=-1), 1, "bad shape"),
    (dict(samples=1 << 31), 1, "too many rows"),
    (dict(x=None), 1, "input pointer"),
    (dict(post_w=None), 1, "input pointer"),
    (dict(gate_rows=3), 1, "gate must have"),
    (dict(gate=None), 1, "gate must have"),
    (dict(delta=None, gate_rows=0, sample_scale=16), 1, "needs delta"),
    (dict(delta=None, gate_rows=0, next_w=None), 1, "input pointer"),
    (dict(x_dtype=1), 2, "float32, bfloat16 or float16"),
    (dict(gate_dtype=7), 2, "float32, bfloat16 or float16"),
    (dict(eps=-1.0), 1, "eps"),
    (dict(h=None), 1, "output pointer"),
    (dict(n=None), 1, "output pointer"),
])
def test_c_forward_refuses_before_any_cuda_call(over, status, msg):
    lib = _lib.load()
    assert lib.ow_norm_fwd(ctypes.byref(_args(**over)), None) == status
    assert msg in lib.ow_last_error().decode()


def test_c_backward_refuses_before_any_cuda_call():
    lib = _lib.load()
    g = _lib.NormGrads(16, 16, 16, 16, 16, 16, 16)
    assert lib.ow_norm_bwd(ctypes.byref(_args()), ctypes.byref(g), None) == 4  # no workspace
    assert "workspace" in lib.ow_last_error().decode()
    for k in ("dx", "ddelta", "dn"):
        g2 = _lib.NormGrads(16, 16, 16, 16, 16, 16, 16)
        setattr(g2, k, None)
        assert lib.ow_norm_bwd(ctypes.byref(_args()), ctypes.byref(g2), None) == 1, k
    assert lib.ow_norm_bwd(ctypes.byref(_args(rstd_h=None)), ctypes.byref(g), None) == 1
    assert lib.ow_norm_bwd(ctypes.byref(_args()), None, None) == 1
    assert lib.ow_norm_bwd_workspace_size(ctypes.byref(_args(channels=0))) == 0
    # three arrays of partial sums, at least one row of 70 channels each
    assert lib.ow_norm_bwd_workspace_size(ctypes.byref(_args())) >= 3 * 70 * 4


def test_post_norm_block_parameters():
    torch.manual_seed(0)
    plain = OmniWeaveBlock(4, 4, 64, 64, "local", 0)
    torch.manual_seed(0)
    post = OmniWeaveBlock(4, 4, 64, 64, "local", 0, post_norm=True)
    assert set(post.state_dict()) - set(plain.state_dict()) == {"post_norm_weight"}
    for k, v in plain.state_dict().items():
        assert torch.equal(v, post.state_dict()[k])
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        post(torch.zeros(1, 4, 4, 64))


@pytest.mark.parametrize("over,grads", [
    (dict(x=18), None), (dict(delta=17), None), (dict(post_w=18), None), (dict(gate=18), None), (dict(next_w=18), None),
    (dict(h=18), None), (dict(n=17), None), (dict(sample_scale=18), None), (dict(rstd_h=18), {}), ({}, dict(dh=18)),
    ({}, dict(dn=17)), ({}, dict(dx=18)), ({}, dict(ddelta=17)), ({}, dict(dpost=18)), ({}, dict(dgate=18)), ({}, dict(dnext=18)),
])
def test_c_entries_refuse_pointers_off_their_alignment(over, grads):
    lib = _lib.load()
    a = _args(n_dtype=2, **over)
    if grads is None:
        status = lib.ow_norm_fwd(ctypes.byref(a), None)
    else:
        g = _lib.NormGrads(16, 16, 16, 16, 16, 16, 16)
        for k, v in grads.items():
            setattr(g, k, v)
        status = lib.ow_norm_bwd(ctypes.byref(a), ctypes.byref(g), None)
    assert status == 1 and "not aligned" in lib.ow_last_error().decode()


def test_refuses_rows_that_their_length_field_does_not_hold():
    c = 2 ** 32 + 8  # 8 in 32 bits
    x, w = torch.zeros(1, 1).expand(1, c), torch.zeros(1).expand(c)
    with pytest.raises(ValueError, match="too many channels"):
        norm.rms_norm(x, w)
    with pytest.raises(ValueError, match="too many channels"):
        norm.norm_residual(x, x, w)
    lib = _lib.load()
    assert lib.ow_norm_fwd(ctypes.byref(_args(channels=2 ** 31 - 1)), None) == 1
    assert "too many channels" in lib.ow_last_error().decode()


@pytest.mark.parametrize("which", ["x", "delta", "weight", "gate", "scale", "next"])
def test_refuses_forward_mode(which):
    """A tangent would be dropped: there is no formula for it here."""
    import torch.autograd.forward_ad as fw

    t = {"x": torch.zeros(2, 3, 8), "delta": torch.zeros(2, 3, 8), "weight": torch.ones(8), "gate": torch.ones(8),
         "scale": torch.ones(2), "next": torch.ones(8)}
    with fw.dual_level():
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            norm.norm_residual(t["x"], t["delta"], t["weight"], t["gate"], sample_scale=t["scale"], next_weight=t["next"])
        if which in ("x", "weight"):
            with pytest.raises(RuntimeError, match="forward-mode"):
                norm.rms_norm(t["x"], t["weight"])


@pytest.mark.parametrize("samples,tokens,c,bf16,parts", [
    (50176, 1, 1024, True, 1),   # a row a sample: one part each
    (262144, 1, 1024, True, 1),
    (128, 196, 512, True, 3),    # as many as make three blocks an SM
    (100_000, 1, 70, False, 1),  # ragged rows as well, while a block takes a sample's rows at once
    (100_000, 1, 777, True, 1),
    (128, 49, 777, True, 4),     # and here every fourth row of a block starts alike
])
def test_backward_workspace_is_what_the_parts_take(samples, tokens, c, bf16, parts):
    lib = _lib.load()
    t = 2 if bf16 else 0
    a = _args(samples=samples, tokens=tokens, channels=c, x_dtype=t, delta_dtype=t, n_dtype=t, gate_rows=samples)
    assert lib.ow_norm_bwd_workspace_size(ctypes.byref(a)) <= samples * parts * 2 * c * 4 + 256


def test_forward_blocks_runs_hooks_and_other_modules():
    """A block that is watched or wrapped is called, not taken apart; a hook in front of it runs before any CUDA call."""
    from omniwave_b200.block import forward_blocks

    class Wrapper(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, x):
            seen.append("wrapper")
            return x + 1

    seen = []
    x = torch.zeros(1, 4, 4, 64)
    for post in (False, True):
        blk = OmniWeaveBlock(4, 4, 64, 64, "local", 0, post_norm=post)
        blk.register_forward_pre_hook(lambda m, a: seen.append("pre"))
        with pytest.raises(RuntimeError, match="CUDA is unavailable"):
            forward_blocks([blk], x)
    assert seen == ["pre", "pre"]
    assert torch.equal(forward_blocks([Wrapper(blk), Wrapper(blk)], x), x + 2)
    assert seen[2:] == ["wrapper", "wrapper"]

    class Shifted(OmniWeaveBlock):
        def forward(self, x):
            return x + 3

    assert torch.equal(forward_blocks([Shifted(4, 4, 64, 64, "local", 0, post_norm=True)], x), x + 3)
    patched = OmniWeaveBlock(4, 4, 64, 64, "local", 0, post_norm=True)
    patched.forward = lambda x: x + 5
    assert torch.equal(forward_blocks([patched], x), x + 5)
    handle = torch.nn.modules.module.register_module_forward_pre_hook(lambda m, a: seen.append("global"))
    try:
        with pytest.raises(RuntimeError, match="CUDA is unavailable"):
            forward_blocks([OmniWeaveBlock(4, 4, 64, 64, "local", 0, post_norm=True)], x)
    finally:
        handle.remove()
    assert seen[-1] == "global"
