"""The feed-forward block where the gated product, and what its backward holds, have more than 2^31 elements."""

from __future__ import annotations

import pytest
import torch

from test_gpu_feed_forward import BF, _define, _inputs, _ok, _run

pytestmark = pytest.mark.gpu


def test_past_two_to_the_31_elements(cuda_device):
    m, k, f, n = 262_209, 16, 8200, 24  # h, act(g), u act'(g), dg and du of 4.3 GB each
    assert m * f > 2 ** 31
    a, dy = _inputs(cuda_device, m, k, f, n, BF)
    leaves = {key: v.detach().requires_grad_() for key, v in a.items()}
    y = _run(leaves, "gelu")
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    with torch.no_grad():
        assert torch.equal(_run(a, "gelu"), y)
    # rows, first and last ones, in full
    rows = torch.tensor([0, 1, 127, 128, m // 2, m - 66, m - 65, m - 2, m - 1], device=cuda_device)
    want = _define(a["x"][rows], a["wg"], a["wu"], a["wd"], a["bg"], a["bu"], a["bd"], a["r"][rows], dy[rows], "gelu", BF)
    _ok(y.detach()[rows], want["y"], "y")
    _ok(grads["x"][rows], want["x"], "dx")
    # some of the hidden features' gradients, over all rows: the others have no part in them
    cols = torch.tensor([0, 7, 8, 255, 256, 4100, f - 9, f - 2, f - 1], device=cuda_device)
    want = _define(a["x"], a["wg"][cols], a["wu"][cols], a["wd"][:, cols], a["bg"][cols], a["bu"][cols], a["bd"], a["r"], dy, "gelu", BF)
    for key in ("wg", "wu", "bg", "bu"):
        _ok(grads[key][cols], want[key], "d" + key)
    _ok(grads["wd"][:, cols], want["wd"], "dwd")
    _ok(grads["bd"], want["bd"], "dbd")
