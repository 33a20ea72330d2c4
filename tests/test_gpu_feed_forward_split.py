"""The feed-forward block's backward where dh = dy Wd is a product of few tiles and long k, split over k.

dh is an intermediate that no caller sees: its size must not bound the gradients'.
Bounds as in ``test_gpu_feed_forward``.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_feed_forward import BF, HF, _both, _define, _inputs, _run

pytestmark = pytest.mark.gpu


def _ok_or_past_f16(got, want, where):
    """Within its bound; a sum (a bias's, over 300 rows of some hundreds) of 65520 or more is infinite in f16, which
    rounds to a multiple of 32 below 65536 and has no number there."""
    want = want.round(HF)
    size, err = want.v.abs(), (got.double() - want.v).abs()
    past, close = size - want.e >= 65520, size + want.e >= 65520
    right = torch.where(torch.isinf(got), close & (got.double().sign() == want.v.sign()), ~past & (err <= want.e))
    assert right.all(), f"{where}: {got[~right][:4]} for {want.v[~right][:4]}"


@pytest.mark.parametrize("act", ["silu", "gelu", "none"])
@pytest.mark.parametrize("m,k,f,n", [(60, 64, 200, 4096), (40, 72, 129, 4100), (300, 64, 200, 4096), (3000, 64, 264, 4096), (60, 64, 201, 4097)],
                         ids=lambda s: str(s))
def test_dh_beyond_f16(cuda_device, m, k, f, n, act):
    """dh of 131072 or so, times a slope of about 2^-8: dg and du are inside f16's range, whatever the number of rows."""
    a, _ = _inputs(cuda_device, m, k, f, n, HF)
    for key in ("x", "bg", "bu"):
        a[key] = (a[key].float() * 2.0 ** -7).to(HF)
    a["wd"] = (4.0 + a["wd"].float()).to(HF)
    dy = torch.full((m, n), 8.0, dtype=HF, device=cuda_device)
    leaves = {key: v.detach().requires_grad_() for key, v in a.items()}
    grads = dict(zip(leaves, torch.autograd.grad(_run(leaves, act), list(leaves.values()), dy)))
    want = _define(*(a[key] for key in ("x", "wg", "wu", "wd", "bg", "bu", "bd", "r")), dy, act, HF)
    for key, g in grads.items():
        if key != "r":
            _ok_or_past_f16(g, want[key], f"{m}x{k}x{f}x{n} {act} d{key}")
    assert all(torch.isfinite(grads[key]).all() for key in ("x", "wg", "wu", "wd"))


@pytest.mark.parametrize("m,k,f,n", [(60, 64, 200, 4096), (40, 72, 129, 4100), (300, 64, 200, 4096), (60, 64, 201, 4097)], ids=lambda s: str(s))
def test_dh_below_f16(cuda_device, m, k, f, n):
    """dh of about 2^-27, which f16 has no numbers for, times act(g) and u act'(g) of about 2^12."""
    a, _ = _inputs(cuda_device, m, k, f, n, HF)
    a["x"] = (a["x"].float() * 2.0 ** 12).to(HF)
    a["wd"] = (a["wd"].float() * 2.0 ** -8).to(HF)
    a["r"] = None
    a = {key: v for key, v in a.items() if v is not None}
    dy = (torch.randn(m, n, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(1)) * 2.0 ** -21).to(HF)
    leaves = {key: a[key].detach().requires_grad_() for key in ("wg", "wu")}
    got = torch.autograd.grad(_run(a | leaves, "none"), list(leaves.values()), dy)
    x, wg, wu, wd, bg, bu = (a[key].double() for key in ("x", "wg", "wu", "wd", "bg", "bu"))
    dh = dy.double() @ wd
    want = ((dh * (x @ wu.t() + bu)).t() @ x, (dh * (x @ wg.t() + bg)).t() @ x)
    for g, w in zip(got, want):
        # dg or du and the gradient rounded, act or slope kept in f16: three roundings, 2^-11 each, of terms that add up at random;
        # dg and du of 2^-15 lie where f16 has steps of 2^-24, half of one off: 2^-10 of them
        assert float((g.double() - w).norm()) <= (3 * 2.0 ** -11 + 2.0 ** -10) * float(w.norm())


@pytest.mark.parametrize("t", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("m,k,f,n", [(512, 1024, 2048, 1024), (200, 512, 1024, 2048), (33, 130, 70, 5000), (64, 64, 8, 9000), (77, 40, 1030, 3001)],
                         ids=lambda s: str(s))
def test_split_products(cuda_device, m, k, f, n, t):
    for act in ("silu", "gelu"):
        a, dy = _inputs(cuda_device, m, k, f, n, t, act)
        first = _both(a, dy, act, f"{m}x{k}x{f}x{n} {act}")
        second = _both(a, dy, act, "again")
        assert all(torch.equal(first[key], second[key]) for key in first)
        wide = torch.zeros(m, n + 3, dtype=t, device=cuda_device)  # dy that is no matrix of 16-byte rows
        wide[:, 1:n + 1] = dy
        assert all(torch.equal(first[key], g) for key, g in _both(a, wide[:, 1:n + 1], act, "strided").items() if key != "r")
