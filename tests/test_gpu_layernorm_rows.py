"""Layer norm's kernels for many rows, at rows of few channels and at rows whose mean is far past the others'."""

from __future__ import annotations

import pytest
import torch

from omniwave_b200 import norm
from test_gpu_layernorm import _both, _inputs

pytestmark = pytest.mark.gpu

F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def _grads(x, w, b, dn, eps):
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    n = norm.layer_norm(*leaves, eps=eps, out_dtype=dn.dtype)
    return (n.detach(), *torch.autograd.grad(n, leaves, dn))


@pytest.mark.parametrize("rows,c", [(30011, 96), (13003, 200), (5003, 520), (40003, 70), (9001, 311), (2003, 1501), (99, 96), (9, 70)],
                         ids=lambda s: str(s))
@pytest.mark.parametrize("t,out", [(F32, F32), (BF, BF), (F32, BF)], ids=["f32", "bf16", "f32-bf16"])
def test_constant_rows_of_any_size(cuda_device, rows, c, t, out):
    """A constant row is its mean: x^ is 0 there, whatever the constant, so all results are those of a row of zeros.

    2^110 times 1 / sqrt(eps) = 2^20 is past f32's range, and a row's sum, of at most 2^11 such values, is exact.
    """
    assert float(torch.tensor(c, dtype=F32) * (1.0 / torch.tensor(c, dtype=F32))) == 1.0  # the mean of the constant is the constant
    g = torch.Generator(device=cuda_device).manual_seed(c)
    x = torch.randn(rows, c, generator=g, device=cuda_device).to(t)
    dn = torch.randn(rows, c, generator=g, device=cuda_device).to(out)
    w, b = torch.randn(c, generator=g, device=cuda_device), torch.randn(c, generator=g, device=cuda_device)
    for at in (slice(None, None, 7), slice(rows - 1, rows), slice(0, 1), slice(rows // 2, rows // 2 + 1)):
        zeros, far = x.clone(), x.clone()
        zeros[at], far[at] = 0.0, 2.0 ** 110
        for what, p, q in zip(("n", "dx", "dw", "db"), _grads(far, w, b, dn, 2.0 ** -40), _grads(zeros, w, b, dn, 2.0 ** -40)):
            assert torch.isfinite(q).all() and torch.equal(p, q), what


@pytest.mark.parametrize("rows,c", [(1_300_001, 2), (900_001, 3), (360_003, 7), (320_001, 8), (160_001, 16), (150_011, 17)], ids=lambda s: str(s))
@pytest.mark.parametrize("t,out", [(F32, F32), (BF, BF), (F32, HF)], ids=["f32", "bf16", "f32-f16"])
def test_many_rows_of_few_channels(cuda_device, rows, c, t, out):
    """Many rows in a chunk of the ring, chunks that end inside a 16-byte unit."""
    x, w, b, dn = _inputs(cuda_device, (rows, c), t, F32, seed=c)
    first = _both(x, w, b, dn, f"{rows}x{c}", out=out)
    assert all(torch.equal(p, q) for p, q in zip(first, _both(x, w, b, dn, f"{rows}x{c}", out=out)))


@pytest.mark.parametrize("t", [F32, BF, HF], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [2_430_001, 5_000_003])
def test_many_rows_of_one_channel(cuda_device, rows, t):
    """A row is its own mean: the bias is left, dx and dw are 0, db is the sum of dn."""
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x, w, b = torch.randn(rows, 1, generator=g, device=cuda_device).to(t), torch.ones(1, device=cuda_device), torch.full((1,), 0.375, device=cuda_device)
    dn = torch.randint(-2, 3, (rows, 1), generator=g, device=cuda_device).to(t)  # its sums are exact
    n, dx, dw, db = _grads(x, w, b, dn, 1e-5)
    assert (n == 0.375).all() and (dx == 0).all() and dw == 0 and db == dn.double().sum()
