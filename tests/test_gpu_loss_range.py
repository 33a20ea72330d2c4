"""Distillation loss on the GPU where logits are masked, far from zero, or divided by small temperatures.

A softmax does not hang on what its logits have in common, so the bounds here go by
the distances d = (m - z) k from the row's largest logit m (k = log2(e) / T), and not by
the logits.  u = 2^-24.  A distance's argument is a difference, the factor k and a
product, each within u of itself, and the special-function unit is within 2^-22: a
term is off by (3 u ln2 d + 2^-22 + u) of itself.  A thread adds its terms in chains of
at most ``links`` additions and moves its sum at most ``moves`` times to a larger pivot;
a move by d is off by as much as a term of that distance is, of a sum that is then
2^-d of the whole, and 2^-d d ln2 is at most 1/e.
"""

from __future__ import annotations

import pytest
import torch

from omniwave_b200 import loss

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def _half(t):
    return U if t == F32 else torch.finfo(t).eps / 2


def _links(v, many):
    # by 224 threads a row, or by a warp where classes are at most 256 or rows are ``many``; joining lanes and warps; single elements
    return v // (32 if many else 224) + 40, v // (32 * 16 if many else 224 * 16) + 10


def _soft(z, temp, v, many):
    """log q, q, the relative error of a row's sum and of each term, in float64 (rows of finite largest logits)."""
    m = z.amax(1, keepdim=True)
    d = (z - m) / temp                       # -inf allowed
    lq = d - d.exp().sum(1, keepdim=True).log()
    q = lq.exp()
    links, moves = _links(v, many)
    term = 3 * U * torch.where(q > 0, -d, 0.0) + 2.0 ** -22 + U
    rel = (q * term).sum(1) + links * U + moves * (2.0 ** -22 + 4 * U)
    return lq, q, rel, term


def _define(z, t, cls, y, temp, weight, g, many=False):
    """reduction "none": the rows' losses, the gradient, and the bounds of their errors."""
    dtype, v, k = z.dtype, z.shape[1], t.shape[1]
    z, t, g = z.double(), t.double(), g.double()
    lq, q, rel, term = _soft(z, temp, v, many)
    l1, q1, rel1, term1 = _soft(z, 1.0, v, many)
    on = cls >= 0
    c = cls.clamp(min=0)
    tt = torch.where(on, t, -torch.inf)
    tm = tt.amax(1, keepdim=True)
    dt = (tt - tm) / temp
    lp = dt - dt.exp().sum(1, keepdim=True).log()
    p = lp.exp()
    relp = 3 * U * torch.where(p > 0, -dt, 0.0) + 2.0 ** -21 + (k // 32 + 12) * U
    relp = relp + (p * relp).sum(1, keepdim=True)
    some = on & (p > 0)
    gap = torch.where(some, lp - lq.gather(1, c), 0.0)
    away = torch.where(some, (z.amax(1, keepdim=True) - z.gather(1, c)) / temp, 0.0)
    soft = temp ** 2 * torch.where(some, p * gap, 0.0).sum(1)
    # entries' distances and the student's at them, each with its probability's error; both logarithms
    esoft = temp ** 2 * (torch.where(some, p * (-dt + away) * (2 * relp + (k // 32 + 12) * U), 0.0).sum(1)
                         + 1.1 * (rel + relp.amax(1)) + 4 * U * (lq.abs().amin(1) + lp.abs().amin(1) + 1))
    hard = -l1.gather(1, y[:, None])[:, 0]
    ehard = 1.1 * rel1 + 4 * U * (l1.abs().amin(1) + 1)
    value = weight * soft + (1 - weight) * hard
    evalue = weight * (esoft + 6 * U * soft.abs()) + (1 - weight) * (ehard + 6 * U * hard.abs())
    a, b = g * weight * temp, g * (1 - weight)
    top = torch.zeros_like(z).scatter_add_(1, c, torch.where(some, p, 0.0) * a[:, None])
    etop = torch.zeros_like(z).scatter_add_(1, c, torch.where(some, p * (relp + 8 * U), 0.0) * a[:, None])
    lab = torch.zeros_like(z).scatter_add_(1, y[:, None], b[:, None])
    dz = a[:, None] * q + b[:, None] * q1 - top - lab
    # with T of 2 or 4 the second probability is the first one's power: 4 times as far off
    edz = (a[:, None] * q * (rel[:, None] + term + 10 * U) + b[:, None] * q1 * (rel1[:, None] + 4 * (term + term1) + 10 * U)
           + etop + 8 * U * lab)
    edz = edz + 2.0 ** -125 * (a + b)[:, None]  # a special-function result below 2^-126 is 0
    edz = edz * 1.05 + _half(dtype) * 1.01 * (dz.abs() + edz)
    return value, evalue * 1.05, dz, edz + (2.0 ** -25 if dtype == HF else 2.0 ** -133)


def _check(z, top, cls, y, temp, weight, where, many=False):
    leaf = z.detach().requires_grad_()
    rows = loss.distill_loss(leaf, top, cls, y, temperature=temp, weight=weight, reduction="none")
    up = torch.linspace(0.5, 2.0, z.shape[0], device=z.device)
    (g,) = torch.autograd.grad(rows, leaf, up)
    want, tol, dz, edz = _define(z.detach(), top, cls, y, temp, weight, up, many)
    rows = rows.detach()
    assert torch.isfinite(rows).all() and torch.isfinite(g).all(), f"{where}: {rows}"
    err = (rows.double() - want).abs()
    assert (err <= tol).all(), f"{where} loss: worst {(err / tol).max().item():.2f} of the bound"
    err = (g.double() - dz).abs()
    assert (err <= edz).all(), f"{where} gradient: worst {(err / edz).max().item():.2f} of the bound"
    mean = loss.distill_loss(z, top, cls, y, temperature=temp, weight=weight)
    assert abs(float(mean) - float(want.mean())) <= float(tol.mean()) + 4 * U * float(want.abs().mean())
    return rows, g


def _inputs(dev, n, v, k, t, seed, live=None):
    """Logits, entries and labels; entries and labels among the first ``live`` classes."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    z = torch.randn(n, v, generator=gen, device=dev) * 2
    live = live or v
    best = (z[:, :live] * 0.7 + torch.randn(n, live, generator=gen, device=dev) * 2).topk(min(k, live), 1)
    return z.to(t), best.values, best.indices, torch.randint(live, (n,), generator=gen, device=dev)


@pytest.mark.parametrize("temp", [1.0, 0.7, 2.0, 4.0])
@pytest.mark.parametrize("t", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,v,live", [(6, 1000, 300), (5, 1001, 37), (4, 40009, 5000), (9, 255, 16), (1000, 2000, 24), (1000, 777, 30)],
                         ids=lambda s: str(s))
def test_classes_masked_with_the_types_lowest_value(cuda_device, n, v, live, t, temp):
    """A masked range, whole vectors and whole threads' shares of it, before, behind and around the live classes."""
    z, top, cls, y = _inputs(cuda_device, n, v, 6, t, 1, live)
    low = torch.finfo(t).min
    many = n >= 888
    for first in (0, v - live, (v - live) // 2):
        zz = torch.full((n, v), low, dtype=t, device=cuda_device)
        zz[:, first:first + live] = z[:, :live]
        _, g = _check(zz, top, cls + first, y + first, temp, 0.5, f"masked but {first}..{first + live}", many)
        dead = torch.ones(v, dtype=torch.bool, device=cuda_device)
        dead[first:first + live] = False
        assert (g[:, dead] == 0).all()
    # rows apart by an odd number of elements: single elements at both ends
    wide = torch.full((n, v + 3), low, dtype=t, device=cuda_device)
    wide[:, 1:1 + live] = z[:, :live]
    _check(wide[:, 1:v + 1], top, cls, y, temp, 0.5, "masked, unaligned", many)


@pytest.mark.parametrize("t", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("v", [40, 1001])
def test_one_live_class_in_a_row(cuda_device, v, t):
    """All but one class masked: its probability is 1, and label and teacher alike cost nothing there."""
    for at in (0, v // 2, v - 1):
        z = torch.full((3, v), torch.finfo(t).min, dtype=t, device=cuda_device)
        z[:, at] = -3.0
        cls = torch.full((3, 1), at, device=cuda_device)
        for temp in (1.0, 0.7, 2.0):
            leaf = z.clone().requires_grad_()
            rows = loss.distill_loss(leaf, torch.ones(3, 1, device=cuda_device), cls, cls[:, 0], temperature=temp, reduction="none")
            (g,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
            assert (rows == 0).all() and (g == 0).all()


@pytest.mark.parametrize("t", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("v", [40, 1000, 1001])
def test_rows_whose_every_class_is_masked(cuda_device, v, t):
    """All logits at the type's lowest value: uniform, as of any other logits that are all alike."""
    for value in (torch.finfo(t).min, torch.finfo(t).max, -1.0e30, 7.0):
        z = torch.full((3, v), value, dtype=t, device=cuda_device)
        top, cls = torch.zeros(3, 2, device=cuda_device), torch.tensor([[0, 1], [2, v - 1], [5, 6]], device=cuda_device)
        y = torch.tensor([0, v - 1, v // 2], device=cuda_device)
        for temp in (1.0, 0.7, 2.0, 4.0):
            _check(z, top, cls, y, temp, 0.5, f"all {value}")


@pytest.mark.parametrize("temp", [1.0, 0.7, 2.0, 4.0])
@pytest.mark.parametrize("n,v", [(6, 1000), (5, 1001), (4, 32000), (9, 200), (1000, 2000)], ids=lambda s: str(s))
@pytest.mark.parametrize("offset", [1000.0, -1000.0, 10000.0])
def test_logits_far_from_zero(cuda_device, n, v, offset, temp):
    z, top, cls, y = _inputs(cuda_device, n, v, 9, F32, 2)
    _check(z + offset, top + offset, cls, y, temp, 0.5, f"at {offset}", n >= 888)


@pytest.mark.parametrize("t", [F32, HF], ids=["f32", "f16"])
@pytest.mark.parametrize("temp", [1e-4, 1e-2, 0.3, 50.0, 1e4])
def test_temperatures(cuda_device, temp, t):
    for n, v in ((6, 1000), (5, 1001), (4, 32000)):
        z, top, cls, y = _inputs(cuda_device, n, v, 40, t, 3)
        _check(z, top, cls, y, temp, 0.7, f"T = {temp}")
        near = (z.float() * temp).to(t)  # a softmax of more than one class at this temperature
        if t == F32:
            _check(near, top * temp, cls, y, temp, 0.7, f"T = {temp}, near")


@pytest.mark.parametrize("offset,temp", [(1000.0, 1.0), (1000.0, 3.0), (0.0, 0.01), (10000.0, 2.0)])
def test_probabilities_keep_their_digits(cuda_device, offset, temp):
    """Without entries' or labels' share a gradient is its probability's: within 1e-5 of 64 bits, whatever is common to the logits."""
    z, top, cls, y = _inputs(cuda_device, 8, 1000, 3, F32, 4)
    z = (z * (temp if temp < 1 else 1.0) + offset).requires_grad_()
    rows = loss.distill_loss(z, top, cls, temperature=temp, weight=1.0, reduction="none")
    (g,) = torch.autograd.grad(rows, z, torch.ones_like(rows))
    q = (z.detach().double() / temp).softmax(1)
    keep = (q > 1e-3).scatter(1, cls, False)
    assert keep.any()
    worst = ((g.double() / temp - q).abs() / q)[keep].max().item()
    assert worst <= 1e-5, worst
    # a row's gradient adds up to 0: q and p to 1 each, each element rounded
    assert (g.double().sum(1).abs() <= temp * (1e-5 + 1000 * U)).all()


def test_a_large_teacher(cuda_device):
    """Entries past what their logarithm holds, or all at their type's lowest value, are entries still."""
    z, top, cls, y = _inputs(cuda_device, 4, 500, 5, F32, 5)
    for fill in (3.0e38, torch.finfo(F32).min, 2.0e30):
        t = torch.full_like(top, fill)
        for temp in (1.0, 0.5):
            _check(z, t, cls, y, temp, 0.5, f"teacher of {fill}")
            rows = loss.distill_loss(z, t, cls, temperature=temp, weight=1.0, reduction="none")
            assert (rows > 0).all()  # uniform over five of 500 classes


@pytest.mark.parametrize("v", [40, 1001, 2000])
@pytest.mark.parametrize("t", [F32, BF], ids=["f32", "bf16"])
def test_entries_at_classes_of_probability_0(cuda_device, v, t):
    z, top, cls, _ = _inputs(cuda_device, 4, v, 6, t, 6)
    top[:, 4:] = -torch.inf
    y = torch.tensor([next(c for c in range(v) if c not in row) for row in cls.tolist()], device=cuda_device)  # beside the entries
    z[0, int(cls[0, 5])] = -torch.inf    # an entry of probability 0 at a class of probability 0: no term
    z[1, int(cls[1, 0])] = -torch.inf    # of positive probability: inf
    z[2, cls[2, :4]] = -torch.inf        # all of them
    for temp in (1.0, 2.0, 0.7):
        leaf = z.detach().requires_grad_()
        rows = loss.distill_loss(leaf, top, cls, y, temperature=temp, weight=0.5, reduction="none")
        (g,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
        assert torch.isfinite(rows[[0, 3]]).all() and (rows[1:3] == torch.inf).all()
        assert torch.isfinite(g).all()   # q is 0 there, p is not
