"""Distillation loss on the GPU against float64.

u = 2^-24.  An exponential's argument, to the base of 2, is one multiply-add
(u of itself) of a logit with a rounded factor (u of the product), so a term of a
softmax is off by ``a`` = 4 u (largest argument + 2) + 2^-22 of itself (the
special-function unit's own error is within 2^-22).  A row's sum adds its terms in
chains of at most classes / 32 + 64 links and rescales at most that often, each
within 2^-22 (nearly all by factors of 1, which are exact; 64 are counted).
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


def _define(z, t, cls, y, temp, weight, reduction, g=None):
    """The loss, its gradient and the bounds of their errors, in float64, term by term."""
    dtype = z.dtype
    z, t = z.double(), t.double()
    n, v = z.shape
    on = cls >= 0
    c = cls.clamp(min=0).long()
    t = torch.where(on, t, -torch.inf)
    has_t = (t > -torch.inf).any(1) & (weight > 0)
    has_y = (y >= 0) if y is not None and weight < 1 else torch.zeros(n, dtype=torch.bool, device=z.device)
    arg = 1.4427 * 2 * torch.where(z.isfinite(), z, 0.0).abs().amax(1) / min(temp, 1.0)
    targ = 1.4427 * 2 * torch.where(t.isfinite(), t, 0.0).abs().amax(1) / temp
    chain = (v // 32 + 64) * U + 64 * 2.0 ** -22
    rel = 4 * U * (arg + 2) + 2.0 ** -22 + chain       # a probability of the student, relative to itself
    relp = 4 * U * (targ + 2) + 2.0 ** -21 + 64 * U    # of the teacher
    ts = torch.where(has_t[:, None], t / temp, 0.0)
    lp = ts.log_softmax(1)
    p = torch.where(on & has_t[:, None], lp.exp(), 0.0)
    lq = (z / temp).log_softmax(1)
    at = lq.gather(1, c)
    gap = torch.where(p > 0, lp - at, 0.0)
    soft = temp ** 2 * torch.where(p > 0, p * gap, 0.0).sum(1)
    esoft = temp ** 2 * (torch.where(p > 0, p * gap.abs(), 0.0).sum(1) * (relp + 64 * U) + 2 * (rel + relp) + 4 * U * (arg + targ))
    l1 = z.log_softmax(1)
    yy = y.clamp(min=0).long() if y is not None else torch.zeros(n, dtype=torch.long, device=z.device)
    hard = torch.where(has_y, -l1.gather(1, yy[:, None])[:, 0], 0.0)
    ehard = torch.where(has_y, 2 * rel + 4 * U * arg, 0.0)
    soft, esoft = torch.where(has_t, soft, 0.0), torch.where(has_t, esoft, 0.0)
    ns, nh = (max(1, int(has_t.sum())), max(1, int(has_y.sum()))) if reduction == "mean" else (1, 1)
    rows, erows = weight * soft / ns + (1 - weight) * hard / nh, weight * esoft / ns + (1 - weight) * ehard / nh
    if reduction == "none":
        value, evalue = rows, erows + 4 * U * (soft + hard)
    else:
        value, evalue = rows.sum(), erows.sum() + 4 * U * (weight * soft / ns + (1 - weight) * hard / nh).abs().sum()
    up = torch.ones(n, device=z.device, dtype=torch.float64) * (1.0 if g is None else g.double())
    a, b = up * weight * temp / ns * has_t, up * (1 - weight) / nh * has_y
    parts = [a[:, None] * lq.exp(), b[:, None] * l1.exp()]
    parts = [torch.where(k[:, None] != 0, x, 0.0) for k, x in zip((a, b), parts)]
    top = torch.zeros_like(z).scatter_add_(1, c, p * a[:, None])
    lab = torch.zeros_like(z).scatter_add_(1, yy[:, None], b[:, None])
    dz = parts[0] + parts[1] - top - lab
    size = parts[0].abs() + parts[1].abs()
    edz = size * (rel[:, None] + 6 * U) + top.abs() * (relp[:, None] + (cls.shape[1] + 6) * U) + 6 * U * lab.abs()
    # a special-function result below 2^-126 is 0
    edz = edz + 2.0 ** -125 * (a.abs() + b.abs())[:, None]
    edz = edz + _half(dtype) * 1.01 * (dz.abs() + edz) + (2.0 ** -25 if dtype == HF else 2.0 ** -133 if dtype == BF else 2.0 ** -149)
    return value, evalue * 1.01 + 1e-30, dz, edz * 1.01


def _inputs(dev, n, v, k, t=F32, tt=F32, idx=torch.int64, seed=0, ragged=True, scale=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    z = (torch.randn(n, v, generator=g, device=dev) * scale).to(t)
    best = (z.double() * 0.7 + torch.randn(n, v, generator=g, device=dev) * scale).topk(min(k, v), 1)
    top, cls = best.values.to(tt), best.indices.to(idx)
    if k > v:  # more room than classes
        top = torch.nn.functional.pad(top, (0, k - v), value=9.0)
        cls = torch.nn.functional.pad(cls, (0, k - v), value=-1)
    y = torch.randint(v, (n,), generator=g, device=dev).to(idx)
    if ragged:
        kept = (torch.rand(n, generator=g, device=dev) * 1.5 * (k + 1)).long()
        cls = torch.where(torch.arange(k, device=dev) < kept[:, None], cls, -1)
        y = torch.where(torch.rand(n, generator=g, device=dev) < 0.2, -100, y)
    return z, top, cls, y


def _both(z, top, cls, y, temp, weight, reduction, where):
    want, tol, _, _ = _define(z, top, cls, y, temp, weight, reduction)
    kw = dict(temperature=temp, weight=weight, reduction=reduction)
    with torch.no_grad():
        plain = loss.distill_loss(z, top, cls, y, **kw)
    assert plain.dtype == F32 and plain.shape == want.shape
    assert ((plain.double() - want).abs() <= tol + U * want.abs()).all(), f"{where} loss: {plain}, {want}"
    leaf = z.detach().requires_grad_()
    got = loss.distill_loss(leaf, top, cls, y, **kw)
    assert torch.equal(got, plain)
    up = torch.randn(got.shape, device=z.device).abs() + 0.5
    _, _, dz, edz = _define(z, top, cls, y, temp, weight, reduction, up)
    (g,) = torch.autograd.grad(got, leaf, up)
    assert g.dtype == z.dtype and g.shape == z.shape
    err = (g.double() - dz).abs()
    assert (err <= edz).all(), f"{where} gradient: worst {(err / edz).max().item():.2f} of the bound"
    return got.detach(), g


CASES = [(1, 1, 1), (1, 2, 1), (3, 5, 8), (8, 1000, 10), (40, 7, 7), (64, 129, 33), (128, 1000, 32), (33, 1023, 64), (17, 1025, 100),
         (5, 4096, 256), (9, 10007, 1), (3, 40009, 1024), (2, 131072, 17), (2000, 12, 3), (700, 2000, 5)]


@pytest.mark.parametrize("n,v,k", CASES, ids=["x".join(map(str, c)) for c in CASES])
@pytest.mark.parametrize("t,tt,idx", [(F32, F32, torch.int64), (BF, HF, torch.int32), (HF, BF, torch.int64)], ids=["f32", "bf16", "f16"])
def test_loss_and_gradient(cuda_device, n, v, k, t, tt, idx):
    for i, (temp, weight, labels, reduction) in enumerate([(2.0, 0.6, True, "mean"), (1.0, 0.5, True, "none"), (0.7, 1.0, False, "sum"),
                                                           (3.0, 0.25, True, "sum"), (4.0, 0.9, True, "mean"),
                                                           (1.0, 0.0, True, "mean"), (5.5, 1.0, True, "mean")]):
        z, top, cls, y = _inputs(cuda_device, n, v, k, t, tt, idx, seed=i, ragged=i % 3 != 2)
        first = _both(z, top, cls, y if labels else None, temp, weight, reduction, f"{n}x{v} top {k} T={temp} w={weight} {reduction}")
        second = _both(z, top, cls, y if labels else None, temp, weight, reduction, "again")
        assert torch.equal(first[0], second[0])


def test_against_differences(cuda_device):
    z, top, cls, y = _inputs(cuda_device, 6, 40, 5, seed=3)
    leaf = z.detach().requires_grad_()
    (g,) = torch.autograd.grad(loss.distill_loss(leaf, top, cls, y, temperature=2.0, weight=0.7), leaf)
    way = torch.randn(z.shape, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(1)).double()

    def value(s):
        return _define(z.double() + s * way, top, cls, y, 2.0, 0.7, "mean")[0]

    want = float((value(1e-5) - value(-1e-5)) / 2e-5)
    got = float((g.double() * way).sum())
    assert abs(got - want) <= 1e-6 * float((g.double() * way).abs().sum())  # about 16 u a term


def test_a_class_named_twice_counts_twice(cuda_device):
    for n, v, k, t in ((4, 50, 12, F32), (3, 3000, 40, BF), (2, 9, 1024, F32)):
        z, top, cls, y = _inputs(cuda_device, n, v, min(k, v), t, seed=5, ragged=False)
        cls = cls.repeat(1, -(-k // cls.shape[1]))[:, :k].contiguous()
        cls[:, k // 2:] = cls[:, :1]                    # half of the entries, and the label, are one class
        top = torch.randn(n, k, device=cuda_device)
        y = cls[:, 0].clone()
        _both(z, top, cls, y, 2.0, 0.5, "mean", f"{v} twice")


def test_rows_with_nothing(cuda_device):
    """No entry, no label, neither: no term, no gradient, whatever the logits hold; all rows so: 0."""
    for v in (20, 3000):
        z, top, cls, y = _inputs(cuda_device, 6, v, 4, seed=6, ragged=False)
        cls[0], cls[1], y[1], y[2], top[3] = -1, -1, -100, -1, -torch.inf
        z[1, 3], z[1, 5] = float("nan"), float("inf")
        leaf = z.detach().requires_grad_()
        rows = loss.distill_loss(leaf, top, cls, y, weight=0.5, reduction="none")
        (g,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
        rows = rows.detach()
        assert rows[1] == 0 and (g[1] == 0).all() and torch.isfinite(rows).all() and torch.isfinite(g).all()
        ce = torch.nn.functional.cross_entropy(z.double(), y.clamp(min=0).long(), reduction="none")
        assert abs(float(rows[0]) - 0.5 * float(ce[0])) < 1e-5 and abs(float(rows[3]) - 0.5 * float(ce[3])) < 1e-5
        for red in ("mean", "sum"):
            leaf = z.detach().requires_grad_()
            out = loss.distill_loss(leaf, top, torch.full_like(cls, -1), torch.full_like(y, -100), reduction=red)
            (g,) = torch.autograd.grad(out, leaf)
            assert out == 0 and (g == 0).all()


def test_masked_classes_and_entries(cuda_device):
    """Classes at -inf have probability 0 and no gradient; entries at -inf count for nothing; a teacher sure of such a class: inf."""
    for v in (40, 2000):
        for t in (F32, BF):
            z, top, cls, y = _inputs(cuda_device, 5, v, 6, t, seed=7, ragged=False)
            dead = torch.zeros(5, v, dtype=torch.bool, device=cuda_device)
            dead[:, ::3] = True
            dead.scatter_(1, cls, False)
            dead.scatter_(1, y[:, None], False)
            z = z.masked_fill(dead, -torch.inf)
            top[:, 4:] = -torch.inf
            lowest = z.masked_fill(dead, torch.finfo(t).min)
            for zz in (z, lowest):
                rows, g = _both(zz, top, cls, y, 2.0, 0.5, "none", f"masked {v}") if zz is lowest else (None, None)
                leaf = zz.detach().requires_grad_()
                out = loss.distill_loss(leaf, top, cls, y, temperature=2.0, weight=0.5, reduction="none")
                (g,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
                assert torch.isfinite(out).all() and torch.isfinite(g).all() and (g[dead] == 0).all()
            z[0, int(cls[0, 5])] = -torch.inf    # an entry of probability 0 at a class of probability 0: no term
            z[1, int(cls[1, 0])] = -torch.inf    # of positive probability: inf
            if int(y[0]) != int(cls[0, 5]) and int(y[1]) != int(cls[1, 0]):
                rows = loss.distill_loss(z, top, cls, y, temperature=2.0, weight=0.5, reduction="none")
                assert torch.isfinite(rows[0]) and rows[1] == float("inf") and torch.isfinite(rows[2:]).all()


def test_bad_classes_and_values_show_in_their_row_alone(cuda_device):
    for v in (30, 5000):
        for t in (F32, HF):
            z, top, cls, y = _inputs(cuda_device, 9, v, 5, t, seed=8, ragged=False)
            want = loss.distill_loss(z, top, cls, y, reduction="none")
            cls[1, 2], y[2], cls[3, 0], top[4, 1], top[5, 0] = v, v, 2 ** 40, float("nan"), float("inf")
            z[6, v // 2], z[7, 0], y[8] = float("nan"), float("inf"), 2 ** 40
            leaf = z.detach().requires_grad_()
            rows = loss.distill_loss(leaf, top, cls, y, reduction="none")
            (g,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
            assert torch.isnan(rows[1:]).all() and torch.equal(rows[:1], want[:1])
            assert torch.isnan(g[1:]).any(1).all() and torch.isfinite(g[0]).all()
            assert torch.isnan(loss.distill_loss(z, top, cls, y))


def test_large_logits(cuda_device):
    for t in (F32, BF):
        z, top, cls, y = _inputs(cuda_device, 7, 1500, 9, t, seed=9, scale=300.0)
        _both(z, top, cls, y, 2.0, 0.5, "mean", "large")
    z = torch.full((2, 600), 3.0e38, device=cuda_device)
    z[:, 0] = -3.0e38
    cls = torch.tensor([[0, 1], [2, 3]], device=cuda_device)
    leaf = z.requires_grad_()
    rows = loss.distill_loss(leaf, torch.zeros(2, 2, device=cuda_device), cls, reduction="none", weight=1.0, temperature=4.0)
    (g,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    # the far class is 6e38 / T away: log q = -1.5e38, half of that counts, T^2 times
    assert not torch.isnan(rows).any() and torch.isfinite(g).all()


def test_strides_offsets_and_shapes(cuda_device):
    z, top, cls, y = _inputs(cuda_device, 12, 500, 6, BF, seed=10)
    want = loss.distill_loss(z, top, cls, y, reduction="none")
    for off, width in ((0, 504), (8, 520), (3, 509)):  # rows apart, in 16-byte units and out of them
        wide = torch.full((12, width), float("nan"), dtype=BF, device=cuda_device)
        wide[:, off:off + 500] = z
        _both(wide[:, off:off + 500], top, cls, y, 2.0, 0.5, "mean", f"offset {off}")
        assert torch.allclose(loss.distill_loss(wide[:, off:off + 500], top, cls, y, reduction="none"), want, rtol=1e-5)
    assert torch.equal(loss.distill_loss(z.view(3, 4, 500), top.view(3, 4, 6), cls.view(3, 4, 6), y.view(3, 4), reduction="none").view(12), want)
    assert torch.allclose(loss.distill_loss(z.t().contiguous().t(), top, cls, y, reduction="none"), want, rtol=1e-5)
    one = loss.distill_loss(z[0], top[0], cls[0], y[0], reduction="none")
    assert one.shape == () and torch.allclose(one, want[0], rtol=1e-5)
    leaf = z[:1].detach().float().requires_grad_()
    rows = loss.distill_loss(leaf.expand(12, 500), top, cls, y, reduction="none")
    (g,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    assert g.shape == (1, 500)
    assert loss.distill_loss(z[:, :500:2], top, cls.clamp(max=249), y.clamp(max=249)).shape == ()


def test_no_rows(cuda_device):
    leaf = torch.zeros(0, 30, device=cuda_device, requires_grad=True)
    top, cls = torch.zeros(0, 3, device=cuda_device), torch.zeros(0, 3, dtype=torch.int64, device=cuda_device)
    for red in ("mean", "sum", "none"):
        out = loss.distill_loss(leaf, top, cls, reduction=red)
        (g,) = torch.autograd.grad(out.sum(), leaf)
        assert g.shape == (0, 30) and out.sum() == 0


def test_larger(cuda_device):
    z, top, cls, y = _inputs(cuda_device, 1000, 32000, 64, BF, seed=11)
    a = _both(z, top, cls, y, 2.0, 0.6, "mean", "1000x32000")
    b = _both(z, top, cls, y, 2.0, 0.6, "mean", "1000x32000")
    assert torch.equal(a[0], b[0])


def test_past_two_to_the_31_elements(cuda_device):
    n, v = 33000, 65536  # rows and gradients of 4.3 GB
    z = torch.empty(n, v, dtype=BF, device=cuda_device)
    z[:] = torch.randn(v, device=cuda_device).to(BF)
    z[-3:] = torch.randn(3, v, device=cuda_device).to(BF)
    top = torch.randn(n, 4, device=cuda_device)
    cls = torch.randint(v, (n, 4), device=cuda_device)
    y = torch.randint(v, (n,), device=cuda_device)
    leaf = z.requires_grad_()
    rows = loss.distill_loss(leaf, top, cls, y, temperature=2.0, reduction="none")
    (g,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    pick = torch.tensor([0, 1, n // 2, n - 4, n - 3, n - 2, n - 1], device=cuda_device)
    want, tol, dz, edz = _define(z.detach()[pick], top[pick], cls[pick], y[pick], 2.0, 0.5, "none")
    assert ((rows.detach()[pick].double() - want).abs() <= tol + U * want.abs()).all()
    assert ((g[pick].double() - dz).abs() <= edz).all()


def test_second_derivative_is_refused(cuda_device):
    z, top, cls, y = _inputs(cuda_device, 4, 20, 3)
    out = loss.distill_loss(z.requires_grad_(), top, cls, y)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(out, z, create_graph=True)


def test_refusals(cuda_device):
    z, top, cls, y = _inputs(cuda_device, 4, 20, 3)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        loss.distill_loss(z.double(), top, cls, y)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        loss.distill_loss(z, top.double(), cls, y)
    with pytest.raises(RuntimeError, match="tensors on"):
        loss.distill_loss(z, top, cls.cpu(), y)
    with pytest.raises(RuntimeError, match="tensors on"):
        loss.distill_loss(z, top, cls, y.cpu())
    with pytest.raises(RuntimeError, match="at most 1024"):
        loss.distill_loss(z, torch.zeros(4, 1025, device=cuda_device), torch.zeros(4, 1025, dtype=torch.int64, device=cuda_device))


def test_captured_and_on_another_stream(cuda_device):
    z, top, cls, y = _inputs(cuda_device, 60, 1200, 8, BF, seed=12)
    leaf = z.detach().requires_grad_()

    def once():
        out = loss.distill_loss(leaf, top, cls, y, temperature=2.0)
        return (out.detach(), *torch.autograd.grad(out, leaf))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = once()
    torch.cuda.current_stream().wait_stream(side)
    here = once()
    assert all(torch.equal(p, q) for p, q in zip(there, here))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = once()
    with torch.no_grad():
        leaf.mul_(0.5)
        y.fill_(-100)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs, once()))


def test_padding_by_zero_class_and_by_lowest_value(cuda_device):
    """Entries padded with class 0 at -inf, or at the type's lowest value, take nothing off class 0."""
    for v, k in ((200, 40), (9000, 300)):
        z, top, cls, y = _inputs(cuda_device, 20, v, k, BF, HF, seed=13, ragged=False)
        for fill in (float("-inf"), torch.finfo(HF).min):
            t, c = top.clone(), cls.clone()
            t[:, k // 3:], c[:, k // 3:] = fill, 0
            short = _both(z, top[:, :k // 3], cls[:, :k // 3], y, 2.0, 0.5, "none", "short")
            leaf = z.detach().requires_grad_()
            rows = loss.distill_loss(leaf, t, c, y, temperature=2.0, weight=0.5, reduction="none")
            (g,) = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
            want, tol, dz, edz = _define(z, top[:, :k // 3], cls[:, :k // 3], y, 2.0, 0.5, "none")
            assert ((rows.detach().double() - want).abs() <= tol + U * want.abs()).all()
            assert ((g.double() - dz).abs() <= edz).all()
            assert torch.allclose(rows.detach(), short[0], rtol=1e-5)


def test_all_entries_one_class(cuda_device):
    """1024 entries of one class: p is spread over them, so sum p (log p - log q) is the class's -log q less p's entropy."""
    for v in (30, 3000):
        z, _, _, y = _inputs(cuda_device, 5, v, 3, F32, seed=14, ragged=False)
        cls, t = torch.full((5, 1024), 7, device=cuda_device), torch.randn(5, 1024, device=cuda_device)
        rows, g = _both(z, t, cls, y, 1.0, 1.0, "none", "one class")
        entropy = -(t.softmax(1) * t.log_softmax(1)).sum(1)
        one = loss.distill_loss(z, t[:, :1], cls[:, :1], y, weight=1.0, reduction="none")
        assert torch.allclose(rows + entropy, one, rtol=1e-5, atol=1e-5)
