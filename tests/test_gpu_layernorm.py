"""Layer norm on the GPU against float64.

u = 2^-24.  A row's sums are trees of at most ``depth`` additions on the way of a
term, each off by u of the partial sum, so by depth u of the sum of magnitudes in
all.  The bounds below follow the formula operation by operation: the mean, the
distances from it, their mean square, its inverse root (within 4 u), the products.
An output is rounded by half(t) of itself.
"""

from __future__ import annotations

import pytest
import torch

from omniwave_b200 import norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def _half(t):
    return U if t == F32 else torch.finfo(t).eps / 2


def _round(e, v, t):
    return e + _half(t) * 1.01 * (v.abs() + e) + (2.0 ** -25 if t == HF else 0.0)


def _depth(c):
    return 48 if c <= 8192 else c // 256 + 24


def _define(x, w, b, dn, eps):
    """Output, gradients and the bounds of their errors before the last rounding, in float64."""
    x, w = x.double(), w.double()
    c, d_ = x.shape[-1], _depth(x.shape[-1])
    rows = x.numel() // c
    m = x.mean(-1, keepdim=True)
    em = (d_ + 2) * U * x.abs().mean(-1, keepdim=True)
    d = x - m
    ed = em + U * (d.abs() + em)
    var = d.square().mean(-1, keepdim=True)
    # the squares are those of distances from the rounded mean, which is the same for the whole row: its own error enters squared
    own = U * (d.abs() + em)
    ev = 2 * (d.abs() * own).mean(-1, keepdim=True) + em ** 2 + own.square().mean(-1, keepdim=True) + (d_ + 4) * U * (var + em ** 2)
    r = (var + eps).rsqrt()
    er = ev / (2 * (var + eps)) * 1.01 + 4 * U  # relative
    assert (ev <= 0.01 * (var + eps)).all()
    hat = d * r
    eh = r * (ed + d.abs() * (er + 2 * U)) * 1.01
    n = hat * w
    en = eh * w.abs() + U * n.abs()
    if b is not None:
        n = n + b.double()
        en = en + U * (n.abs() + b.double().abs())
    out, tol = {"n": n}, {"n": en}
    if dn is not None:
        g = dn.double()
        u = g * w
        mu, mx = u.mean(-1, keepdim=True), (u * hat).mean(-1, keepdim=True)
        emu = (d_ + 3) * U * u.abs().mean(-1, keepdim=True)
        emx = (u.abs() * eh).mean(-1, keepdim=True) + (d_ + 4) * U * (u * hat).abs().mean(-1, keepdim=True)
        inner = U * u.abs() + emu + eh * (mx.abs() + emx) + hat.abs() * emx + 3 * U * (u.abs() + mu.abs() + (hat * mx).abs())
        out["dx"] = r * (u - mu - hat * mx)
        tol["dx"] = (er + U) * out["dx"].abs() + 1.01 * r * inner
        chain = rows // 148 + 96
        dims = tuple(range(x.dim() - 1))
        out["dw"], out["db"] = (g * hat).sum(dims), g.sum(dims)
        tol["dw"] = (g.abs() * eh).sum(dims) + (chain + 1) * U * (g.abs() * (hat.abs() + eh)).sum(dims)
        tol["db"] = chain * U * g.abs().sum(dims)
    return out, tol


def _ok(got, want, tol, where):
    err = (got.double() - want).abs()
    tol = _round(tol, want, got.dtype)
    assert (err <= tol).all(), f"{where}: worst {(err / tol.clamp(min=1e-300)).max().item():.2f} of the bound"


def _inputs(dev, shape, t, wt, seed=0, shift=0.3):
    g = torch.Generator(device=dev).manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device=dev)

    c = shape[-1]
    return (r(*shape) + shift).to(t), (1 + 0.2 * r(c)).to(wt), (0.3 * r(c)).to(wt), r(*shape)


def _both(x, w, b, dn, where, eps=1e-5, out=None):
    out = out or x.dtype
    dn = dn.to(out)
    want, tol = _define(x, w, b, dn, eps)
    with torch.no_grad():
        plain = norm.layer_norm(x, w, b, eps=eps, out_dtype=out)
    assert plain.dtype == out and plain.shape == x.shape
    _ok(plain, want["n"], tol["n"], f"{where} n")
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    n = norm.layer_norm(leaves[0], leaves[1], leaves[2] if b is not None else None, eps=eps, out_dtype=out)
    assert torch.equal(n, plain)
    grads = torch.autograd.grad(n, leaves, dn)
    for k, g, leaf in zip(("dx", "dw", "db"), grads, leaves):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        _ok(g, want[k], tol[k], f"{where} {k}")
    return grads


CHANNELS = [1, 2, 7, 8, 16, 63, 64, 65, 70, 128, 129, 256, 264, 511, 512, 520, 777, 1000, 1024, 1032, 2048, 2056, 4096, 4104, 5001,
            8192, 8193, 8200, 20000]


@pytest.mark.parametrize("c", CHANNELS)
@pytest.mark.parametrize("t,out,wt", [(F32, F32, F32), (F32, BF, F32), (BF, BF, F32), (HF, HF, HF), (BF, F32, BF)],
                         ids=["f32", "f32-bf16", "bf16", "f16", "bf16-f32"])
def test_channels(cuda_device, c, t, out, wt):
    for rows in (1, 3, 40):
        x, w, b, dn = _inputs(cuda_device, (rows, c), t, wt, seed=rows)
        if c == 1:  # nothing but its mean: the norm is 0 and the bias is left
            assert torch.equal(norm.layer_norm(x, w, b, out_dtype=out), b.to(out).expand(rows, 1))
            continue
        _both(x, w, b, dn, f"{rows}x{c}", out=out)
        _both(x, w, None, dn, f"{rows}x{c} no bias", out=out)


@pytest.mark.parametrize("shape", [(128, 3136, 128), (64, 196, 1024), (33, 49, 777), (100_000, 24), (2000, 4096), (700, 8192), (50, 12345)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("t", [F32, BF], ids=["f32", "bf16"])
def test_larger(cuda_device, shape, t):
    x, w, b, dn = _inputs(cuda_device, shape, t, F32, seed=1)
    first = _both(x, w, b, dn, str(shape))
    second = _both(x, w, b, dn, str(shape))
    assert all(torch.equal(p, q) for p, q in zip(first, second))  # bit for bit


@pytest.mark.parametrize("shape", [(100_001, 25), (50_000, 56), (40_003, 70), (20_001, 131), (9001, 311), (10_000, 400), (4001, 777),
                                   (3001, 888), (2600, 1000), (1701, 1501), (1301, 2000), (1001, 3001), (901, 3504), (501, 5001),
                                   (403, 7016)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("t,out", [(F32, F32), (F32, HF), (BF, BF), (HF, HF)], ids=["f32", "f32-f16", "bf16", "f16"])
def test_many_rows(cuda_device, shape, t, out):
    """Rows enough for the streaming kernels: whole vectors, part of a split, single channels, a last unit that is not whole."""
    x, w, b, dn = _inputs(cuda_device, shape, t, F32, seed=11)
    first = _both(x, w, b, dn, str(shape), out=out)
    assert all(torch.equal(p, q) for p, q in zip(first, _both(x, w, b, dn, str(shape), out=out)))
    # the bytes around the arrays' ends are nobody's business: a view that ends inside a larger array
    flat = torch.full((x.numel() + 64,), float("nan"), dtype=t, device=cuda_device)
    inner = flat[:x.numel()].view(shape).copy_(x)
    assert torch.equal(norm.layer_norm(inner, w, b, out_dtype=out), norm.layer_norm(x, w, b, out_dtype=out))


def test_rows_far_from_zero(cuda_device):
    """The variance survives a mean a thousand times the deviation, and one channel a thousand times the others."""
    for c in (64, 777, 1024):
        x, w, b, dn = _inputs(cuda_device, (50, c), F32, F32, seed=2, shift=1000.0)
        _both(x, w, b, dn, f"mean {c}")
        x, w, b, dn = _inputs(cuda_device, (50, c), F32, F32, seed=3)
        x[:, 0] = 1000.0
        _both(x, w, b, dn, f"channel {c}")


def test_constant_rows_and_eps(cuda_device):
    x = torch.full((5, 96), 3.0, device=cuda_device)
    w, b = torch.full((96,), 2.0, device=cuda_device), torch.full((96,), 0.5, device=cuda_device)
    assert torch.equal(norm.layer_norm(x, w, b), b.expand(5, 96))
    x[:, ::2] = -3.0  # mean 0, variance 9
    n = norm.layer_norm(x, w, None, eps=7.0)
    assert torch.equal(n, torch.sign(x) * 1.5)  # 3 / 4 * 2


def test_what_is_not_finite_stays_in_its_row(cuda_device):
    for c in (70, 512, 9000):
        for t in (F32, BF):
            x, w, b, dn = _inputs(cuda_device, (20, c), t, F32, seed=4)
            want = norm.layer_norm(x, w, b)
            x[3, c // 2], x[7, 0], x[8, c - 1] = float("nan"), float("inf"), float("-inf")
            n = norm.layer_norm(x, w, b)
            bad = torch.zeros(20, dtype=torch.bool, device=cuda_device)
            bad[[3, 7, 8]] = True
            assert torch.isnan(n[bad]).any(-1).all() and torch.equal(n[~bad], want[~bad])
            leaf = x.detach().requires_grad_()
            (dx,) = torch.autograd.grad(norm.layer_norm(leaf, w, b), leaf, dn.to(t))
            assert torch.isnan(dx[bad]).any(-1).all() and torch.isfinite(dx[~bad]).all()


def test_offsets_strides_and_shapes(cuda_device):
    x, w, b, dn = _inputs(cuda_device, (12, 5, 96), BF, F32, seed=5)
    want = norm.layer_norm(x, w, b)
    flat = torch.zeros(x.numel() + 3, dtype=BF, device=cuda_device)
    for off in (1, 3):  # rows that are no 16-byte units
        xo = flat[off:off + x.numel()].view(x.shape).copy_(x)
        got = norm.layer_norm(xo, w, b)
        assert (got.double() - want.double()).abs().max() <= 2.0 ** -6  # another order of the sums: one step of values up to 4
        wo = torch.zeros(97, device=cuda_device)
        wo[1:] = w
        _both(xo, wo[1:], b, dn, f"offset {off}")
    assert torch.equal(norm.layer_norm(x.transpose(0, 1), w, b), want.transpose(0, 1))
    wide = torch.zeros(60, 200, dtype=BF, device=cuda_device)
    wide[:, 8:104] = x.view(60, 96)
    assert torch.equal(norm.layer_norm(wide[:, 8:104], w, b), want.view(60, 96))
    assert torch.equal(norm.layer_norm(x[0, 0], w, b), want[0, 0])
    one = x[:1, :1].detach().float().requires_grad_()
    n = norm.layer_norm(one.expand(12, 5, 96), w, b)
    (g,) = torch.autograd.grad(n, one, torch.ones_like(n))  # the broadcast row gets the sum
    want_g, tol = _define(one.detach().expand(12, 5, 96), w, b, torch.ones(12, 5, 96, device=cuda_device), 1e-5)
    assert ((g.double() - want_g["dx"].sum((0, 1), keepdim=True)).abs()
            <= (tol["dx"] + 64 * U * want_g["dx"].abs()).sum((0, 1), keepdim=True) + 1e-12).all()


def test_empty_and_partial_gradients(cuda_device):
    x, w, b, dn = _inputs(cuda_device, (6, 40), F32, F32, seed=6)
    e = torch.zeros(0, 40, device=cuda_device, requires_grad=True)
    wl, bl, xl = (t.detach().requires_grad_() for t in (w, b, x))
    n = norm.layer_norm(e, wl, bl)
    ge = torch.autograd.grad(n.sum(), [e, wl, bl])
    assert n.shape == (0, 40) and ge[0].shape == (0, 40) and (ge[1] == 0).all() and (ge[2] == 0).all()
    full = torch.autograd.grad(norm.layer_norm(xl, wl, bl), [xl, wl, bl], dn)
    for i, leaf in enumerate((xl, wl, bl)):
        args = [x, w, b]
        args[i] = leaf
        (one,) = torch.autograd.grad(norm.layer_norm(*args), leaf, dn)
        assert torch.equal(one, full[i])


def test_gradient_against_differences(cuda_device):
    x, w, b, dn = _inputs(cuda_device, (9, 56), F32, F32, seed=7)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(norm.layer_norm(*leaves), leaves, dn)
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    way = [torch.randn(t.shape, generator=gen, device=cuda_device).double() for t in leaves]

    def loss(s):
        a, c, d = [t.double() + s * v for t, v in zip((x, w, b), way)]
        a = a - a.mean(-1, keepdim=True)
        return ((a * (a.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * c + d) * dn.double()).sum()

    want = float((loss(1e-5) - loss(-1e-5)) / 2e-5)
    got = float(sum((p.double() * v).sum() for p, v in zip(grads, way)))
    size = float(sum((p.double() * v).abs().sum() for p, v in zip(grads, way)))
    assert abs(got - want) <= 100 * U * size + 1e-7 * size  # a gradient is within 100 u of its terms here; the quotient's own error


def test_autocast_gives_its_type(cuda_device):
    x, w, b, _ = _inputs(cuda_device, (4, 32), F32, F32)
    with torch.autocast("cuda", dtype=BF):
        assert norm.layer_norm(x, w, b).dtype == BF
        assert norm.layer_norm(x, w, b, out_dtype=F32).dtype == F32


def test_second_derivative_is_refused(cuda_device):
    x, w, b, _ = _inputs(cuda_device, (4, 32), F32, F32)
    n = norm.layer_norm(x.requires_grad_(), w, b)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(n.sum(), x, create_graph=True)


def test_refusals(cuda_device):
    x, w = torch.zeros(4, 16, device=cuda_device), torch.zeros(16, device=cuda_device)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        norm.layer_norm(x.double(), w)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        norm.layer_norm(x, w, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="tensors on"):
        norm.layer_norm(x, w, w.cpu())


def test_captured_and_on_another_stream(cuda_device):
    x, w, b, dn = _inputs(cuda_device, (300, 200), BF, F32, seed=9)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]

    def once():
        n = norm.layer_norm(*leaves)
        return (n.detach(), *torch.autograd.grad(n, leaves, dn.to(BF)))

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
        leaves[0].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs, once()))


def test_past_two_to_the_31_elements(cuda_device):
    n, c = 2_200_000, 1000  # 4.4 GB in 16 bits
    x = torch.empty(n, c, dtype=BF, device=cuda_device)
    x[:] = torch.randn(c, device=cuda_device).to(BF)
    x[-40:] = torch.randn(40, c, device=cuda_device).to(BF)
    w, b = torch.randn(c, device=cuda_device), torch.randn(c, device=cuda_device)
    leaf = x.requires_grad_()
    y = norm.layer_norm(leaf, w, b)
    pick = torch.tensor([0, 1, n // 2, *range(n - 41, n)], device=cuda_device)
    dn = torch.zeros_like(x)
    dn[pick] = torch.randn(len(pick), c, device=cuda_device).to(BF)
    (dx,) = torch.autograd.grad(y, leaf, dn)
    want, tol = _define(x.detach()[pick], w, b, dn[pick], 1e-5)
    _ok(y.detach()[pick], want["n"], tol["n"], "n")
    _ok(dx[pick], want["dx"], tol["dx"], "dx")
    rest = torch.ones(n, dtype=torch.bool, device=cuda_device)
    rest[pick] = False
    assert not dx[rest][:: 1000].any()


def test_two_captured_graphs_and_a_wait_that_gives_up(cuda_device):
    """Two graphs replayed in turn do not share what they work in; a wait that runs out is reported, and the next call is right."""
    from omniwave_b200 import _lib

    x, w, b, dn = _inputs(cuda_device, (4000, 1024), BF, F32, seed=10)
    dn = dn.to(BF)

    def once(t):
        leaves = [v.detach().requires_grad_() for v in (t, w, b)]
        n = norm.layer_norm(*leaves)
        return (n.detach(), *torch.autograd.grad(n, leaves, dn))

    want = [once(x), once(x * 2)]
    graphs, outs = [], []
    y = x * 2
    for t in (x, y):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(once(t))
        graphs.append(g)
    for i in (0, 1, 0):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs[i], want[i]))
    lib = _lib.load()
    try:
        assert lib.ow_debug_wait_probe(1_000_000) == 0
        once(x)
        torch.cuda.synchronize()
    finally:
        lib.ow_debug_wait_probe(0)
    assert _lib.device_fault(0, reset=True) == 1
    assert all(torch.equal(p, q) for p, q in zip(once(x), want[0]))
