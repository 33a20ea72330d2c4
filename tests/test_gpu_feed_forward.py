"""The gated feed-forward block on the GPU against float64.

Errors are carried along with the values, operation by operation (``Num``): a
matrix product of 16-bit operands sums exact products in f32, in any order, within
(terms + 8) u of the sum of their magnitudes; elementwise operations round once in
f32; a 16-bit result is off by half(t) of itself.  The activations are within 8 u
(|z| + 1) of theirs, gelu's bf16 tail within 4e-4 of itself; slopes change by at
most 0.8 |dz| (silu'' <= 0.5, gelu'' <= 0.8), values by 1.13 |dz|.  The backward
holds act(g) and u act'(g) in 16 bits, which is no further off than from g and u in
16 bits (|act(g)| <= |g|); dh may be rounded to 16 bits before the gate's formula,
and the biases' gradients are sums of dg and du that may have been.
"""

from __future__ import annotations

import pytest
import torch

from omniwave_b200 import distill_loss, feed_forward, layer_norm, linear
from omniwave_b200.train import TrainStep

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def _half(t):
    return U if t == F32 else torch.finfo(t).eps / 2


class Num:
    """A value and the bound of its error."""

    def __init__(self, v, e=None):
        self.v, self.e = v.double(), torch.zeros_like(v, dtype=torch.float64) if e is None else e

    def size(self):
        return self.v.abs() + self.e

    def __mul__(self, o):
        e = self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e
        return Num(self.v * o.v, e + U * self.size() * o.size())

    def __add__(self, o):
        v = self.v + o.v
        e = self.e + o.e
        return Num(v, e + U * (v.abs() + e))

    def __matmul__(self, o):
        e = self.v.abs() @ o.e + self.e @ o.size()
        return Num(self.v @ o.v, e + (self.v.shape[1] + 8) * U * (self.size() @ o.size()))

    def t(self):
        return Num(self.v.t(), self.e.t())

    def sum0(self):
        return Num(self.v.sum(0), self.e.sum(0) + (self.v.shape[0] + 8) * U * self.size().sum(0))

    def round(self, t):
        return Num(self.v, self.e + _half(t) * 1.01 * self.size() + (2.0 ** -25 if t == HF else 0.0))


def _act(z, act, t):
    v = z.v
    own = 8 * U * (v.abs() + 1)
    if act == "none":
        return z, Num(torch.ones_like(v))
    if act == "relu":  # tested where the sums are exact, or far from 0
        assert ((v.abs() > z.e) | (v == 0)).all()
        return Num(v.clamp(min=0), torch.where(v > 0, z.e, 0.0)), Num((v > 0).double())
    if act == "silu":
        s = torch.sigmoid(v)
        a, d = v * s, s * (1 + v * (1 - s))
    else:
        cdf = 0.5 * (1 + torch.erf(v / 2 ** 0.5))
        a, d = v * cdf, cdf + v * torch.exp(-v * v / 2) / (2 * torch.pi) ** 0.5
        own = own + (4e-4 if t == BF else 1e-5) * v.abs() * 0.5 * torch.erfc(v.abs() / 2 ** 0.5)
    return Num(a, 1.13 * z.e + own), Num(d, 0.8 * z.e + own)


def _define(x, wg, wu, wd, bg, bu, bd, r, dy, act, t):
    x, wg, wu, wd, dy = (Num(v) for v in (x, wg, wu, wd, dy))
    g, u = x @ wg.t(), x @ wu.t()
    if bg is not None:
        g = g + Num(bg)
    if bu is not None:
        u = u + Num(bu)
    if act == "relu":
        g.e = torch.zeros_like(g.e)  # inputs chosen so that g's sums are exact
    h = (_act(g, act, t)[0] * u).round(t)
    y = h @ wd.t()
    if bd is not None:
        y = y + Num(bd)
    if r is not None:
        y = y + Num(r)
    out = {"y": y}
    # relu's g are exact multiples of 2^-9 (0 stays 0, nothing is subnormal)
    g16, u16 = Num(g.v, _half(t) * 1.01 * g.v.abs()) if act == "relu" else g.round(t), u.round(t)
    a, s = _act(g16, act, t)
    dh = (dy @ wd).round(t)
    dg, du = dh * u16 * s, dh * a
    dg, du = dg.round(t), du.round(t)
    out["bg"], out["bu"], out["bd"] = dg.sum0(), du.sum0(), dy.sum0()  # of dg and du as they are rounded, or before
    out["x"] = dg @ wg + du @ wu
    out["wg"], out["wu"], out["wd"] = dg.t() @ x, du.t() @ x, dy.t() @ h
    return out


def _ok(got, want, where):
    want = want.round(got.dtype)
    err = (got.double() - want.v).abs()
    assert got.shape == want.v.shape and (err <= want.e).all(), f"{where}: worst {(err / want.e.clamp(min=1e-300)).max().item():.2f} of the bound"


def _inputs(dev, m, k, f, n, t, act="silu", seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device=dev)

    x, wg, wu, wd = r(m, k).to(t), (r(f, k) * k ** -0.5).to(t), (r(f, k) * k ** -0.5).to(t), (r(n, f) * f ** -0.5).to(t)
    bg = (r(f) * 0.3).to(t)
    if act == "relu":  # eighths times 64ths: sums of products are exact in f32, so g's sign is; biases of 512ths too
        x, wg = (x.float() * 8).round().clamp(-8, 8).div(8).to(t), (wg.float() * 64).round().clamp(-8, 8).div(64).to(t)
        bg = (bg.float() * 64).round().clamp(-64, 64).div(64).to(t)
    return dict(x=x, wg=wg, wu=wu, wd=wd, bg=bg, bu=(r(f) * 0.3).to(t), bd=(r(n) * 0.3).to(t), r=r(m, n).to(t)), r(m, n).to(t)


def _run(a, act):
    return feed_forward.gated_feed_forward(a["x"], a["wg"], a["wu"], a["wd"], gate_bias=a.get("bg"), up_bias=a.get("bu"),
                                           down_bias=a.get("bd"), activation=act, residual=a.get("r"))


def _both(a, dy, act, where):
    t = a["x"].dtype
    with torch.no_grad():
        plain = _run(a, act)
    leaves = {k: v.detach().requires_grad_() for k, v in a.items()}
    y = _run(leaves, act)
    assert torch.equal(y, plain) and y.dtype == t
    want = _define(*(a.get(k) for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd", "r")), dy, act, t)
    _ok(plain, want["y"], f"{where} y")
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    for k, g in grads.items():
        assert g.dtype == a[k].dtype
        if k == "r":
            assert torch.equal(g, dy)
        else:
            _ok(g, want[k], f"{where} d{k}")
    return grads


SHAPES = [(1, 8, 8, 8), (1, 1024, 2048, 1024), (2, 64, 7, 33), (3, 70, 33, 70), (5, 2048, 16, 24), (8, 300, 129, 64), (9, 64, 64, 64),
          (17, 8, 8, 8), (31, 72, 40, 16), (40, 63, 45, 20), (128, 64, 64, 64), (129, 65, 257, 65), (200, 1000, 24, 8), (256, 512, 1024, 256),
          (300, 129, 130, 129), (1000, 48, 128, 48), (333, 2048, 300, 100), (60, 4096, 200, 64), (2500, 72, 40, 72)]


@pytest.mark.parametrize("m,k,f,n", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
@pytest.mark.parametrize("t", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("act,drop", [("silu", ""), ("silu", "bg bu bd r"), ("gelu", "bu"), ("none", "bg bd"), ("relu", "r")])
def test_forward_and_gradients(cuda_device, m, k, f, n, t, act, drop):
    a, dy = _inputs(cuda_device, m, k, f, n, t, act)
    a = {key: v for key, v in a.items() if key not in drop.split()}
    _both(a, dy, act, f"{m}x{k}x{f}x{n} {act}")


@pytest.mark.parametrize("m,k,f,n,act", [(25088, 512, 1024, 512, "gelu"), (12544, 1024, 2048, 1024, "silu"), (4096, 256, 2048, 256, "silu"),
                                         (50_000, 64, 128, 64, "none"), (777, 1000, 2040, 136, "silu"), (2048, 2056, 264, 2056, "gelu")])
def test_larger(cuda_device, m, k, f, n, act):
    a, dy = _inputs(cuda_device, m, k, f, n, BF, act, seed=1)
    first = _both(a, dy, act, f"{m}x{k}x{f}x{n}")
    second = _both(a, dy, act, f"{m}x{k}x{f}x{n}")
    assert all(torch.equal(first[key], second[key]) for key in first)  # bit for bit


@pytest.mark.parametrize("k", [8, 56, 72, 1000, 2048, 8192])
@pytest.mark.parametrize("t", [BF, HF], ids=["bf16", "f16"])
def test_a_few_rows(cuda_device, k, t):
    # around the row counts where the kernel changes; hidden features that do not fill a warp's 8; long k, that is split
    for m in (1, 7, 8, 9, 16, 17, 32, 33):
        for f in (1, 8, 9, 64, 1000):
            a, dy = _inputs(cuda_device, m, k, f, 24, t, seed=m)
            want = _define(*(a[key] for key in ("x", "wg", "wu", "wd", "bg", "bu", "bd", "r")), dy, "silu", t)["y"]
            y = _run(a, "silu")
            _ok(y, want, f"{m}x{k}x{f}")
            assert torch.equal(y, _run(a, "silu"))
            for pad in (8, 3):  # rows that lie apart, in 16-byte units and out of them
                b = dict(a)
                for key in ("x", "wg", "wu", "wd", "r"):
                    wide = torch.full((a[key].shape[0], a[key].shape[1] + pad), float("nan"), dtype=t, device=cuda_device)
                    wide[:, :a[key].shape[1]] = a[key]
                    b[key] = wide[:, :a[key].shape[1]]
                _ok(_run(b, "silu"), want, f"{m}x{k}x{f} pad {pad}")


def test_strides_offsets_and_shapes(cuda_device):
    a, dy = _inputs(cuda_device, 60, 96, 40, 48, BF, seed=2)
    want = _run(a, "silu")
    packed = torch.cat([a["wg"], a["wu"]])
    assert torch.equal(_run(a | {"wg": packed[:40], "wu": packed[40:]}, "silu"), want)
    wide = torch.zeros(60, 200, dtype=BF, device=cuda_device)
    for off in (0, 8, 3):
        wide[:, off:off + 96] = a["x"]
        assert torch.equal(_run(a | {"x": wide[:, off:off + 96]}, "silu"), want)
    assert torch.equal(_run(a | {"x": a["x"].view(3, 4, 5, 96), "r": a["r"].view(3, 4, 5, 48)}, "silu").view(60, 48), want)
    assert torch.equal(_run(a | {"x": a["x"].t().contiguous().t(), "wd": a["wd"].t().contiguous().t()}, "silu"), want)
    assert _run({key: v for key, v in a.items() if key != "r"} | {"x": a["x"][0]}, "silu").shape == (48,)
    p = packed.clone().requires_grad_()  # the gradient of a packed weight
    (gp,) = torch.autograd.grad(_run(a | {"wg": p[:40], "wu": p[40:]}, "silu"), p, dy)
    wg, wu = a["wg"].detach().requires_grad_(), a["wu"].detach().requires_grad_()
    g2 = torch.autograd.grad(_run(a | {"wg": wg, "wu": wu}, "silu"), [wg, wu], dy)
    assert torch.equal(gp, torch.cat(g2))
    one = a["x"][:1].clone().requires_grad_()
    y = _run(a | {"x": one.expand(60, 96)}, "silu")
    (g,) = torch.autograd.grad(y, one, dy)
    x = a["x"][:1].expand(60, 96).contiguous().requires_grad_()
    (gx,) = torch.autograd.grad(_run(a | {"x": x}, "silu"), x, dy)
    assert (g.double() - gx.double().sum(0, keepdim=True)).abs().max() <= 2 * _half(BF) * gx.double().abs().sum(0).max()


def test_one_weight_for_gate_and_up(cuda_device):
    a, dy = _inputs(cuda_device, 50, 64, 32, 16, HF, seed=3)
    w = a["wg"].detach().requires_grad_()
    (g,) = torch.autograd.grad(_run(a | {"wg": w, "wu": w}, "silu"), w, dy)
    wg, wu = a["wg"].detach().requires_grad_(), a["wg"].detach().clone().requires_grad_()
    g2 = torch.autograd.grad(_run(a | {"wg": wg, "wu": wu}, "silu"), [wg, wu], dy)
    assert torch.equal(g, g2[0] + g2[1])


def test_autocast_with_f32_parameters(cuda_device):
    torch.manual_seed(0)
    m, k, f, n = 500, 72, 104, 72
    a, dy = _inputs(cuda_device, m, k, f, n, F32, seed=4)
    leaves = {key: v.requires_grad_() for key, v in a.items()}
    with torch.autocast("cuda", dtype=BF):
        y = _run(leaves, "gelu")
        assert y.dtype == BF
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.to(BF))))
    held = {key: (v.detach() if key[0] == "b" else v.detach().to(BF)) for key, v in a.items()}
    want = _define(*(held[key] for key in ("x", "wg", "wu", "wd", "bg", "bu", "bd", "r")), dy.to(BF), "gelu", BF)
    _ok(y.detach(), want["y"], "y")
    for key, g in grads.items():
        assert g.dtype == F32
        if key == "x":  # rounded to 16 bits before it is cast up
            _ok(g, want["x"].round(BF), "dx")
        elif key != "r":
            _ok(g, want[key], f"d{key}")


def test_gradients_against_differences(cuda_device):
    for act in ("silu", "gelu", "none"):
        a, dy = _inputs(cuda_device, 40, 24, 32, 16, HF, act, seed=5)
        leaves = {key: v.detach().requires_grad_() for key, v in a.items()}
        grads = torch.autograd.grad(_run(leaves, act), list(leaves.values()), dy)
        gen = torch.Generator(device=cuda_device).manual_seed(1)
        way = [torch.randn(v.shape, generator=gen, device=cuda_device).double() for v in a.values()]

        def loss(s):
            x, wg, wu, wd, bg, bu, bd, r = [v.double() + s * w for v, w in zip(a.values(), way)]
            act_ = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "none": lambda v: v}[act]
            return (((act_(x @ wg.t() + bg) * (x @ wu.t() + bu)) @ wd.t() + bd + r) * dy.double()).sum()

        want = float((loss(1e-5) - loss(-1e-5)) / 2e-5)
        got = float(sum((p.double() * v).sum() for p, v in zip(grads, way)))
        size = float(sum((p.double() * v).abs().sum() for p, v in zip(grads, way)))
        assert abs(got - want) <= 6 * _half(HF) * size  # g, u, h, dh, dg or du and each gradient rounded to f16


def test_what_is_not_finite_stays_in_its_row(cuda_device):
    for m in (4, 30, 200):
        for k in (64, 70):
            a, _ = _inputs(cuda_device, m, k, 50, 24, BF)
            want = _run(a, "silu")
            a["x"][m // 2, k // 3] = float("nan")
            y = _run(a, "silu")
            rows = torch.arange(m, device=cuda_device) != m // 2
            assert torch.isnan(y[m // 2]).all() and torch.equal(y[rows], want[rows])


def test_f16_projections_beyond_its_range(cuda_device):
    """A gate of -1.4e6 is 0, and so is its slope; the kept projections stay finite."""
    for m in (5, 100):
        x = torch.full((m, 16), -300.0, dtype=HF, device=cuda_device, requires_grad=True)
        wg = torch.full((8, 16), 300.0, dtype=HF, device=cuda_device)
        wd = torch.ones(4, 8, dtype=HF, device=cuda_device)
        for act in ("relu", "silu", "gelu"):
            y = feed_forward.gated_feed_forward(x, wg, wg, wd, activation=act)
            (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
            assert (y == 0).all() and (g == 0).all()


def test_empty_and_partial_gradients(cuda_device):
    for m in (20, 300):
        a, dy = _inputs(cuda_device, m, 24, 40, 16, BF)
        leaves = {key: v.detach().requires_grad_() for key, v in a.items()}
        full = dict(zip(leaves, torch.autograd.grad(_run(leaves, "silu"), list(leaves.values()), dy)))
        for key in a:
            leaf = a[key].detach().requires_grad_()
            (one,) = torch.autograd.grad(_run(a | {key: leaf}, "silu"), leaf, dy)
            assert torch.equal(one, full[key]), key
        two = {key: a[key].detach().requires_grad_() for key in ("wu", "bd")}
        got = torch.autograd.grad(_run({key: v for key, v in (a | two).items() if key != "bg"}, "silu"), list(two.values()), dy)
        assert torch.equal(got[1], full["bd"])
    e = {**a, "x": torch.zeros(0, 24, dtype=BF, device=cuda_device), "r": torch.zeros(0, 16, dtype=BF, device=cuda_device)}
    leaves = {key: v.detach().requires_grad_() for key, v in e.items()}
    y = _run(leaves, "silu")
    grads = torch.autograd.grad(y.sum(), list(leaves.values()))
    assert y.shape == (0, 16) and all((g == 0).all() and g.shape == v.shape for g, v in zip(grads, leaves.values()))


def test_second_derivative_is_refused(cuda_device):
    a, _ = _inputs(cuda_device, 20, 16, 8, 8, BF)
    x = a["x"].requires_grad_()
    y = _run(a, "silu")
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_refusals(cuda_device):
    a, _ = _inputs(cuda_device, 4, 16, 8, 8, F32)
    with pytest.raises(RuntimeError, match="not 16-bit"):
        _run(a, "silu")
    b = {key: v.to(BF) for key, v in a.items()}
    for key in ("wg", "wu", "wd", "r"):
        with pytest.raises(RuntimeError, match="without autocast"):
            _run(b | {key: a[key]}, "silu")
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        _run(b | {"bu": b["bu"].double()}, "silu")
    with pytest.raises(RuntimeError, match="tensors on"):
        _run(b | {"wd": b["wd"].cpu()}, "silu")


def test_captured_and_on_another_stream(cuda_device):
    for m in (8, 300):
        a, dy = _inputs(cuda_device, m, 128, 96, 64, BF, seed=6)
        leaves = {key: v.detach().requires_grad_() for key, v in a.items()}

        def once():
            y = _run(leaves, "silu")
            return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), dy))

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
            leaves["x"].mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, once()))


def test_a_wait_that_gives_up_is_reported(cuda_device):
    from omniwave_b200 import _lib

    a, dy = _inputs(cuda_device, 300, 128, 96, 64, BF, seed=7)
    leaves = {key: v.detach().requires_grad_() for key, v in a.items()}

    def once():
        y = _run(leaves, "silu")
        return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), dy))

    want = once()
    lib = _lib.load()
    try:
        assert lib.ow_debug_wait_probe(1_000_000) == 0
        once()
        torch.cuda.synchronize()
    finally:
        lib.ow_debug_wait_probe(0)
    assert _lib.device_fault(0, reset=True) == 1
    assert all(torch.equal(p, q) for p, q in zip(once(), want))


def test_two_threads(cuda_device):
    """Calls from two threads on streams of their own, forward and backward."""
    import threading

    cases = [_inputs(cuda_device, m, 128, 200, 64, BF, seed=m) for m in (40, 700)]

    def once(a, dy):
        leaves = {key: v.detach().requires_grad_() for key, v in a.items()}
        y = _run(leaves, "gelu")
        return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), dy))

    want = [once(*c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = once(*cases[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


class _Net(torch.nn.Module):
    """norm -> feed-forward -> residual, twice, and a head: the operators as a model has them."""

    def __init__(self, c, f, classes):
        super().__init__()
        p = torch.nn.Parameter
        self.ln = torch.nn.ModuleList(torch.nn.LayerNorm(c) for _ in range(2))
        self.w = torch.nn.ParameterList(p(torch.randn(*s) * s[1] ** -0.5) for _ in range(2) for s in ((f, c), (f, c), (c, f)))
        self.b = torch.nn.ParameterList(p(torch.randn(s) * 0.1) for _ in range(2) for s in (f, f, c))
        self.head = torch.nn.Linear(c, classes)

    def forward(self, x, own=True):
        for i, ln in enumerate(self.ln):
            wg, wu, wd = self.w[3 * i:3 * i + 3]
            bg, bu, bd = self.b[3 * i:3 * i + 3]
            if own:
                n = layer_norm(x, ln.weight, ln.bias, eps=ln.eps)
                x = feed_forward.gated_feed_forward(n, wg, wu, wd, gate_bias=bg, up_bias=bu, down_bias=bd, residual=x)
            else:
                n = torch.nn.functional.layer_norm(x, x.shape[-1:], ln.weight, ln.bias, ln.eps)
                lin = torch.nn.functional.linear
                x = lin(torch.nn.functional.silu(lin(n, wg, bg)) * lin(n, wu, bu), wd, bd) + x
        x = x.mean(1)
        return linear.linear(x, self.head.weight, self.head.bias) if own else self.head(x)


def _net_loss(net, x, y, top, cls, temp, weight):
    z = net(x, own=False)
    lp = (top.double() / temp).log_softmax(1)
    soft = (lp.exp() * (lp - (z / temp).log_softmax(1).gather(1, cls))).sum(1).mean() * temp ** 2
    return weight * soft + (1 - weight) * torch.nn.functional.cross_entropy(z, y)


def test_together_in_a_training_step(cuda_device):
    """Norm, feed-forward, head and loss under autocast: the loss and every gradient against the same model in float64."""
    torch.manual_seed(1)
    net = _Net(96, 160, 50).to(cuda_device)
    x, y = torch.randn(32, 9, 96, device=cuda_device), torch.randint(50, (32,), device=cuda_device)
    top, cls = (torch.randn(32, 50, device=cuda_device) * 2).topk(8, 1)
    with torch.autocast("cuda", dtype=BF):
        z = net(x)
        value = distill_loss(z, top, cls, y, temperature=2.0, weight=0.6)
    grads = torch.autograd.grad(value, list(net.parameters()))
    exact = _Net(96, 160, 50).to(cuda_device).double()
    exact.load_state_dict({k: v.double() for k, v in net.state_dict().items()})
    want = _net_loss(exact, x.double(), y, top, cls, 2.0, 0.6)
    exact_grads = torch.autograd.grad(want, list(exact.parameters()))
    # about ten 16-bit roundings stand on the way to a gradient, each 2^-8 of its value at most and independent of the others
    assert abs(value.item() - want.item()) <= 10 * 2.0 ** -8 * want.item()
    for (name, _), g, w in zip(net.named_parameters(), grads, exact_grads):
        assert g.dtype == F32
        assert float((g.double() - w).norm()) <= 10 * 2.0 ** -8 * float(w.norm()), name


def test_training_step_with_a_teacher_eager_and_captured(cuda_device):
    torch.manual_seed(2)
    x, y = torch.randn(16, 9, 96, device=cuda_device), torch.randint(50, (16,), device=cuda_device)
    teacher = (torch.randn(16, 50, device=cuda_device) * 2).topk(8, 1)
    state = _Net(96, 160, 50).state_dict()
    losses = []
    for graphed in (False, True):
        net = _Net(96, 160, 50).to(cuda_device)
        net.load_state_dict(state)
        step = TrainStep(net, optimizer="fused", cuda_graph=graphed, graph_warmup=2, distill_weight=0.7, distill_temperature=2.0)
        losses.append([float(step.step(x, y, teacher=teacher)) for _ in range(5)])
        step.check_finite()
        if graphed:
            with pytest.raises(ValueError, match="captured with a teacher"):
                step.step(x, y)
    assert losses[0] == losses[1]
    with torch.autocast("cuda", dtype=BF):
        net.load_state_dict(state)
        first = distill_loss(net(x), *teacher, y, temperature=2.0, weight=0.7).item()
    assert losses[0][0] == first
