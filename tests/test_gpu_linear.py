"""Linear with its epilogue on the GPU against float64.

Operands are 16-bit values; products of two are exact in f32.  The tensor
core and the CUDA cores add K of them, in any order, to within (K + 8) u of the
sum of their magnitudes (u = 2^-24; an f32 sum of n terms is off by at most
n - 1 roundings of its partial sums).  Bias and residual add one rounding each.
The activations are within 8 u (|z| + 1) of theirs (fast exponential and
division, a few steps each) and pass z's own error on with a slope of at most
1.13.  An output is rounded by half(t) of itself.
The backward holds z in 16 bits, off by half(t) |z| plus z's error; the slopes
change by at most 1.13 |dz| (silu'' <= 0.5, gelu'' <= 0.8; relu' jumps at 0, so
relu is tested on values whose sums are exact).  dz is rounded to 16 bits, half(t) of itself, when there is an
activation, and then summed.
"""

from __future__ import annotations

import pytest
import torch

from omniwave_b200 import _lib, linear
from omniwave_b200.optim import AdamW

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def _half(t):
    return U if t == F32 else torch.finfo(t).eps / 2


def _act(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    cdf = 0.5 * (1 + torch.erf(z / 2 ** 0.5))
    return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5


def _define(x, w, b, r, dy, act, t):
    """Outputs, gradients and the bounds of their errors, in float64."""
    x, w, dy = x.double(), w.double(), dy.double()
    m, k = x.shape
    n = w.shape[0]
    h = _half(t)
    z = x @ w.t()
    zm = x.abs() @ w.abs().t()
    if b is not None:
        z, zm = z + b.double(), zm + b.double().abs()
    ez = (k + 10) * U * zm if act != "relu" else torch.zeros_like(zm)  # relu's inputs add up exactly
    y, slope = _act(z, act)
    ey = 1.13 * ez + (8 * U * (z.abs() + 1) if act != "none" else 0.0)
    if r is not None:
        y = y + r.double()
        ey = ey + 2 * U * (y.abs() + r.double().abs())
    tiny = 2.0 ** -25 if t == HF else 0.0
    out, tol = {"y": y}, {"y": ey + h * 1.01 * (y.abs() + ey) + tiny}
    if act == "none":
        dz, edz = dy, torch.zeros_like(dy)
    else:
        eslope = 1.13 * (ez + h * 1.01 * z.abs() + tiny) + 8 * U * (z.abs() + 1)
        if act == "relu":
            assert ((z.abs() > ez + tiny) | (z == 0)).all()
            eslope = torch.zeros_like(z)
        dz = dy * slope
        edz = dy.abs() * eslope
    # as it is summed for the bias, and as the products take it
    edb = edz + (U * dz.abs())
    ez16 = edz + (h * 1.01 * (dz.abs() + edz) + tiny if act != "none" else 0.0)
    for name, a, ea, c, terms in (("dx", dz, ez16, w, n), ("dw", dz.t(), ez16.t(), x, m)):
        out[name] = a @ c
        e = ea @ c.abs() + (terms + 8) * U * ((a.abs() + ea) @ c.abs())
        tol[name] = (e, out[name])
    out["db"] = dz.sum(0)
    tol["db"] = (edb.sum(0) + (m + 8) * U * (dz.abs() + edb).sum(0), out["db"])
    return out, tol


def _ok(got, want, tol, where):
    if isinstance(tol, tuple):
        e, v = tol
        tol = e + _half(got.dtype) * 1.01 * (v.abs() + e) + (2.0 ** -25 if got.dtype == HF else 0.0)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"{where}: worst {(err / tol.clamp(min=1e-300)).max().item():.2f} of the bound"


def _inputs(dev, m, k, n, t, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device=dev)

    return (r(m, k).to(t), (r(n, k) * k ** -0.5).to(t), (r(n) * 0.3).to(t), r(m, n).to(t), r(m, n).to(t))


def _both(x, w, b, r, dy, act, where):
    want, tol = _define(x, w, b, r, dy, act, x.dtype)
    with torch.no_grad():
        plain = linear.linear(x, w, b, activation=act, residual=r)
    assert plain.dtype == x.dtype and plain.shape == want["y"].shape
    _ok(plain, want["y"], tol["y"], f"{where} y")
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b, r)]
    y = linear.linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    assert torch.equal(y, plain)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    for name, g, leaf in zip(["dx", "dw"] + ["db"] * (b is not None) + ["dr"] * (r is not None), grads,
                             [t for t in leaves if t is not None]):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        if name == "dr":
            assert torch.equal(g, dy)
        else:
            _ok(g, want[name], tol[name], f"{where} {name}")
    return grads


SHAPES = [(1, 8, 1), (1, 1024, 2048), (2, 64, 7), (3, 70, 33), (5, 2048, 16), (8, 300, 129), (9, 64, 64), (17, 8, 8),
          (100, 63, 45), (128, 64, 64), (129, 65, 257), (200, 1000, 24), (256, 512, 1024), (300, 129, 130),
          (1000, 48, 128), (333, 2048, 300), (2500, 72, 40)]


@pytest.mark.parametrize("m,k,n", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
@pytest.mark.parametrize("t", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("act,bias,res", [("none", False, False), ("gelu", True, True), ("silu", True, False),
                                          ("none", True, True), ("relu", False, True)])
def test_forward_and_gradients(cuda_device, m, k, n, t, act, bias, res):
    x, w, b, r, dy = _inputs(cuda_device, m, k, n, t)
    if act == "relu":  # eighths: products are 64ths, and sums of up to 2^18 are exact in f32, so z's sign is
        x, w = (x.float() * 8).round().clamp(-8, 8).div(8).to(t), (w.float() * 64).round().clamp(-8, 8).div(8).to(t)
    _both(x, w, b if bias else None, r if res else None, dy, act, f"{m}x{k}x{n}")


@pytest.mark.parametrize("m,k,n,act", [(25088, 512, 1024, "gelu"), (12544, 2048, 1024, "none"), (4096, 256, 2048, "silu"),
                                       (50_000, 64, 64, "none"), (777, 4096, 136, "silu")])
def test_larger(cuda_device, m, k, n, act):
    x, w, b, r, dy = _inputs(cuda_device, m, k, n, BF, seed=1)
    a = _both(x, w, b, r, dy, act, f"{m}x{k}x{n}")
    c = _both(x, w, b, r, dy, act, f"{m}x{k}x{n}")
    assert all(torch.equal(p, q) for p, q in zip(a, c))  # bit for bit


def test_strides_offsets_and_shapes(cuda_device):
    """Views with long rows, odd offsets and odd strides, batched shapes, broadcast inputs."""
    x, w, b, r, dy = _inputs(cuda_device, 60, 96, 40, BF, seed=2)
    want = linear.linear(x, w, b, activation="silu", residual=r)
    wide = torch.zeros(60, 200, dtype=BF, device=cuda_device)
    for off in (0, 8, 3):
        wide[:, off:off + 96] = x
        assert torch.equal(linear.linear(wide[:, off:off + 96], w, b, activation="silu", residual=r), want)
    flat = torch.zeros(60 * 96 + 1, dtype=BF, device=cuda_device)
    xo = flat[1:].view(60, 96).copy_(x)
    ww = torch.zeros(40, 97, dtype=BF, device=cuda_device)
    ww[:, :96] = w
    rr = torch.zeros(60, 41, dtype=BF, device=cuda_device)
    rr[:, 1:] = r
    assert torch.equal(linear.linear(xo, ww[:, :96], b, activation="silu", residual=rr[:, 1:]), want)
    assert torch.equal(linear.linear(x.view(3, 4, 5, 96), w, b, activation="silu", residual=r.view(3, 4, 5, 40)).view(60, 40),
                       want)
    xt = x.t().contiguous().t()
    assert torch.equal(linear.linear(xt, w, b, activation="silu", residual=r), want)
    assert linear.linear(x[0], w, b).shape == (40,)
    xe = x[:1].expand(60, 96)
    assert torch.equal(linear.linear(xe, w), linear.linear(xe.contiguous(), w))
    one = torch.randn(1, 96, device=cuda_device).to(BF).requires_grad_()
    y = linear.linear(one.expand(60, 96), w)
    (g,) = torch.autograd.grad(y, one, torch.ones_like(y))  # the broadcast row gets the sum
    exact = 60 * w.double().sum(0)
    # each of 60 rows rounded to 16 bits, their sum once more
    assert ((g.double() - exact).abs() <= 3 * _half(BF) * 60 * w.double().abs().sum(0)).all()


def test_autocast_with_f32_parameters(cuda_device):
    torch.manual_seed(0)
    lin = torch.nn.Linear(72, 48).to(cuda_device)
    x = torch.randn(500, 72, device=cuda_device, requires_grad=True)
    dy = torch.randn(500, 48, device=cuda_device).to(BF)
    with torch.autocast("cuda", dtype=BF):
        y = linear.linear(x, lin.weight, lin.bias, activation="gelu")
        assert y.dtype == BF
    grads = torch.autograd.grad(y, [x, lin.weight, lin.bias], dy)
    want, tol = _define(x.detach().to(BF), lin.weight.detach().to(BF), lin.bias.detach(), None, dy, "gelu", BF)
    _ok(y.detach(), want["y"], tol["y"], "y")
    for g, k in zip(grads, ("dx", "dw", "db")):
        assert g.dtype == F32
        e, v = tol[k]
        # dx is rounded to 16 bits before it is cast up; dw and db stay f32
        bound = e + (_half(BF) * 1.01 * (v.abs() + e) if k == "dx" else U * v.abs())
        assert ((g.double() - want[k]).abs() <= bound).all(), k


def test_gradients_against_differences(cuda_device):
    """gelu and silu: the loss along a random direction changes as the gradients say (differences in float64)."""
    for act in ("gelu", "silu"):
        x, w, b, r, dy = _inputs(cuda_device, 40, 24, 32, HF, seed=4)
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        grads = torch.autograd.grad(linear.linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3]),
                                    leaves, dy)
        g = torch.Generator(device=cuda_device).manual_seed(1)
        way = [torch.randn(t.shape, generator=g, device=cuda_device).double() for t in leaves]

        def loss(s):
            a, c, d, e = [t.double() + s * v for t, v in zip((x, w, b, r), way)]
            return ((_act(a @ c.t() + d, act)[0] + e) * dy.double()).sum()

        want = float((loss(1e-5) - loss(-1e-5)) / 2e-5)
        got = float(sum((p.double() * v).sum() for p, v in zip(grads, way)))
        size = float(sum((p.double() * v).abs().sum() for p, v in zip(grads, way)))
        assert abs(got - want) <= 4 * _half(HF) * size  # z, dz and each gradient rounded to f16


@pytest.mark.parametrize("k", [8, 56, 72, 1000, 2048, 4104, 8192])
@pytest.mark.parametrize("t", [BF, HF], ids=["bf16", "f16"])
def test_a_few_rows(cuda_device, k, t):
    # around the row counts where the kernel changes; features that do not fill a warp's 16; long k, that is split
    for m in (1, 7, 8, 9, 16, 17, 31, 32, 33):
        for n in (1, 15, 16, 17, 64, 1000):
            x, w, b, r, dy = _inputs(cuda_device, m, k, n, t, seed=m)
            want, tol = _define(x, w, b, r, dy, "silu", t)
            y = linear.linear(x, w, b, activation="silu", residual=r)
            _ok(y, want["y"], tol["y"], f"{m}x{k}x{n}")
            assert torch.equal(y, linear.linear(x, w, b, activation="silu", residual=r))
            # rows that lie apart, in 16-byte units and out of them: the same function, perhaps another kernel
            for pad in (8, 3):
                xs, ws, rs = (torch.full((a.shape[0], a.shape[1] + pad), float("nan"), dtype=t, device=cuda_device)
                              for a in (x, w, r))
                for a, c in ((xs, x), (ws, w), (rs, r)):
                    a[:, : c.shape[1]] = c
                y = linear.linear(xs[:, :k], ws[:, :k], b, activation="silu", residual=rs[:, :n])
                _ok(y, want["y"], tol["y"], f"{m}x{k}x{n} pad {pad}")


@pytest.mark.parametrize("m,k,n", [(16, 8192, 4096), (17, 4096, 4096), (32, 4096, 4097), (2, 4090, 4096)])
def test_a_few_rows_of_large_weights(cuda_device, m, k, n):
    _both(*_inputs(cuda_device, m, k, n, BF), "gelu", f"{m}x{k}x{n}")


def test_rows_and_features_do_not_mix(cuda_device):
    # what is not a number in one row of x or of the weight stays in its row or column of the result
    for m in (4, 16, 30, 40):
        for k in (64, 70, 4096):
            x, w, *_ = _inputs(cuda_device, m, k, 50, BF)
            want = linear.linear(x, w)
            x[m // 2, k // 3], w[7, k - 1], w[49, 0] = float("nan"), float("inf"), float("-inf")
            y = linear.linear(x, w)
            rows, cols = torch.arange(m, device=cuda_device) != m // 2, torch.ones(50, dtype=torch.bool, device=cuda_device)
            cols[7] = cols[49] = False
            assert torch.isnan(y[m // 2]).all() and not torch.isfinite(y[:, ~cols]).any()
            assert torch.equal(y[rows][:, cols], want[rows][:, cols])


def test_special_values(cuda_device):
    x = torch.zeros(4, 16, dtype=BF, device=cuda_device)
    x[1, 0], x[2, 0], x[3, 0] = float("inf"), float("nan"), -3e4
    w = torch.ones(8, 16, dtype=BF, device=cuda_device)
    for act in ("none", "relu", "silu", "gelu"):
        for rows in (x, x.repeat(40, 1)):  # both kernels
            y = linear.linear(rows, w, activation=act)
            assert (y[0] == 0).all() and (y[1] == float("inf")).all() and torch.isnan(y[2]).all()
            assert (y[3] == (-29952.0 if act == "none" else 0.0)).all()
    big = torch.full((10, 16), -300.0, dtype=HF, device=cuda_device, requires_grad=True)  # z = -1.4e6: beyond f16
    w = torch.full((8, 16), 300.0, dtype=HF, device=cuda_device)
    for act in ("relu", "silu", "gelu"):
        y = linear.linear(big, w, activation=act)
        (g,) = torch.autograd.grad(y, big, torch.ones_like(y))
        assert (y == 0).all() and (g == 0).all()


def test_empty_and_partial_gradients(cuda_device):
    x, w, b, r, dy = _inputs(cuda_device, 20, 24, 16, BF)
    wl, bl = w.detach().requires_grad_(), b.detach().requires_grad_()
    e = torch.zeros(0, 24, dtype=BF, device=cuda_device, requires_grad=True)
    y = linear.linear(e, wl, bl, activation="gelu")
    ge = torch.autograd.grad(y.sum(), [e, wl, bl])
    assert y.shape == (0, 16) and ge[0].shape == (0, 24) and (ge[1] == 0).all() and (ge[2] == 0).all()
    full = torch.autograd.grad(linear.linear(x.requires_grad_(), wl, bl, activation="silu"), [x, wl, bl], dy)
    x = x.detach()
    (only_w,) = torch.autograd.grad(linear.linear(x, wl, b, activation="silu"), [wl], dy)
    (only_b,) = torch.autograd.grad(linear.linear(x, w, bl, activation="silu"), [bl], dy)
    (only_x,) = torch.autograd.grad(linear.linear(x.requires_grad_(), w, b, activation="silu"), [x], dy)
    assert torch.equal(only_x, full[0]) and torch.equal(only_w, full[1]) and torch.equal(only_b, full[2])
    rl = r.detach().requires_grad_()
    (only_r,) = torch.autograd.grad(linear.linear(x.detach(), w, residual=rl), [rl], dy)
    assert torch.equal(only_r, dy)


def test_second_derivative_is_refused(cuda_device):
    x, w, *_ = _inputs(cuda_device, 20, 16, 8, BF)
    y = linear.linear(x.requires_grad_(), w, activation="silu")
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_refusals(cuda_device):
    x, w = torch.zeros(4, 16, device=cuda_device), torch.zeros(8, 16, device=cuda_device)
    with pytest.raises(RuntimeError, match="not 16-bit"):
        linear.linear(x, w)
    with pytest.raises(RuntimeError, match="without autocast"):
        linear.linear(x.to(BF), w)
    with pytest.raises(RuntimeError, match="without autocast"):
        linear.linear(x.to(BF), w.to(BF), residual=torch.zeros(4, 8, device=cuda_device))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        linear.linear(x.to(BF), w.to(BF), torch.zeros(8, dtype=torch.float64, device=cuda_device))
    with pytest.raises(RuntimeError, match="tensors on"):
        linear.linear(x.to(BF), w.to(BF).cpu())


def test_captured_and_on_another_stream(cuda_device):
    x, w, b, r, dy = _inputs(cuda_device, 300, 128, 96, BF, seed=6)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]

    def once():
        y = linear.linear(*leaves, activation="silu", residual=r)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

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
        leaves[0].mul_(-0.5)
    graph.replay()
    want = once()
    assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_first_cuda_call_of_a_thread(cuda_device):
    """A thread without a context of its own yet (as autograd's may be) can make the call."""
    import threading

    x, w, *_ = _inputs(cuda_device, 200, 64, 64, BF)
    linear.linear(x, w)  # its workspace is in the allocator's cache now: the thread's first CUDA call is the kernel's
    got: list = []

    def call():
        try:
            got.append(linear.linear(x, w))
        except Exception as exc:  # handed to the test
            got.append(exc)

    t = threading.Thread(target=call)
    t.start()
    t.join()
    assert torch.is_tensor(got[0]), got[0]
    assert torch.equal(got[0], linear.linear(x, w))


@pytest.mark.parametrize("m,k,n", [(200, 64, 64), (8192, 128, 1024)], ids=["one-sm", "sm-pairs"])
def test_wait_that_runs_out_is_reported(cuda_device, m, k, n):
    """The GEMM's bounded waits report to the library's fault word, as every pipelined kernel's do."""
    x, w, *_ = _inputs(cuda_device, m, k, n, BF)
    want = linear.linear(x, w)
    lib = _lib.load()
    assert lib.ow_debug_wait_probe(1_000_000) == 0
    try:
        linear.linear(x, w)
    finally:
        lib.ow_debug_wait_probe(0)
    assert _lib.device_fault(cuda_device.index or 0, reset=True) == 1
    assert torch.equal(linear.linear(x, w), want)


def test_two_threads_and_streams_at_once(cuda_device):
    """Calls of two threads on streams of their own, small and pair-sized products mixed, give what each gives alone."""
    import threading

    shapes = [(8192, 256, 512), (300, 512, 256), (5, 1024, 777), (2000, 72, 1000)]
    ins = [_inputs(cuda_device, *s, BF, seed=i) for i, s in enumerate(shapes)]
    want = [linear.linear(x, w, b, activation="gelu", residual=r) for x, w, b, r, _ in ins]
    torch.cuda.synchronize()
    got: dict = {}

    def work(name):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[name] = [[linear.linear(x, w, b, activation="gelu", residual=r) for x, w, b, r, _ in ins]
                         for _ in range(10)]
            torch.cuda.current_stream().synchronize()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    for rounds in got.values():
        for outs in rounds:
            assert all(torch.equal(a, e) for a, e in zip(outs, want))
    assert len(got) == 2


def test_outputs_of_more_than_2_31_elements(cuda_device):
    m, k, n = 2_100_000, 16, 1032
    g = torch.Generator(device=cuda_device).manual_seed(0)
    x = torch.randn(m, k, generator=g, device=cuda_device, dtype=BF)
    w = torch.randn(n, k, generator=g, device=cuda_device, dtype=BF)
    y = linear.linear(x, w, activation="silu")
    tail = slice(m - 300, m)
    assert torch.equal(y[tail], linear.linear(x[tail], w, activation="silu"))
    assert torch.equal(y[:300], linear.linear(x[:300], w, activation="silu"))
    wl = w.requires_grad_()
    y = linear.linear(x, wl, activation="silu")
    dy = torch.zeros_like(y)
    dy[tail] = 1.0  # only the last rows count
    (dw,) = torch.autograd.grad(y, wl, dy)
    (want,) = torch.autograd.grad(linear.linear(x[tail], wl, activation="silu"), wl, dy[tail])
    # the same products, grouped otherwise: f32 sums of 300 terms, then one rounding each
    mag = x[tail].float().abs().sum(0)[None, :] * 1.13
    assert ((dw.float() - want.float()).abs() <= 2 * 308 * U * mag + 2 * _half(BF) * want.float().abs()).all()


def test_run_of_the_operators_together(cuda_device):
    """Norms, two linears with their epilogues and the optimizer as a residual network uses them, against float64
    autograd; 16-bit roundings of a chain of six operators are at most 16 half steps relative to the largest value."""
    from omniwave_b200 import norm

    torch.manual_seed(0)
    c, hid = 128, 256
    names = ["w1", "b1", "w2", "b2", "pre", "post", "gate"]
    make = {"w1": torch.randn(hid, c) * c ** -0.5, "b1": torch.randn(hid) * 0.1, "w2": torch.randn(c, hid) * hid ** -0.5,
            "b2": torch.randn(c) * 0.1, "pre": 1 + 0.1 * torch.randn(c), "post": 1 + 0.1 * torch.randn(c),
            "gate": 0.5 + 0.1 * torch.randn(c)}
    ps = {k: torch.nn.Parameter(v.to(cuda_device).to(BF)) for k, v in make.items()}
    x = torch.randn(4, 50, c, device=cuda_device).to(BF)
    dy = torch.randn(4, 50, c, device=cuda_device).to(BF)

    def net(p, x):
        n = norm.rms_norm(x, p["pre"])
        d = linear.linear(linear.linear(n, p["w1"], p["b1"], activation="silu"), p["w2"], p["b2"], residual=n)
        return norm.norm_residual(x, d, p["post"], p["gate"])

    def net64(p, x):
        rms = lambda v: v * (v.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
        n = rms(x) * p["pre"]
        d = torch.nn.functional.silu(n @ p["w1"].t() + p["b1"]) @ p["w2"].t() + p["b2"] + n
        return x + p["gate"] * rms(d) * p["post"]

    p64 = {k: v.detach().double().requires_grad_() for k, v in ps.items()}
    y64 = net64(p64, x.double())
    g64 = torch.autograd.grad(y64, [p64[k] for k in names], dy.double())
    opt = AdamW(list(ps.values()), lr=1e-2, weight_decay=0.0, max_norm=1e6, skip_nonfinite=True)
    y = net(ps, x)
    y.backward(dy)
    tol = 16 * _half(BF)
    assert (y.double() - y64).abs().max() <= tol * y64.abs().max()
    for k, g in zip(names, g64):
        assert (ps[k].grad.double() - g).abs().max() <= tol * g.abs().max(), k
    before = {k: v.detach().clone() for k, v in ps.items()}
    opt.step()
    for k, g in zip(names, g64):
        step = ps[k].detach().double() - before[k].double()
        sure = g.abs() > tol * g.abs().max()  # a first step is lr against the gradient's sign
        assert ((step + 1e-2 * torch.sign(g)).abs()[sure] <= 1e-4 + _half(BF) * 1.01 * ps[k].double().abs()[sure]).all(), k


def _gelu_cases(dev, t):
    """Every finite z of the type with -20 < z < 20, as inputs that an identity weight passes on exactly."""
    v = torch.arange(65536, dtype=torch.int32, device=dev).to(torch.int16).view(t)
    v = v[torch.isfinite(v) & (v.abs() < 20)]
    return torch.cat([v, v.new_zeros(-v.numel() % 1920)])


def _gelu_bound(z, t):
    """gelu, its slope, and how far a result may be off.

    Forward: the tail Phi(-|z|) is 2^q(|z|), whose fit is off by 7e-6 of it (f16, up to |z| = 6), 3.1e-4 (bf16, up to 6)
    or 6.3e-4 (further out), under a third of bf16's half step.  Of q's 8 fused steps each is rounded by u of its partial
    sum; the sums' magnitudes add up to less than 8.5 (1 + z^2) after all later factors, and log 2 of that is the tail's:
    12 (1 + z^2) u, with 4 u of the exponential and 2 u of the products.
    Slope: the tail is t P(t) exp(-z^2 / 2), fitted to 3e-7 up to 6 and 3e-5 further out.  The exponent's three roundings
    make 3 u z^2 / 2, the exponential 4 u, t 3 u, the seven terms, whose magnitudes add up to twice their sum, 12 u, the
    products 3 u; the density takes no more.
    Below 2^-126 an exponential is 0: of gelu that drops |z| Phi(-|z|) where the tail is less than that (z < -12.8), of
    the slope z phi = z exp(-z^2 / 2) / sqrt(2 pi), less than 0.4 |z| 2^-126 (z < -13.2), and less than 2^-126 of Phi.
    Past 6, f16's gelu is under half its smallest step."""
    a = z.abs()
    phi, cdf, tail = (torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5,
                      *(0.5 * torch.special.erfc(v / 2 ** 0.5) for v in (-z, a)))
    fit = torch.full_like(z, 7e-6) if t == HF else torch.where(a <= 6, 3.1e-4, 6.3e-4)
    rel = fit + (18 + 12 * z * z) * U
    tiny, h = 2.0 ** -25 if t == HF else 2.0 ** -126, _half(t)
    y, s = z * cdf, cdf + z * phi
    drop = torch.where(tail < 1.001 * 2.0 ** -126, a * tail, 0.0)
    ty = (rel * a * tail + 2 * U * y.abs()) * (1 + h) + h * y.abs() + tiny + drop
    ts = (torch.where(a <= 6, 3e-7, 3e-5) + (24 + 2 * z * z) * U) * (cdf + a * phi) * (1 + h) + h * s.abs()
    return (y, ty), (s, ts + tiny * (1 + 0.4 * a))


@pytest.mark.parametrize("t", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("k,rows", [(16, None), (16, 8), (15, 4)], ids=["gemm", "units", "rows"])
def test_gelu_keeps_its_bits_in_the_tail(cuda_device, t, k, rows):
    """Forward (all three kernels) and slope, to little more than the rounding of the result, for every 16-bit z."""
    v = _gelu_cases(cuda_device, t)
    eye = torch.eye(k, device=cuda_device, dtype=t)
    for x in [v.view(-1, k)] if rows is None else v.view(-1, rows, k)[::7]:
        (y, ty), (s, ts) = _gelu_bound(x.double(), t)
        x = x.detach().requires_grad_(rows is None)
        got = linear.linear(x, eye, activation="gelu")
        err = (got.detach().double() - y).abs()
        assert (err <= ty).all(), (float((err / ty).max()), float(x.detach().reshape(-1)[(err / ty).argmax()]))
        if rows is None:
            (dx,) = torch.autograd.grad(got, x, torch.ones_like(got))  # dz, rounded to 16 bits
            err = (dx.double() - s).abs()
            assert (err <= ts).all(), (float((err / ts).max()), float(x.detach().reshape(-1)[(err / ts).argmax()]))


def test_gelu_keeps_its_bits_where_k_is_split(cuda_device):
    """The same through the kernel that adds split products: one row block, 8192 of k, of which one term is not 0."""
    t, k = HF, 8192
    v = _gelu_cases(cuda_device, t)[-64 * 64:].view(64, 64)
    x, w = torch.zeros(64, k, device=cuda_device, dtype=t), torch.zeros(64, k, device=cuda_device, dtype=t)
    x[:, 5000:5064] = v
    w[:, 5000:5064] = torch.eye(64, device=cuda_device, dtype=t)
    (y, ty), _ = _gelu_bound(v.double(), t)
    assert ((linear.linear(x, w, activation="gelu").double() - y).abs() <= ty).all()


def test_forward_mode_is_refused(cuda_device):
    import torch.autograd.forward_ad as fw

    from omniwave_b200 import norm

    x, w, g = torch.randn(4, 64, device=cuda_device, dtype=BF), torch.eye(64, device=cuda_device, dtype=BF), torch.ones(64, device=cuda_device)
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: linear.linear(d, w), lambda: linear.linear(x, w, residual=d), lambda: norm.rms_norm(d, g),
                     lambda: norm.norm_residual(x, d, g), lambda: linear.linear(d, torch.nn.Parameter(w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
