"""Norms with gate and residual on the GPU against float64.

Tolerances count roundings; u = 2^-24, half(t) = half a step of a type.  A row's
sum of C squares in f32 is off by at most (C / 8 + 12) u of itself when 8 or
more threads share it (each adds C / 8 at most, then they meet in a tree), so
its rsqrt by half of that and one step of the function: r is within
e_r = (C / 16 + 8) u.  A value that is a product of r and a few factors is off
by e_r + 6 u, and h or n by that of its terms' magnitudes and half(t) of itself.
The backward's means over C terms are off by (C / 8 + 12) u of the sum of their
terms' magnitudes; with two r in them, E = (C / 4 + 64) u bounds all of a row's
relative errors against the magnitudes.  A weight's gradient adds its rows in
chains of at most rows / 4 + 64 terms: it is off by (E + (rows / 4 + 64) u) of
the sum of its terms' magnitudes.
"""

from __future__ import annotations

import pytest
import torch

from omniwave_b200 import _lib, norm
from omniwave_b200.block import OmniWeaveBlock, forward_blocks

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-6


def _half(t):
    return U if t == F32 else torch.finfo(t).eps / 2


def _inputs(dev, shape, st, dt, gate, seed=0, wt=F32):
    g = torch.Generator(device=dev).manual_seed(seed)
    b, c = shape[0], shape[-1]

    def r(s, t, a=1.0, m=0.0):
        return (torch.randn(s, generator=g, device=dev) * a + m).to(t)

    d = {"x": r(shape, st), "delta": r(shape, dt, 0.7), "post": r((c,), wt, 0.2, 1.0), "pre": r((c,), wt, 0.2, 1.0)}
    if gate:
        d["gate"] = r((c,) if gate == "c" else (b, c), wt, 0.3, 0.2)
    d["scale"] = (torch.rand(b, generator=g, device=dev) < 0.7).float() / 0.7
    d["dh"], d["dn"] = r(shape, st), r(shape, st)
    return d


def _spread(v, shape):
    return v if v.dim() == 1 else v.reshape(shape[0], *([1] * (len(shape) - 2)), shape[-1])


def _define(d, use_scale, kind):
    """Outputs, gradients and the magnitudes their errors are relative to, in float64."""
    x, c = d["x"].double(), d["x"].shape[-1]
    shape = tuple(x.shape)
    out, mag = {}, {}
    s = d["scale"].double().reshape(-1, *([1] * (len(shape) - 1))) if use_scale else 1.0
    h = x
    hm = x.abs()
    if kind != "pre":
        de = d["delta"].double()
        rd = ((de * de).mean(-1, keepdim=True) + EPS).rsqrt()
        dd = de * rd
        q = _spread(d["gate"].double(), shape) if "gate" in d else torch.ones((), dtype=torch.float64, device=x.device)
        wp = d["post"].double()
        e = s * q * wp * dd
        h, hm = x + e, x.abs() + e.abs()
        out["h"], mag["h"] = h, hm
    D, Dm = (d["dh"].double(), d["dh"].double().abs()) if kind != "pre" else (0.0, 0.0)
    if kind != "post":
        rh = ((h * h).mean(-1, keepdim=True) + EPS).rsqrt()
        # r_h takes h's own error as well: relative to mean(hm |h|) r_h^2
        amp = 1 + (hm * h.abs()).mean(-1, keepdim=True) * rh * rh
        hh, hhm = h * rh, hm * rh * amp
        out["n"], mag["n"] = hh * d["pre"].double(), hhm * d["pre"].double().abs()
        dn = d["dn"].double()
        u = dn * d["pre"].double()
        D = D + rh * (u - hh * (u * hh).mean(-1, keepdim=True))
        Dm = Dm + rh * amp * (u.abs() + hhm * (u.abs() * hhm).mean(-1, keepdim=True))
        out["d_pre"] = (dn * hh).reshape(-1, c).sum(0)
        mag["d_pre"] = (dn.abs() * hhm).reshape(-1, c).sum(0)
    out["d_x"], mag["d_x"] = D, Dm
    if kind != "pre":
        k = s * q * wp
        b_ = k * D
        out["d_delta"] = rd * (b_ - dd * (b_ * dd).mean(-1, keepdim=True))
        bm = k.abs() * Dm if torch.is_tensor(k) else Dm
        mag["d_delta"] = rd * (bm + dd.abs() * (bm * dd.abs()).mean(-1, keepdim=True))
        out["d_post"] = (s * q * D * dd).reshape(-1, c).sum(0)
        mag["d_post"] = ((s * q).abs() * Dm * dd.abs()).reshape(-1, c).sum(0)
        if "gate" in d:
            f, fm = s * D * dd * wp, (s * Dm if torch.is_tensor(s) else Dm) * dd.abs() * wp.abs()
            red = (lambda t: t.reshape(-1, c).sum(0)) if d["gate"].dim() == 1 else (
                lambda t: t.reshape(shape[0], -1, c).sum(1))
            out["d_gate"], mag["d_gate"] = red(f), red(fm)
    return out, mag


def _call(d, use_scale, kind, out_dtype=None):
    if kind == "pre":
        return {"n": norm.rms_norm(d["x"], d["pre"], eps=EPS, out_dtype=out_dtype)}
    r = norm.norm_residual(d["x"], d["delta"], d["post"], d.get("gate"), sample_scale=d["scale"] if use_scale else None,
                           next_weight=d["pre"] if kind == "pair" else None, eps=EPS, out_dtype=out_dtype)
    return {"h": r[0], "n": r[1]} if kind == "pair" else {"h": r}


def _check(got, want, mag, c, rows, where=""):
    for k, v in got.items():
        e = (c / 4 + 64) * U
        if k in ("d_pre", "d_post", "d_gate"):
            e += (rows / 4 + 64) * U
        err = (v.double() - want[k]).abs()
        bound = e * mag[k] + _half(v.dtype) * want[k].abs() * (1 + 1e-3) + (2.0 ** -25 if v.dtype == HF else 0.0)
        assert (err <= bound).all(), f"{where} {k}: worst {(err / bound.clamp(min=1e-300)).max().item():.2f} of the bound"


SHAPES = [(1, 1, 1), (2, 3, 7), (1, 1, 1024), (3, 49, 70), (2, 5, 128), (4, 11, 40), (3, 130, 256), (2, 9, 512),
          (2, 33, 1000), (1, 7, 1024), (2, 3, 1032), (2, 5, 2048), (1, 3, 2049), (1, 5, 4096), (2, 2, 8192), (1, 2, 8200),
          (5, 1, 129), (300, 4, 4, 64), (7, 513)]


@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
@pytest.mark.parametrize("st,dt", [(F32, F32), (F32, BF), (BF, BF), (HF, HF)], ids=["f32", "f32bf16", "bf16", "f16"])
@pytest.mark.parametrize("kind,gate,use_scale", [("pre", None, False), ("post", "c", True), ("pair", "bc", True),
                                                 ("pair", None, False)], ids=["pre", "post", "gated", "pair"])
def test_forward_and_gradients(cuda_device, shape, st, dt, kind, gate, use_scale):
    d = _inputs(cuda_device, shape, st, dt, gate)
    want, mag = _define(d, use_scale, kind)
    c, rows = shape[-1], d["x"].numel() // shape[-1]
    with torch.no_grad():
        plain = _call(d, use_scale, kind)
    _check(plain, want, mag, c, rows, "forward")
    names = ["x"] + ([] if kind == "pre" else ["delta", "post"] + (["gate"] if gate else [])) + (
        [] if kind == "post" else ["pre"])
    leaves = {k: d[k].clone().requires_grad_() for k in names}
    out = _call({**d, **leaves}, use_scale, kind)
    assert all(torch.equal(out[k], plain[k]) for k in out)
    grads = torch.autograd.grad(list(out.values()), list(leaves.values()), [d["d" + k] for k in out])
    for k, g in zip(names, grads):
        assert g.dtype == leaves[k].dtype and g.shape == leaves[k].shape
    _check({"d_" + k: g for k, g in zip(names, grads)}, want, mag, c, rows, "backward")
    again = torch.autograd.grad(list(_call({**d, **leaves}, use_scale, kind).values()), list(leaves.values()),
                                [d["d" + k] for k in out])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_gradients_against_differences(cuda_device):
    """Along a random direction in all inputs the loss changes as the gradients say (differences in float64)."""
    d = _inputs(cuda_device, (3, 5, 72), F32, F32, "c", seed=5)
    names = ["x", "delta", "post", "gate", "pre"]
    leaves = {k: d[k].clone().requires_grad_() for k in names}
    out = _call({**d, **leaves}, True, "pair")
    grads = torch.autograd.grad(list(out.values()), list(leaves.values()), [d["dh"], d["dn"]])
    g = torch.Generator(device=cuda_device).manual_seed(9)
    way = {k: torch.randn(d[k].shape, generator=g, device=cuda_device).double() for k in names}

    def loss(t):
        o, _ = _define({**d, **{k: d[k].double() + t * way[k] for k in names}}, True, "pair")
        return (o["h"] * d["dh"].double()).sum() + (o["n"] * d["dn"].double()).sum()

    step = 1e-5
    want = float((loss(step) - loss(-step)) / (2 * step))
    got = float(sum((a.double() * way[k]).sum() for a, k in zip(grads, names)))
    size = float(sum((a.double() * way[k]).abs().sum() for a, k in zip(grads, names)))
    # f32 gradients: (72 / 4 + 64) u of magnitudes a few times the terms'; the difference itself is good to step^2
    assert abs(got - want) <= 1e-4 * size


@pytest.mark.parametrize("dn_only", [True, False])
def test_one_of_two_outputs_used(cuda_device, dn_only):
    d = _inputs(cuda_device, (2, 7, 96), F32, F32, "c")
    names = ["x", "delta", "post", "gate", "pre"]
    leaves = {k: d[k].clone().requires_grad_() for k in names}
    h, n = norm.norm_residual(leaves["x"], leaves["delta"], leaves["post"], leaves["gate"], next_weight=leaves["pre"], eps=EPS)
    zero = {**d, "dh": torch.zeros_like(d["dh"])} if dn_only else {**d, "dn": torch.zeros_like(d["dn"])}
    want, mag = _define(zero, False, "pair")
    used, dy = (n, d["dn"]) if dn_only else (h, d["dh"])
    grads = torch.autograd.grad(used, list(leaves.values()), dy, allow_unused=True)
    _check({"d_" + k: g for k, g in zip(names, grads)}, want, mag, 96, 14)


def test_special_rows(cuda_device):
    """Rows of zeros, of one huge element, and a NaN that stays in its row."""
    x = torch.zeros(1, 4, 64, device=cuda_device)
    x[0, 1, 3] = 1e18
    x[0, 2] = float("nan")
    x[0, 3] = 2.0
    w = torch.ones(64, device=cuda_device)
    n = norm.rms_norm(x, w)
    assert (n[0, 0] == 0).all()
    assert abs(float(n[0, 1, 3]) - 8.0) < 1e-5 and float(n[0, 1].abs().sum()) == float(n[0, 1, 3])
    assert torch.isnan(n[0, 2]).all()
    assert ((n[0, 3] - 1).abs() < 1e-6).all()
    h, n = norm.norm_residual(torch.ones_like(x), torch.zeros_like(x), w, next_weight=w)
    assert (h == 1).all() and ((n - 1).abs() < 1e-6).all()  # nothing to add: eps keeps the norm finite


def test_layouts_devices_and_autocast(cuda_device):
    d = _inputs(cuda_device, (4, 6, 80), F32, F32, "c", seed=2)
    want = norm.rms_norm(d["x"], d["pre"])
    xt = d["x"].transpose(0, 1).contiguous().transpose(0, 1)  # strided, same values
    assert torch.equal(norm.rms_norm(xt, d["pre"]), want)
    buf = torch.empty(4 * 6 * 80 + 1, device=cuda_device)
    xo = buf[1:].view(4, 6, 80).copy_(d["x"])  # off 16-byte alignment: other vectors, another order of the sums
    assert ((norm.rms_norm(xo, d["pre"]) - want).abs() <= (80 / 4 + 64) * U * want.abs()).all()
    with torch.autocast("cuda", dtype=BF):
        assert norm.rms_norm(d["x"], d["pre"]).dtype == BF
        h, n = norm.norm_residual(d["x"], d["delta"], d["post"], next_weight=d["pre"])
        assert h.dtype == F32 and n.dtype == BF
    assert norm.rms_norm(d["x"], d["pre"], out_dtype=HF).dtype == HF
    assert norm.rms_norm(d["x"][0, 0], d["pre"]).shape == (80,)
    for wt in (BF, HF):
        e = _inputs(cuda_device, (2, 3, 88), BF, BF, "bc", wt=wt)
        w64, mag = _define(e, True, "pair")
        names = ["x", "delta", "post", "gate", "pre"]
        leaves = {k: e[k].clone().requires_grad_() for k in names}
        out = _call({**e, **leaves}, True, "pair")
        _check({k: v.detach() for k, v in out.items()}, w64, mag, 88, 6)
        grads = torch.autograd.grad(list(out.values()), list(leaves.values()), [e["dh"], e["dn"]])
        _check({"d_" + k: g for k, g in zip(names, grads)}, w64, mag, 88, 6)
        assert grads[2].dtype == wt


@pytest.mark.parametrize("c", [64, 70, 300, 1025])
@pytest.mark.parametrize("st,dt", [(F32, BF), (BF, BF)], ids=["f32bf16", "bf16"])
def test_unaligned_arrays(cuda_device, c, st, dt):
    """Inputs and incoming gradients that start beside a 16-byte boundary, forward and gradients."""
    d = _inputs(cuda_device, (3, 11, c), st, dt, "bc", seed=8)
    for k in ("x", "delta", "dh", "dn"):
        buf = torch.empty(d[k].numel() + 1, dtype=d[k].dtype, device=cuda_device)
        d[k] = buf[1:].view(d[k].shape).copy_(d[k])
    want, mag = _define(d, True, "pair")
    names = ["x", "delta", "post", "gate", "pre"]
    leaves = {k: d[k].detach().requires_grad_() for k in names}
    out = _call({**d, **leaves}, True, "pair")
    _check({k: v.detach() for k, v in out.items()}, want, mag, c, 33)
    grads = torch.autograd.grad(list(out.values()), list(leaves.values()), [d["dh"], d["dn"]])
    _check({"d_" + k: g for k, g in zip(names, grads)}, want, mag, c, 33)


@pytest.mark.parametrize("c", [7, 70, 129, 2049])
@pytest.mark.parametrize("t", [F32, BF])
def test_rows_do_not_see_their_neighbours(cuda_device, c, t):
    """A row of NaN between others, whose 16-byte units it shares when C is ragged: they are as without it."""
    d = _inputs(cuda_device, (2, 9, c), t, t, "c", seed=4)
    names = ["x", "delta"]

    def run(d):
        leaves = {k: d[k].clone().requires_grad_() for k in names}
        out = _call({**d, **leaves}, True, "pair")
        grads = torch.autograd.grad(list(out.values()), list(leaves.values()), [d["dh"], d["dn"]])
        return [v.detach().reshape(18, c) for v in out.values()] + [g.reshape(18, c) for g in grads]

    want = run(d)
    bad = {**d, "x": d["x"].clone(), "delta": d["delta"].clone(), "dh": d["dh"].clone()}
    for r in (0, 5, 17):
        for k in ("x", "delta", "dh"):
            bad[k].view(18, c)[r] = float("nan")
    got = run(bad)
    fine = torch.ones(18, dtype=torch.bool, device=cuda_device)
    fine[[0, 5, 17]] = False
    for g, w in zip(got, want):
        assert torch.equal(g[fine], w[fine])
        assert torch.isnan(g[0]).all() and torch.isnan(g[17]).all()


def test_more_than_2_31_elements(cuda_device):
    rows, c = 33_600_000, 64
    x = torch.randn(1, rows, c, device=cuda_device, dtype=BF)
    d = x.roll(1, 1)
    w = torch.linspace(0.5, 1.5, c, device=cuda_device)
    h, n = norm.norm_residual(x, d, w, w, next_weight=w)
    for part in (slice(0, 40), slice(rows - 40, rows)):
        hp, np_ = norm.norm_residual(x[:, part].contiguous(), d[:, part].contiguous(), w, w, next_weight=w)
        assert torch.equal(h[:, part], hp) and torch.equal(n[:, part], np_)
    del h, n
    xl, dl = x.requires_grad_(), d.requires_grad_()
    h, n = norm.norm_residual(xl, dl, w, w, next_weight=w)
    gx, gd = torch.autograd.grad([h, n], [xl, dl], [d.detach(), x.detach()])
    part = slice(rows - 40, rows)
    xs, ds = (t.detach()[:, part].contiguous().requires_grad_() for t in (x, d))
    hs, ns = norm.norm_residual(xs, ds, w, w, next_weight=w)
    sx, sd = torch.autograd.grad([hs, ns], [xs, ds], [ds.detach(), xs.detach()])
    assert torch.equal(gx[:, part], sx) and torch.equal(gd[:, part], sd)


def test_empty(cuda_device):
    w = torch.ones(16, device=cuda_device, requires_grad=True)
    x = torch.zeros(0, 5, 16, device=cuda_device, requires_grad=True)
    h, n = norm.norm_residual(x, x * 1, w, w, next_weight=w)
    assert h.shape == n.shape == (0, 5, 16)
    (h.sum() + n.sum()).backward()
    assert (w.grad == 0).all() and x.grad.shape == (0, 5, 16)


def test_second_derivative_is_refused(cuda_device):
    x = torch.randn(2, 3, 8, device=cuda_device, requires_grad=True)
    y = norm.rms_norm(x, torch.ones(8, device=cuda_device))
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_refusals(cuda_device):
    x, w = torch.zeros(2, 3, 8, device=cuda_device), torch.ones(8, device=cuda_device)
    with pytest.raises(RuntimeError, match="dtype"):
        norm.rms_norm(x.double(), w)
    with pytest.raises(RuntimeError, match="dtype"):
        norm.norm_residual(x, x, w, w.to(torch.int32))
    with pytest.raises(RuntimeError, match="tensors on"):
        norm.rms_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="dtype"):
        norm.rms_norm(x, w, out_dtype=torch.float64)
    s = torch.ones(2, device=cuda_device)
    with pytest.raises(ValueError, match="no gradient"):
        norm.norm_residual(x, x, w, sample_scale=s.requires_grad_())
    with pytest.raises(ValueError, match="sample_scale"):
        norm.norm_residual(x, x, w, sample_scale=torch.ones(3, device=cuda_device))


def test_captured_training_step(cuda_device):
    """Forward and backward captured, replayed on new inputs.

    No eager autograd graph of the same leaves is alive during the capture: PyTorch's engine would make the stream of
    that graph's leaf nodes wait for the captured one, which it refuses for any operator.
    """
    d = _inputs(cuda_device, (2, 10, 64), F32, F32, "c", seed=3)
    names = ["x", "delta", "post", "gate", "pre"]
    leaves = {k: d[k].clone().requires_grad_() for k in names}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def once():
        out = _call({**d, **leaves}, True, "pair")
        return torch.autograd.grad(list(out.values()), list(leaves.values()), [d["dh"], d["dn"]])

    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = once()
    with torch.no_grad():
        leaves["x"].mul_(-0.5)
    graph.replay()
    want = once()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def _block(dev, post, seed=0, c=128, drop=0.0):
    torch.manual_seed(seed)
    b = OmniWeaveBlock(14, 14, c, 64, "local", 0, layer_scale_init=0.3, post_norm=post, drop_path_rate=drop).to(dev)
    with torch.no_grad():
        b.norm_weight.add_(torch.randn_like(b.norm_weight) * 0.1)
        if post:
            b.post_norm_weight.add_(torch.randn_like(b.post_norm_weight) * 0.1)
    return b


def test_post_norm_blocks(cuda_device):
    """A row of post-norm and plain blocks against the formula on the framework's own operator, forward and gradients."""
    from omniwave_b200.ops import bigemm_delta_cuda

    blocks = [_block(cuda_device, True, 0), _block(cuda_device, True, 1), _block(cuda_device, False, 2),
              _block(cuda_device, True, 3)]
    g = torch.Generator(device=cuda_device).manual_seed(0)
    x = torch.randn(2, 14, 14, 128, device=cuda_device, generator=g)
    dy = torch.randn(2, 14, 14, 128, device=cuda_device, generator=g)

    def formula(x):
        for b in blocks:
            if not b.post_norm:
                x = b(x)
                continue
            rms = lambda v, w: v * (v.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w  # noqa: E731
            d = bigemm_delta_cuda(x=rms(x, b.norm_weight), plan=b.plan, a_u=b.a_u, a_v=b.a_v, a_o=b.a_o, b_u=b.b_u,
                                  b_v=b.b_v, b_o=b.b_o, gamma=torch.ones_like(b.gamma))
            x = x + b.gamma * rms(d, b.post_norm_weight)
        return x

    ps = [p for b in blocks for p in b.parameters()]
    a = forward_blocks(blocks, x)
    want = formula(x)
    assert (a - want).abs().max() <= 1e-4 * want.abs().max()  # the operator's own f32 gate
    ga = torch.autograd.grad(a, ps, dy)
    gw = torch.autograd.grad(want, ps, dy)
    for p, q in zip(ga, gw):
        assert (p - q).abs().max() <= 1e-3 * q.abs().max()
    assert torch.equal(blocks[0](x), forward_blocks(blocks[:1], x))
    with torch.autocast("cuda", dtype=BF):  # a mixed-precision step runs and stays near
        m = forward_blocks(blocks, x)
        assert m.dtype == F32
        assert (m - want).abs().max() <= 5e-2 * want.abs().max()
        torch.autograd.grad(m, ps, dy)
    # drop-path: all samples kept or left out with a probability; a seeded run repeats
    d = _block(cuda_device, True, 4, drop=0.5).train()
    torch.manual_seed(1)
    y1 = d(x)
    torch.manual_seed(1)
    assert torch.equal(y1, d(x))


@pytest.mark.parametrize("c", [64, 70, 777])
def test_a_gate_for_each_of_many_samples_of_one_token(cuda_device, c):
    shape, st = (100_000, 1, c), BF
    d = _inputs(cuda_device, shape, st, st, "bc")
    want, mag = _define(d, True, "pair")
    names = ["x", "delta", "post", "gate", "pre"]
    leaves = {k: d[k].requires_grad_() for k in names}
    out = _call(d | leaves, True, "pair")
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(list(out.values()), [leaves[k] for k in names], [d["dh"], d["dn"]])
    # dx, ddelta, the gate's f32 gradient and the partial sums: two rows of f32 a sample
    assert torch.cuda.max_memory_allocated() - held <= 1.05 * 100_000 * c * (2 * 2 + 4 + 2 * 4) + (1 << 22)
    got = {k: v.detach() for k, v in out.items()} | {"d_" + k: g for k, g in zip(names, grads)}
    _check(got, want, mag, c, 100_000, f"c={c}")


@pytest.mark.parametrize("c", [40, 64, 70, 129, 512, 777, 1000, 1032, 2049, 4096, 8200])
@pytest.mark.parametrize("samples,tokens", [(300, 1), (300, 7), (3, 500), (700, 40)])
@pytest.mark.parametrize("t,off", [(BF, 0), (BF, 1), (F32, 0)], ids=["bf16", "bf16-off", "f32"])
def test_backward_stays_in_its_workspace(cuda_device, c, samples, tokens, t, off):
    """The C entry, given the bytes that it asked for in front of a guard; gradients off 16 bytes as well."""
    if samples * tokens * c > 30_000_000:
        tokens = max(1, 30_000_000 // (samples * c))
    shape = (samples, tokens, c)
    d = _inputs(cuda_device, shape, t, t, "bc")
    rows, n = samples * tokens, samples * tokens * c
    code = _lib.DTYPE_CODE[t]
    stats = torch.ones(2, rows, device=cuda_device)
    outs = {k: torch.zeros(n + 1, dtype=t, device=cuda_device)[off:off + n] for k in ("dx", "dd")}
    dp, dg, dq = torch.empty(c, device=cuda_device), torch.empty(samples, c, device=cuda_device), torch.empty(c, device=cuda_device)
    a = _lib.Norm(samples, tokens, c, d["x"].data_ptr(), code, d["delta"].data_ptr(), code, d["post"].data_ptr(), 0,
                  d["gate"].data_ptr(), 0, samples, None, d["pre"].data_ptr(), 0, EPS, None, None, code,
                  stats[0].data_ptr(), stats[1].data_ptr(), None, 0)
    g = _lib.NormGrads(d["dh"].data_ptr(), d["dn"].data_ptr(), outs["dx"].data_ptr(), outs["dd"].data_ptr(), dp.data_ptr(),
                       dg.data_ptr(), dq.data_ptr())
    lib = _lib.load()
    need = lib.ow_norm_bwd_workspace_size(a)
    ws = torch.full((need + (1 << 20),), 0x5A, dtype=torch.uint8, device=cuda_device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _lib.check(lib.ow_norm_bwd(a, g, torch.cuda.current_stream().cuda_stream), "ow_norm_bwd")
    assert (ws[need:] == 0x5A).all()
    # the sums against the definition, with the 1 / rms that was given (1): dnext = sum dn h, h = x + q wp delta
    h = d["x"].double() + d["gate"].double()[:, None] * d["post"].double() * d["delta"].double()
    want, mag = (d["dn"].double() * h).sum((0, 1)), (d["dn"].double().abs() * h.abs()).sum((0, 1))
    assert ((dq.double() - want).abs() <= (64 + rows / 4 + 64) * U * mag + U * want.abs()).all()


def test_forward_blocks_with_hooks(cuda_device):
    """Hooked blocks see their own inputs and outputs, and the chain's result is that of the blocks called in turn."""
    blocks = [_block(cuda_device, True, s) for s in range(3)]
    x = torch.randn(2, 14, 14, 128, device=cuda_device, dtype=BF)
    with torch.autocast("cuda", dtype=BF):
        want = x
        for b in blocks:
            want = b(want)
        seen = []
        handles = [b.register_forward_hook(lambda m, a, o: seen.append((a[0], o))) for b in blocks]
        got = forward_blocks(blocks, x)
        assert torch.equal(got, want) and len(seen) == 3
        assert seen[0][0] is x and seen[2][1] is got and all(torch.equal(seen[i][1], seen[i + 1][0]) for i in (0, 1))
        handles.pop(1).remove()
        handles.pop(0).remove()
        seen.clear()
        last = forward_blocks(blocks, x)  # the first two are fused, the third is called
        assert len(seen) == 1 and torch.equal(blocks[2](forward_blocks(blocks[:2], x)), last)
        handles.pop().remove()
        blocks[1].register_forward_hook(lambda m, a, o: o * 0)
        assert torch.equal(forward_blocks(blocks, x), blocks[2](torch.zeros_like(x)))
