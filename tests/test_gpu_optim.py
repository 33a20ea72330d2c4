"""AdamW over many tensors on the GPU against float64 arithmetic.

Tolerances count roundings.  u = 2^-24 is half a step of f32.  m and v take
three roundings and one of a rounded constant each, relative to the magnitudes
they are summed from: 4 u.  Of the update alpha m / (sqrt(v) rc2 + eps), with
M = b1 |m| + (1 - b1) |g|: alpha = lr / (1 - b1^t) takes 6 u (lr, log b1 and its
product, expm1f's one step = 2 u, the division), rc2 half of 4 u and rsqrtf's two
steps = 4 u, sqrt(v) half of v's 4 u and its own step = 2 u, product and sum 2 u,
the division's two steps = 4 u, the last product 1 u, and m itself 4 u: 27 u of
alpha M / denom.  The decay and the last subtraction take 4 u of |p|.
Clipping multiplies g once more, by a coefficient rounded once: 2 u on g, 4 u
on v.  A 16-bit parameter is rounded once more, by half a step of its type.
"""

from __future__ import annotations

import copy
import math

import pytest
import torch

from omniwave_b200 import _lib, optim
from omniwave_b200.train import TrainStep

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.999, 1e-8, 0.05


def _params(dev, sizes, dtype=F32, seed=0, offset=0):
    """Parameters that are views of one buffer, each ``offset`` elements further than 16-byte alignment."""
    g = torch.Generator(device=dev).manual_seed(seed)
    ps = []
    for n in sizes:
        buf = torch.zeros(n + 64, dtype=dtype, device=dev)
        p = buf[offset:offset + n]
        p.copy_(torch.randn(n, generator=g, device=dev) * 0.1)
        q = torch.nn.Parameter(p)
        gb = torch.zeros(n + 64, dtype=dtype, device=dev)
        q.grad = gb[offset:offset + n]
        q.grad.copy_(torch.randn(n, generator=g, device=dev) * 1e-2)
        ps.append(q)
    return ps


def _step64(p, g, m, v, t, clip=1.0, lr=LR, wd=WD):
    """One step in float64; returns p, m, v and the bounds of their errors in f32."""
    g = g * clip
    ms, vs = B1 * m.abs() + (1 - B1) * g.abs(), B2 * v + (1 - B2) * g * g
    m, v = B1 * m + (1 - B1) * g, vs
    denom = (v / (1 - B2 ** t)).sqrt() + EPS
    alpha = lr / (1 - B1 ** t)
    pn = p * (1 - lr * wd) - alpha * m / denom
    return pn, m, v, 4 * U * p.abs() + 30 * U * alpha * ms / denom, 6 * U * ms, 8 * U * vs


@pytest.mark.parametrize("dtype", [F32, BF, HF], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes,offset", [
    ([1], 0), ([255, 256, 257, 1], 0), ([5000, 3], 1), ([1000, 70 * 129, 8], 3), ([100_003, 16], 0),
    ([(7 * i) % 600 + 1 for i in range(530)], 0),  # more tensors than one launch takes
], ids=["one", "edges", "off1", "off3", "long", "many"])
def test_matches_float64(cuda_device, sizes, offset, dtype):
    ps = _params(cuda_device, sizes, dtype, offset=offset)
    around = [p.data.new_empty(0).set_(p.untyped_storage()).clone() for p in ps]
    opt = optim.AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    m = [torch.zeros(n, dtype=torch.float64, device=cuda_device) for n in sizes]
    v = [x.clone() for x in m]
    n0 = _lib.load().ow_launch_count()
    for t in (1, 2, 3):
        old = [p.detach().double() for p in ps]
        gs = [p.grad.double() for p in ps]
        opt.step()
        for i, p in enumerate(ps):
            want, mw, vw, ep, em, ev = _step64(old[i], gs[i], m[i], v[i], t)
            s = opt.state[p]
            half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
            err = (p.detach().double() - want).abs()
            # a subnormal f16 is off by half its smallest step
            assert (err <= ep + half * want.abs() * (1 + 1e-3) + (2.0 ** -25 if dtype == HF else 0.0)).all(), (t, i, err.max())
            assert ((s["exp_avg"].double() - mw).abs() <= em).all(), (t, i)
            assert ((s["exp_avg_sq"].double() - vw).abs() <= ev).all(), (t, i)
            assert float(s["step"]) == t
            m[i], v[i] = s["exp_avg"].double(), s["exp_avg_sq"].double()
            p.grad.mul_(0.5 if t == 1 else -1.0)
    assert _lib.load().ow_launch_count() - n0 == 3 * math.ceil(len(sizes) / 512)
    for p, a, n in zip(ps, around, sizes):  # nothing beside the parameter was written
        whole = p.data.new_empty(0).set_(p.untyped_storage())
        assert torch.equal(whole[:offset], a[:offset]) and torch.equal(whole[offset + n:], a[offset + n:])


def _random20(slots, step):
    mask = 0xFFFFFFFF
    h = ((slots & mask) * 0x9E3779B1 + (slots >> 32) * 0x85EBCA6B + step * 0xC2B2AE35) & mask
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & mask
    h = ((h ^ (h >> 15)) * 0x846CA68B) & mask
    h = h ^ (h >> 16)
    return (((h & 0xFFFF) << 4) | 8).double() / 2 ** 20, (((h >> 16) << 4) | 8).double() / 2 ** 20


@pytest.mark.parametrize("sizes,dtype", [([1], F32), ([257, 3, 255], F32), ([4096 + 17], BF), ([300, 20_000], F32)])
def test_8bit_states_follow_their_definition(cuda_device, sizes, dtype):
    """Codes equal the float64 definition's, but where the value lies nearer to the next code than f32 may be off.

    A moment is a sum of magnitude M that may cancel, off by 4 u M (three roundings and a constant's); its block's
    largest, top, is off by 4 u max M, and the scale and its inverse take 2 u more.  So the value a = |m| 448 / top is
    off by 4 u M 448 / top and by (4 u max M / top + 4 u) a, taken here as 16 u (M 448 + a max M) / top."""
    ps = _params(cuda_device, sizes, dtype)
    opt = optim.AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8)
    held = opt.buffers[0]
    total = held["exp_avg"].numel()
    real = torch.zeros(total, dtype=torch.bool, device=cuda_device)
    gflat = torch.zeros(total, dtype=torch.float64, device=cuda_device)
    at = 0
    for p in ps:
        real[at:at + p.numel()] = True
        at += -(-p.numel() // 256) * 256
    assert at == total and held["exp_avg_scale"].numel() == total // 256

    def decode(k):
        return held[k].double() * held[k + "_scale"].double().repeat_interleave(256)

    for t in (1, 2, 3):
        gflat.zero_()
        gflat[real] = torch.cat([p.grad.double().reshape(-1) for p in ps])
        m = B1 * decode("exp_avg") + (1 - B1) * gflat
        mag = B1 * decode("exp_avg").abs() + (1 - B1) * gflat.abs()
        v = B2 * decode("exp_avg_sq") + (1 - B2) * gflat * gflat
        opt.step()
        r1, r2 = _random20(torch.arange(total, device=cuda_device), t)
        for k, val, r, mags in (("exp_avg", m, r1, mag), ("exp_avg_sq", v, r2, v)):
            top = val.abs().view(-1, 256).amax(1)
            big = mags.view(-1, 256).amax(1)
            scale = held[k + "_scale"].double()
            assert ((scale - top / 448).abs() <= 8 * U * big / 448).all()
            a = val.abs() * (448 / top.clamp(min=1e-38)).repeat_interleave(256)
            off = 16 * U * (mags * 448 + a * big.repeat_interleave(256)) / top.clamp(min=1e-38).repeat_interleave(256)
            quantum = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
            x = a / quantum + r
            want = (torch.floor(x) * quantum).clamp(max=448.0)
            if k == "exp_avg_sq":
                want = torch.where(a > 0, want.clamp(min=2.0 ** -9), want)
                assert (held[k][real].float() > 0).all()  # positive second moments stay positive
            sure = ((x - torch.round(x)).abs() > off / quantum) & ((a - 8 * quantum).abs() > off)
            assert sure.double().mean() > 0.9  # the comparison is not empty
            got = held[k].double()
            assert torch.equal(got[sure], (want * torch.sign(val))[sure]), (t, k)
            assert ((got.abs() - a).abs() <= quantum + off + 2.0 ** -9).all()
            assert (got[~real] == 0).all()
        for p in ps:
            p.grad.mul_(-0.7)


def test_8bit_second_moment_decays_in_the_mean(cuda_device):
    """1000 steps without gradient: v falls to 0.999^1000.  Rounding to nearest would leave it where it is.

    One step moves a code up or down with a chance p of at most 0.001 / (1/16), a variance of p (1/8)^2 relative to
    v^2, so 1000 steps spread v by at most 0.5; the mean over 65536 elements is off by less than 5 * 0.5 / 256 = 1%,
    and the block's largest element, held exactly, by nothing."""
    p = torch.nn.Parameter(torch.zeros(65536, device=cuda_device))
    p.grad = torch.zeros_like(p)
    opt = optim.AdamW([p], lr=0.0, betas=(B1, B2), weight_decay=0.0, state_bits=8)
    h = opt.buffers[0]
    codes = torch.randint(40, 120, (65536,), dtype=torch.uint8, device=cuda_device)
    codes[::256] = 126
    h["exp_avg_sq"].view(torch.uint8).copy_(codes)
    h["exp_avg_sq_scale"].fill_(1.0)
    v0 = h["exp_avg_sq"].double().view(-1, 256)[:, 1:]
    for _ in range(1000):
        opt.step()
    v = h["exp_avg_sq"].double().view(-1, 256) * h["exp_avg_sq_scale"].double()[:, None]
    ratio = float(v[:, 1:].sum() / v0.sum()) / 0.999 ** 1000
    assert abs(ratio - 1) < 0.03, ratio
    assert not torch.isnan(p).any()


def test_clip_norm_and_reproducibility(cuda_device):
    sizes = [70_001, 3, 512, 9999]
    runs = []
    for _ in range(2):
        ps = _params(cuda_device, sizes, seed=3)
        opt = optim.AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_norm=0.5)
        old = [p.detach().double() for p in ps]
        opt.step()
        runs.append([p.detach().clone() for p in ps] + [opt.grad_norm.clone()])
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    norm = torch.cat([p.grad.double() for p in ps]).norm()
    assert abs(float(opt.grad_norm) - float(norm)) <= 2 * U * float(norm)  # f64 sums, rounded once
    clip = min(1.0, 0.5 / (float(norm) + 1e-6))
    assert clip < 1.0
    for p, o in zip(ps, old):
        z = torch.zeros_like(o)
        want, _, _, ep, _, _ = _step64(o, p.grad.double(), z, z, 1, clip)
        assert ((p.detach().double() - want).abs() <= ep).all()


def test_clipping_asked_for_later_and_no_more(cuda_device):
    sizes = [300, 5000]
    late, first, never = (_params(cuda_device, sizes, seed=4) for _ in range(3))
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    a, b, c = optim.AdamW(late, **kw), optim.AdamW(first, max_norm=0.25, **kw), optim.AdamW(never, **kw)
    a.max_norm = 0.25
    a.step(), b.step(), c.step()
    assert torch.equal(a.grad_norm, b.grad_norm)
    for key in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(a.buffers[0][key], b.buffers[0][key]) and not torch.equal(a.buffers[0][key], c.buffers[0][key])
    a.load_state_dict(c.state_dict())
    with torch.no_grad():
        for p, q in zip(late, never):
            p.copy_(q)
    a.max_norm = None
    a.step(), c.step()
    assert all(torch.equal(p, q) for p, q in zip(late, never))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nonfinite_gradient_leaves_everything(cuda_device, bits, bad):
    ps = _params(cuda_device, [300, 5000, 1])
    opt = optim.AdamW(ps, lr=LR, state_bits=bits, max_norm=1.0, skip_nonfinite=True)
    found = torch.zeros((), device=cuda_device)
    opt.step(found_inf=found)
    assert float(found) == 0.0
    before = [p.detach().clone() for p in ps] + [t.view(torch.uint8).clone() for t in opt.buffers[0].values()]
    keep = float(ps[1].grad[4321])
    ps[1].grad[4321] = bad
    opt.step(found_inf=found)
    after = [p.detach() for p in ps] + [t.view(torch.uint8) for t in opt.buffers[0].values()]
    assert float(found) == 1.0 and not math.isfinite(float(opt.grad_norm))
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    ps[1].grad[4321] = keep
    opt.step(found_inf=found)  # the caller's flag alone calls the step off too
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    opt.step(found_inf=found.zero_())
    assert not torch.equal(before[1], ps[1].detach()) and float(opt.state[ps[1]]["step"]) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_nonfinite_gradient_that_is_not_called_off(cuda_device, bits):
    """It makes its own parameter NaN at once, and spoils no other block's."""
    ps = _params(cuda_device, [1024])
    opt = optim.AdamW(ps, lr=LR, state_bits=bits)
    ps[0].grad[300] = float("nan")
    opt.step()
    bad = torch.isnan(ps[0].detach())
    assert bad[300] and int(bad.sum()) == 1
    ps[0].grad[300] = 0.0
    opt.step()
    bad = torch.isnan(ps[0].detach())
    assert bad[300] and not bad[:256].any() and not bad[512:].any()
    assert bits == 8 or int(bad.sum()) == 1


def test_huge_finite_gradients_are_finite(cuda_device):
    """Squares that overflow f32 do not call a step off."""
    p = torch.nn.Parameter(torch.zeros(1000, device=cuda_device))
    p.grad = torch.full_like(p, 1e30)
    opt = optim.AdamW([p], lr=LR, weight_decay=0.0, max_norm=1.0, skip_nonfinite=True)
    found = torch.zeros((), device=cuda_device)
    opt.step(found_inf=found)
    assert float(found) == 0.0
    assert abs(float(opt.grad_norm) / (1e30 * 1000 ** 0.5) - 1) < 1e-6
    assert torch.allclose(p.detach(), torch.full_like(p, -LR), rtol=1e-4)  # the first step's size is lr


def test_norm_over_more_tensors_than_one_launch_takes(cuda_device):
    sizes = [(11 * i) % 700 + 1 for i in range(1100)]
    ps = _params(cuda_device, sizes, seed=6)
    for p in ps[::7]:
        p.grad = None
    opt = optim.AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, max_norm=0.3)
    old = [p.detach().double() for p in ps]
    opt.step()
    norm = torch.cat([p.grad.double() for p in ps if p.grad is not None]).norm()
    assert abs(float(opt.grad_norm) - float(norm)) <= 2 * U * float(norm)
    clip = min(1.0, 0.3 / (float(norm) + 1e-6))
    for i, (p, o) in enumerate(zip(ps, old)):
        if i % 7 == 0:
            assert torch.equal(p.detach().double(), o) and float(opt.state[p]["step"]) == 0
            continue
        z = torch.zeros_like(o)
        want, _, _, ep, _, _ = _step64(o, p.grad.double(), z, z, 1, clip)
        assert ((p.detach().double() - want).abs() <= ep).all()
        assert float(opt.state[p]["step"]) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_of_more_than_2_31_elements(cuda_device, bits):
    n = 2 ** 31 + 777
    p = torch.nn.Parameter(torch.zeros(n, device=cuda_device, dtype=BF))
    p.grad = torch.zeros_like(p)
    tail = torch.randn(5000, device=cuda_device).to(BF)
    p.grad[-5000:] = tail
    opt = optim.AdamW([p], lr=LR, weight_decay=0.0, state_bits=bits, max_norm=1e9)
    opt.step()
    q = torch.nn.Parameter(torch.zeros(5000, device=cuda_device, dtype=BF))
    q.grad = tail.clone()
    optim.AdamW([q], lr=LR, weight_decay=0.0, state_bits=bits, max_norm=1e9).step()
    assert torch.equal(p.detach()[-5000:], q.detach()) and not p.detach()[:-5000].any()
    assert abs(float(opt.grad_norm) - float(tail.double().norm())) <= 2 * U * float(tail.double().norm())


def test_without_gradient_no_step_and_groups(cuda_device):
    a, b, c = _params(cuda_device, [500, 300, 200])
    b.grad = None
    e = torch.nn.Parameter(torch.zeros(0, device=cuda_device))
    e.grad = torch.zeros_like(e)
    opt = optim.AdamW([{"params": [a, b, e]}, {"params": [c], "lr": 0.0, "weight_decay": 0.0, "state_bits": 8}],
                      lr=LR, weight_decay=WD, max_norm=1e9)
    old = [p.detach().clone() for p in (a, b, c)]
    opt.step()
    assert not torch.equal(a, old[0]) and torch.equal(b, old[1]) and torch.equal(c, old[2])
    assert float(opt.state[a]["step"]) == 1 and float(opt.state[b]["step"]) == 0 and float(opt.state[c]["step"]) == 1
    norm = torch.cat([a.grad, c.grad]).double().norm()  # over both groups
    assert abs(float(opt.grad_norm) - float(norm)) <= 2 * U * float(norm)
    for p in (a, c):
        p.grad = None
    opt.step()
    assert float(opt.state[a]["step"]) == 1


def test_layouts_and_moving_gradients(cuda_device):
    """Transposed parameters, gradients of other strides, gradients in new memory each step: as torch's AdamW."""
    torch.manual_seed(0)
    w = [torch.randn(33, 20, device=cuda_device).t(), torch.randn(4, 6, 5, 7, device=cuda_device).to(
        memory_format=torch.channels_last)]
    mine, ref = [torch.nn.Parameter(x.clone()) for x in w], [torch.nn.Parameter(x.clone()) for x in w]
    assert mine[0].stride() == (1, 20)
    opt = optim.AdamW(mine, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    tor = torch.optim.AdamW(ref, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    for t in range(3):
        for i, (p, q) in enumerate(zip(mine, ref)):
            g = torch.randn(p.shape, device=cuda_device) if t else torch.ones(1, device=cuda_device).expand(p.shape)
            q.grad = g.clone()
            p.grad = g  # contiguous, or expanded: not the parameter's strides
        opt.step()
        tor.step()
    for p, q in zip(mine, ref):
        # 3 steps of at most lr (1 + a few) each, both sides with at most 40 u of a step's size and 4 u of p
        assert ((p - q).abs() <= 3 * 2 * (40 * U * 4 * LR + 4 * U * q.abs())).all()
        assert opt.state[p]["exp_avg"].stride() == p.stride()


def test_captured_step_follows_the_lr_tensor(cuda_device):
    lr = torch.full((), LR, device=cuda_device)
    ps, qs = _params(cuda_device, [1000, 77]), _params(cuda_device, [1000, 77])
    opt = optim.AdamW(ps, lr=lr, max_norm=1.0, skip_nonfinite=True)
    ref = optim.AdamW(qs, lr=LR, max_norm=1.0, skip_nonfinite=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    ref.step()
    for k in range(3):
        lr.fill_(LR / (k + 1))
        ref.param_groups[0]["lr"] = float(lr)
        graph.replay()
        ref.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert float(opt.state[ps[0]]["step"]) == 4


def test_on_another_stream(cuda_device):
    ps, qs = _params(cuda_device, [200_000]), _params(cuda_device, [200_000])
    a, b = optim.AdamW(ps, lr=LR), optim.AdamW(qs, lr=LR)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    b.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ps[0], qs[0])


def test_checkpoints(cuda_device):
    """torch's AdamW checkpoint loads, this one's loads back and there, a deep copy goes on alike; 8 bits round trip."""
    ps, qs = _params(cuda_device, [1000, 33]), _params(cuda_device, [1000, 33])
    tor = torch.optim.AdamW(qs, lr=LR, weight_decay=WD)
    tor.step()
    opt = optim.AdamW(ps, lr=1.0)
    opt.load_state_dict(tor.state_dict())
    assert opt.param_groups[0]["lr"] == LR and opt.param_groups[0]["weight_decay"] == WD
    for p, q in zip(ps, qs):
        assert torch.equal(opt.state[p]["exp_avg"], tor.state[q]["exp_avg"]) and float(opt.state[p]["step"]) == 1
    torch.optim.AdamW(qs, lr=LR).load_state_dict(opt.state_dict())
    eight = optim.AdamW(ps, lr=LR, state_bits=8)
    with pytest.raises(ValueError, match="state_bits"):
        eight.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="size of optimizer's group"):
        optim.AdamW(ps[:1], lr=LR).load_state_dict(opt.state_dict())
    eight.step()
    saved = copy.deepcopy(eight.state_dict())
    twin_p, twin = copy.deepcopy((ps, eight))
    assert twin.param_groups[0]["params"][0] is twin_p[0]
    for p, t in zip(ps, twin_p):
        t.grad = p.grad.clone()
    eight.step()
    twin.step()
    assert all(torch.equal(p, t) for p, t in zip(ps, twin_p))
    ps2 = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    back = optim.AdamW(ps2, lr=LR, state_bits=8)
    back.load_state_dict(saved)
    assert float(back.state[ps2[0]]["step"]) == 1
    for k, v in back.buffers[0].items():
        assert v.dtype == eight.buffers[0][k].dtype


def test_refusals(cuda_device):
    z = torch.zeros(8, device=cuda_device)
    with pytest.raises(RuntimeError, match="dtype"):
        optim.AdamW([torch.nn.Parameter(z.double())])
    with pytest.raises(RuntimeError, match="densely"):
        optim.AdamW([z[::2].requires_grad_()])
    with pytest.raises(RuntimeError, match="CUDA is unavailable"):
        optim.AdamW([torch.nn.Parameter(z), torch.nn.Parameter(torch.zeros(3))])
    p = torch.nn.Parameter(z.clone())
    with pytest.raises(ValueError, match="more than once"):
        optim.AdamW([p, p])
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([p], state_bits=16)
    opt = optim.AdamW([p])
    p.grad = torch.zeros_like(p)
    with pytest.raises(ValueError, match="found_inf"):
        opt.step(found_inf=torch.zeros(2, device=cuda_device))
    opt.param_groups[0]["lr"] = torch.zeros((), dtype=torch.float64, device=cuda_device)
    with pytest.raises(ValueError, match="tensor lr"):
        opt.step()
    opt.param_groups[0]["lr"] = 1e-3
    p.data = p.data.to(BF)
    p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError, match="moved"):
        opt.step()


@pytest.mark.parametrize("graph", [False, True])
def test_train_step_fused_follows_torch(cuda_device, graph):
    """TrainStep with this optimizer against torch's on the same model, batches and clipping, and its fail-fast."""
    def make(kind):
        torch.manual_seed(0)
        m = torch.nn.Sequential(torch.nn.Linear(24, 40), torch.nn.SiLU(), torch.nn.Linear(40, 7)).to(cuda_device)
        return m, TrainStep(m, lr=LR, amp_dtype=None, clip_norm=0.2, ema_decay=0.9, cuda_graph=graph, optimizer=kind)

    (ma, a), (mb, b) = make("torch"), make("fused")
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for k in range(6):
        x = torch.randn(16, 24, device=cuda_device, generator=g)
        y = torch.randint(0, 7, (16,), device=cuda_device, generator=g)
        la, lb = a.step(x, y), b.step(x, y)
        # six steps of at most a few lr; a rounding of a gradient near zero may turn into a part of lr
        assert abs(float(la) - float(lb)) <= 1e-3 * abs(float(la))
    a.check_finite()
    b.check_finite()
    for p, q in zip(ma.parameters(), mb.parameters()):
        assert (p - q).abs().max() <= 0.05 * LR
    before = [p.detach().clone() for p in mb.parameters()]
    b.step(x.fill_(float("inf")), y)
    with pytest.raises(FloatingPointError):
        b.check_finite()
    assert all(torch.equal(p, q) for p, q in zip(before, mb.parameters()))


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_unclipped_gradients_whose_squares_overflow(cuda_device, dtype):
    """v = inf takes m / inf = 0 off its parameter, as the formula in f32 does, at once and for good; others go on."""
    (p,) = _params(cuda_device, [1000], dtype, seed=8)
    huge = torch.tensor([1e21, -1e21, 1e25, -1e30, 3e38], device=cuda_device)  # (1 - b2) g^2 is past f32
    large = torch.tensor([1e10, -1e18, 1e19, 3e20], device=cuda_device)        # and here it is not
    p.grad[:5], p.grad[500:504] = huge.to(dtype), large.to(dtype)
    opt = optim.AdamW([p], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, skip_nonfinite=True)
    found = torch.zeros((), device=cuda_device)
    m, v = torch.zeros(1000, dtype=torch.float64, device=cuda_device), torch.zeros(1000, dtype=torch.float64, device=cuda_device)
    half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    for t in (1, 2, 3):
        old, g = p.detach().double(), p.grad.double()
        opt.step(found_inf=found)
        want, _, _, ep, _, _ = _step64(old, g, m, v, t)
        want[:5], ep[:5] = old[:5] * (1 - LR * WD), 4 * U * old[:5].abs()
        err = (p.detach().double() - want).abs()
        assert (err <= ep + half * want.abs() * (1 + 1e-3)).all(), (t, err.max())
        m, v = opt.state[p]["exp_avg"].double(), opt.state[p]["exp_avg_sq"].double()
        assert torch.isinf(v[:5]).all() and torch.isfinite(v[5:]).all() and torch.isfinite(m).all()
        p.grad[:5] = 1e-2
        p.grad[500:504] *= 0.5
    assert float(found) == 0.0


def test_small_second_moments_without_eps(cuda_device):
    """Steps of gradients so small that v is below the smallest normal f32, taken from the v that is held."""
    n = 1000
    p = torch.nn.Parameter(torch.zeros(n, device=cuda_device))
    p.grad = torch.logspace(-20.6, -17, n, device=cuda_device)
    p.grad[::2] *= -1
    opt = optim.AdamW([p], lr=LR, betas=(B1, B2), eps=0.0, weight_decay=0.0)
    for t in (1, 2, 3):
        old = p.detach().double()
        opt.step()
        m, v = opt.state[p]["exp_avg"].double(), opt.state[p]["exp_avg_sq"].double()
        assert (v > 0).all() and float(v[0]) < 2.0 ** -140
        step = LR / (1 - B1 ** t) * m / (v / (1 - B2 ** t)).sqrt()
        # m and v are the held ones here, so less than the 30 u of a step from the gradient
        assert ((p.detach().double() - (old - step)).abs() <= 30 * U * step.abs() + 4 * U * old.abs()).all(), t


def _twins(dev, n, at, grad, **kw):
    """Two 8-bit optimizers over the same parameter, the first with ``grad`` at ``at`` and the second with 0 there."""
    (p,), (q,) = _params(dev, [n], seed=9), _params(dev, [n], seed=9)
    p.grad[at], q.grad[at] = grad, 0.0
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8) | kw
    return p, q, optim.AdamW([p], **kw), optim.AdamW([q], **kw)


def _others_equal(p, q, a, b, at):
    rest = torch.ones(p.numel(), dtype=torch.bool, device=p.device)
    rest[at] = False
    assert torch.equal(p.detach()[rest], q.detach()[rest])
    for k, t in a.buffers[0].items():
        t, w = t.view(torch.uint8), b.buffers[0][k].view(torch.uint8)
        if k in ("exp_avg", "exp_avg_sq"):
            t, w = t[:p.numel()][rest], w[:p.numel()][rest]
        assert torch.equal(t, w), k


def test_8bit_overflow_of_one_element_stays_with_it(cuda_device):
    """Its v is past f32, so it takes no step; it goes on from m = 0 and its block's largest v, the others as ever."""
    at = torch.tensor([300, 301, 1023], device=cuda_device)
    p, q, a, b = _twins(cuda_device, 1024, at, torch.tensor([1e30, -1e25, 3e38], device=cuda_device), skip_nonfinite=True)
    found = torch.zeros((), device=cuda_device)
    old = p.detach().double()
    a.step(found_inf=found), b.step()
    assert float(found) == 0.0
    assert ((p.detach().double() - old * (1 - LR * WD)).abs() <= 4 * U * old.abs())[at].all()
    _others_equal(p, q, a, b, at)
    h = a.buffers[0]
    assert not h["exp_avg"].float()[at].any()
    v = h["exp_avg_sq"].float()
    assert (v[at] == 448).all() and (v.view(-1, 256)[torch.tensor([1, 3])].amax(1) == 448).all()
    p.grad[at] = q.grad[at]  # 0: the block's largest v falls like any, so the scales stay alike
    a.step(), b.step()
    _others_equal(p, q, a, b, at)
    before = p.detach().clone()
    p.grad[at] = 1e-2
    a.step()
    moved = (p.detach() - before * (1 - LR * WD))[at]
    # m = 0.1 g, c1 = 0.271; v >= 0.001 g^2, c2 = 0.003: at most 0.37 / 0.577 lr
    assert (moved < 0).all() and (moved.abs() <= LR).all()


def test_8bit_overflow_of_a_whole_block(cuda_device):
    """No v of the block can be held: it is zeros, and its moments start over."""
    at = torch.arange(256, 512, device=cuda_device)
    p, q, a, b = _twins(cuda_device, 1024, at, torch.full((256,), 1e30, device=cuda_device), skip_nonfinite=True)
    old = p.detach().double()
    a.step(), b.step()
    assert ((p.detach().double() - old * (1 - LR * WD)).abs() <= 4 * U * old.abs())[at].all()
    _others_equal(p, q, a, b, at)
    for k in ("exp_avg", "exp_avg_sq"):
        assert float(a.buffers[0][k + "_scale"][1]) == 0.0 and not a.buffers[0][k].float()[at].any()
    p.grad[at] = 1e-2
    before = p.detach().clone()
    a.step()
    moved = (p.detach() - before * (1 - LR * WD))[at]
    # m = 0.1 g, c1 = 0.19; v = 0.001 g^2, c2 = 0.001999: 0.526 / 0.707 lr
    assert ((moved / -LR - 0.744).abs() < 0.01).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_8bit_gradient_that_is_not_finite_stays_with_its_element(cuda_device, bad):
    """When it does not call the step off: its parameter and moments are NaN from then on, and no other's."""
    at = torch.tensor([300, 777], device=cuda_device)
    p, q, a, b = _twins(cuda_device, 1024, at, bad)
    for _ in range(3):
        a.step(), b.step()
        assert torch.isnan(p.detach()[at]).all()
        _others_equal(p, q, a, b, at)
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.isnan(a.buffers[0][k].float()[at]).all()
        p.grad[at] = 0.0


def test_8bit_second_moments_too_small_to_hold(cuda_device):
    """Where a block's v are held as zeros its m are too, so no step is longer than one from moments of zero."""
    p = torch.nn.Parameter(torch.zeros(512, device=cuda_device))
    p.grad = torch.full_like(p, 1e-17)  # (1 - b2) g^2 = 1e-37, below 2^-100
    opt = optim.AdamW([p], lr=LR, betas=(B1, B2), eps=1e-30, weight_decay=0.0, state_bits=8)
    opt.buffers[0]["step"].fill_(20_000)  # both corrections are 1
    for k in range(8):
        before = p.detach().clone()
        opt.step()
        # 0.1 / sqrt(0.001), where moments held apart would reach 1 / sqrt(0.001)
        assert ((before - p.detach()).abs() <= LR * 0.1 / 0.001 ** 0.5 * (1 + 1e-5)).all(), k
        assert not any(t.view(torch.uint8).any() for name, t in opt.buffers[0].items() if name != "step")
    p.grad.zero_()
    before = p.detach().clone()
    opt.step()
    assert torch.equal(p.detach(), before)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_counts_as_a_write_to_its_parameters(cuda_device, bits):
    """A backward pass that needs the weights from before a step is refused, as after torch's AdamW."""
    from omniwave_b200 import linear, norm

    x = torch.randn(64, 64, device=cuda_device, dtype=BF).requires_grad_()
    w, idle = (torch.nn.Parameter(torch.randn(64, 64, device=cuda_device, dtype=BF) / 8) for _ in range(2))
    scale = torch.nn.Parameter(torch.ones(64, device=cuda_device))
    opt = optim.AdamW([w, idle, scale], lr=LR, state_bits=bits)
    for out in (linear.linear(x, w), norm.rms_norm(x, scale)):
        before = [t._version for t in (w, scale)]
        out.float().sum().backward(retain_graph=True)
        opt.step()
        moved = [t._version > v for t, v in zip((w, scale), before)]
        assert any(moved) and idle._version == 0
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.float().sum().backward()


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
def test_checkpoints_of_16_bit_parameters(cuda_device, dtype):
    """torch holds their moments in their own type: they load here exactly, and this one's load there."""
    ps, qs = _params(cuda_device, [1000, 33], dtype), _params(cuda_device, [1000, 33], dtype)
    tor = torch.optim.AdamW(qs, lr=LR, weight_decay=WD)
    tor.step()
    opt = optim.AdamW(ps, lr=LR)
    opt.load_state_dict(tor.state_dict())
    for p, q in zip(ps, qs):
        for k in ("exp_avg", "exp_avg_sq"):
            assert tor.state[q][k].dtype == dtype and opt.state[p][k].dtype == F32
            assert torch.equal(opt.state[p][k], tor.state[q][k].float())
        assert float(opt.state[p]["step"]) == 1
    opt.step()
    tor.load_state_dict(opt.state_dict())
    for p, q in zip(ps, qs):
        assert torch.equal(tor.state[q]["exp_avg"], opt.state[p]["exp_avg"].to(dtype)) and float(tor.state[q]["step"]) == 2
    eight = optim.AdamW(ps, lr=LR, state_bits=8)
    eight.step()
    wrong = eight.state_dict()  # its inner dicts are the optimizer's own
    wrong["state"] = {k: dict(v) for k, v in wrong["state"].items()}
    wrong["state"][0]["exp_avg"] = wrong["state"][0]["exp_avg"].float()  # values, where codes belong
    with pytest.raises(ValueError, match="exp_avg"):
        eight.load_state_dict(wrong)


def test_checkpoints_of_other_rules_are_refused(cuda_device):
    """What this optimizer does not do (maximize, amsgrad, coupled decay) is refused, before anything changes."""
    def made(kind, **kw):
        (q,) = _params(cuda_device, [500])
        o = kind([q], lr=LR, weight_decay=WD, **kw)
        o.step()
        return o.state_dict()

    (p,) = _params(cuda_device, [500])
    opt = optim.AdamW([p], lr=0.5)
    opt.step()
    before = {k: t.clone() for k, t in opt.buffers[0].items()}
    for sd, match in ((made(torch.optim.AdamW, maximize=True), "maximize"), (made(torch.optim.AdamW, amsgrad=True), "amsgrad"),
                      (made(torch.optim.Adam), "decoupled")):
        with pytest.raises(ValueError, match=match):
            opt.load_state_dict(sd)
        assert all(torch.equal(t, before[k]) for k, t in opt.buffers[0].items()) and opt.param_groups[0]["lr"] == 0.5
    (q,) = _params(cuda_device, [500])
    plain = torch.optim.Adam([q], lr=LR)  # without decay the rules are one
    plain.step()
    opt.load_state_dict(plain.state_dict())
    assert opt.param_groups[0]["lr"] == LR and opt.param_groups[0]["weight_decay"] == 0


def test_loading_keeps_a_schedule_and_runs_hooks(cuda_device):
    """A scheduler's own entries of a group come with a checkpoint; registered load hooks run, as torch runs them."""
    (p,), (q,) = _params(cuda_device, [300]), _params(cuda_device, [300])
    tor = torch.optim.AdamW([q], lr=LR)
    sched = torch.optim.lr_scheduler.OneCycleLR(tor, max_lr=0.3, total_steps=10)
    for _ in range(3):
        tor.step()
        sched.step()
    opt = optim.AdamW([p], lr=1.0)
    calls = []

    def pre(o, sd):
        calls.append(("pre", o, float(o.state[p]["step"])))
        sd["param_groups"][0]["eps"] = 0.25
        return sd

    handles = [opt.register_load_state_dict_pre_hook(pre),
               opt.register_load_state_dict_post_hook(lambda o: calls.append(("post", o, float(o.state[p]["step"]))))]
    sd = tor.state_dict()
    opt.load_state_dict(sd)
    assert calls == [("pre", opt, 0.0), ("post", opt, 3.0)]
    g, t = opt.param_groups[0], tor.param_groups[0]
    assert g["eps"] == 0.25 and g["state_bits"] == 32 and g["params"] == [p]
    for k in ("lr", "betas", "initial_lr", "max_lr", "min_lr"):
        assert g[k] == t[k], k
    for h in handles:
        h.remove()
    here = torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=0.3, total_steps=10)
    here.load_state_dict(sched.state_dict())
    opt.load_state_dict(tor.state_dict())
    for _ in range(4):
        for o, s in ((opt, here), (tor, sched)):
            o.step()
            s.step()
        assert g["lr"] == t["lr"] and g["betas"] == t["betas"]


def test_a_group_that_cannot_be_added_leaves_nothing(cuda_device, monkeypatch):
    """A failure half way (the memory of its second bucket, say) leaves no bucket that later steps would move."""
    (kept,) = _params(cuda_device, [300])
    opt = optim.AdamW([kept], lr=LR, max_norm=1.0)
    more = _params(cuda_device, [500]) + _params(cuda_device, [500], BF)
    before = [p.detach().clone() for p in more]
    made, real = [], optim._Bucket

    def failing(*args):
        if made:
            raise RuntimeError("no memory")
        made.append(real(*args))
        return made[0]

    monkeypatch.setattr(optim, "_Bucket", failing)
    with pytest.raises(RuntimeError, match="no memory"):
        opt.add_param_group({"params": more})
    monkeypatch.setattr(optim, "_Bucket", real)
    assert len(opt.param_groups) == 1 and len(opt.buffers) == 1 and list(opt.state) == [kept]
    opt.step()
    assert all(torch.equal(p, b) for p, b in zip(more, before))
    opt.add_param_group({"params": more})
    opt.step()
    assert len(opt.buffers) == 3 and not any(torch.equal(p, b) for p, b in zip(more, before))


def test_a_captured_step_outlives_a_group_added_later(cuda_device):
    """Its sums of squares stay its own: a replay writes to no memory that others have been given since."""
    ps = _params(cuda_device, [5000, 300])
    opt = optim.AdamW(ps, lr=LR, max_norm=0.5)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    at, size = opt._partials.data_ptr(), opt._partials.nbytes
    opt.add_param_group({"params": _params(cuda_device, [700_000])})
    assert opt._partials.data_ptr() != at and any(t is not None and t.data_ptr() == at for t in opt._replaced)
    others = [torch.full((size,), 7, dtype=torch.uint8, device=cuda_device) for _ in range(200)]
    want = _params(cuda_device, [5000, 300])
    ref = optim.AdamW(want, lr=LR, max_norm=0.5)
    ref.step(), ref.step()
    graph.replay()
    torch.cuda.synchronize()
    assert all((t == 7).all() for t in others)
    assert all(torch.equal(p, q) for p, q in zip(ps, want))
