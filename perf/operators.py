"""The operators around the BiGEMM block and in its training step, as cases to measure.

Three operators, each in a plain form (elementary torch operations in 32 bits)
and, with ``own``, as a program calls it in ``omniwave_b200``:

* ``norm``   RMSNorm before a block (``norm.rms_norm``) and after it, fused with
  the block's gate, the per-sample residual scale, the residual add and the next
  block's RMSNorm (``norm.norm_residual``); forward, or forward and backward;
* ``linear`` ``act(x W^T + b) + residual`` (``linear.linear``); forward, or
  forward and backward;
* ``adamw``  one AdamW step over many tensors at once (``optim.AdamW``), the
  moments held in 32 or in 8 bits, with global-norm clipping and the skip of a
  step whose gradients are not finite.
"""

import math
import random

import torch

own = False

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6          # of the norms
BLOCK = 256         # elements that share a scale in the 8-bit states; also the alignment of a tensor's state
TINY = 2.0 ** -100  # a block whose largest magnitude is below this is held as zeros
BETA1, BETA2, ADAM_EPS, LR, DECAY, MAX_NORM = 0.9, 0.999, 1e-8, 1e-3, 0.05, 1.0
STEPS_BEFORE = 10   # the optimizer is measured in the middle of a run
ROOT_HALF, INV_ROOT_2PI = math.sqrt(0.5), 1.0 / math.sqrt(2.0 * math.pi)


# ------------------------------------------------------------------ cases
def _norm(name, b, t, c, stream, delta, kind, gate, drop, train):
    return {"name": name, "op": "norm", "b": b, "t": t, "c": c, "stream": stream, "delta": delta, "kind": kind,
            "gate": gate, "drop": drop, "train": train}


def _linear(name, m, k, n, dtype, act, bias, residual, train):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "train": train}


def _adamw(name, tensors, elements, dtype, bits, clip):
    return {"name": name, "op": "adamw", "tensors": tensors, "elements": elements, "dtype": dtype, "bits": bits,
            "clip": clip}


def listed():
    return [
        # One image's single token on its way through a block at inference: latency.
        _norm("norm_one_token", 1, 1, 1024, "bf16", "bf16", "pair", "c", False, False),
        # The stage-1 map of the model's training batch: f32 residual stream, 16-bit branch, drop-path.
        _norm("norm_stage1_train", 128, 56 * 56, 128, "f32", "bf16", "pair", "c", True, True),
        # The stage-3 map in a 16-bit model with a gate of its own for every sample.
        _norm("norm_stage3_gated", 128, 14 * 14, 512, "bf16", "bf16", "pair", "bc", True, True),
        # The pre-norm alone on a ragged map: 7 x 7 tokens of 70 channels.
        _norm("norm_pre_ragged", 33, 7 * 7, 70, "f32", "f32", "pre", "none", False, True),
        # One token through a widening projection at inference: latency.
        _linear("linear_one_token", 1, 1024, 2048, "bf16", "silu", True, False, False),
        # Stage-4 tokens of the inference batch through a narrowing projection into the residual stream.
        _linear("linear_stage4_infer", 256 * 49, 2048, 1024, "f16", "none", True, True, False),
        # Stage-3 tokens of the training batch through a widening projection.
        _linear("linear_stage3_train", 128 * 196, 512, 1024, "bf16", "gelu", True, False, True),
        # A wide model's projection in training, the largest product.
        _linear("linear_wide_train", 32768, 4096, 4096, "bf16", "silu", True, True, True),
        # Fine-tuning a classifier's last few tensors: latency.
        _adamw("adamw_head", 3, 5000, "f32", 32, False),
        # The model's own parameters: 128 tensors, 10.2 M elements, clipped.
        _adamw("adamw_model", 128, 10_232_040, "f32", 32, True),
        # The same with the moments in 8 bits.
        _adamw("adamw_model_8bit", 128, 10_232_040, "f32", 8, True),
        # A model sixteen times as large, in 16 bits with 8-bit moments.
        _adamw("adamw_large_8bit", 400, 160_000_000, "bf16", 8, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 else max(lo, n // 8 * 8) if n >= 8 else n


def draw(rng):
    op = rng.choice(("norm", "linear", "adamw"))
    if op == "norm":
        c = _size(rng, 16, 4096)
        b = _log(rng, 1, 256)
        t = _log(rng, 1, max(1, min(3136, 50_000_000 // (b * c))))
        stream = rng.choice(("f32", "bf16", "f16"))
        delta = stream if rng.random() < 0.5 else {"f32": rng.choice(("bf16", "f16"))}.get(stream, stream)
        kind = rng.choice(("pre", "post", "pair", "pair"))
        gate = "none" if kind == "pre" else rng.choice(("c", "c", "bc", "none"))
        c_ = _norm("", b, t, c, stream, delta, kind, gate, kind != "pre" and rng.random() < 0.4, rng.random() < 0.6)
    elif op == "linear":
        m, k, n = _log(rng, 1, 32768), _size(rng, 16, 4096), _size(rng, 16, 4096)
        c_ = _linear("", m, k, n, rng.choice(("bf16", "f16")), rng.choice(("none", "relu", "silu", "gelu")),
                     rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.6)
    else:
        tensors = _log(rng, 1, 400)
        c_ = _adamw("", tensors, _log(rng, max(200, 4 * tensors), 120_000_000), rng.choice(("f32", "f32", "bf16")),
                    rng.choice((32, 8)), rng.random() < 0.5)
    del c_["name"]
    return c_


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(g, shape, dtype, scale=1.0, shift=0.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dtype)


def _sizes(case):
    """Sizes of ``tensors`` tensors with ``elements`` elements in all: a few large ones and many small ones."""
    n, total = case["tensors"], case["elements"]
    r = random.Random(n * 1_000_003 + total)
    w = [math.exp(r.gauss(0.0, 2.0)) for _ in range(n)]
    s = [max(1, int((total - n) * x / sum(w))) for x in w]
    s[-1] += max(0, total - sum(s))
    return s


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "norm":
        b, t, c = case["b"], case["t"], case["c"]
        st, dt, train = T[case["stream"]], T[case["delta"]], case["train"]
        s["x"] = _randn(g, (b, t, c), st).requires_grad_(train)
        s["pre"] = _randn(g, (c,), torch.float32, 0.1, 1.0).requires_grad_(train)
        if case["kind"] != "pre":
            s["delta"] = _randn(g, (b, t, c), dt, 0.7).requires_grad_(train)
            s["post"] = _randn(g, (c,), torch.float32, 0.1, 1.0).requires_grad_(train)
        if case["gate"] != "none":
            shape = (c,) if case["gate"] == "c" else (b, c)
            s["gate"] = _randn(g, shape, torch.float32, 0.1, 0.5).requires_grad_(train)
        if case["drop"]:  # drop-path: one sample in five leaves its branch out
            s["scale"] = (torch.rand(b, generator=g, device="cuda") < 0.8).float() / 0.8
        if train:
            s["dh"], s["dn"] = _randn(g, (b, t, c), st, 1e-2), _randn(g, (b, t, c), st, 1e-2)
    elif case["op"] == "linear":
        m, k, n, dt, train = case["m"], case["k"], case["n"], T[case["dtype"]], case["train"]
        s["x"] = _randn(g, (m, k), dt).requires_grad_(train)
        s["w"] = _randn(g, (n, k), dt, k ** -0.5).requires_grad_(train)
        if case["bias"]:
            s["b"] = _randn(g, (n,), dt, 0.1).requires_grad_(train)
        if case["residual"]:
            s["r"] = _randn(g, (m, n), dt).requires_grad_(train)
        if train:
            s["dy"] = _randn(g, (m, n), dt, 1e-2)
    else:
        sizes, dt = _sizes(case), T[case["dtype"]]
        at, total = [], 0
        for n in sizes:
            at.append(total)
            total += -(-n // BLOCK) * BLOCK
        used = torch.zeros(total, dtype=torch.bool, device="cuda")
        for o, n in zip(at, sizes):
            used[o:o + n] = True
        s["used"] = used
        s["param"] = _randn(g, (total,), torch.float32, 0.05).mul_(used).to(dt)
        s["grad"] = _randn(g, (total,), torch.float32, 1e-3).mul_(used).to(dt)
        m = _randn(g, (total,), torch.float32, 3e-4).mul_(used)
        v = _randn(g, (total,), torch.float32, 1e-3).square_().mul_(0.01).add_(1e-9).mul_(used)
        if case["bits"] == 8:
            zero = torch.full_like(m, 0.5)
            s["m"], s["m_scale"] = _hold(m, zero, False)
            s["v"], s["v_scale"] = _hold(v, zero, True)
        else:
            s["m"], s["v"] = m, v
        s["step"] = torch.full((), float(STEPS_BEFORE), device="cuda")
        if own:
            from omniwave_b200 import optim

            params = []
            for o, n in zip(at, sizes):
                p = torch.nn.Parameter(s["param"][o:o + n])
                p.grad = s["grad"][o:o + n]
                params.append(p)
            opt = optim.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY,
                              state_bits=case["bits"], max_norm=MAX_NORM if case["clip"] else None,
                              skip_nonfinite=case["clip"])
            held = opt.buffers[0]
            held["step"].fill_(STEPS_BEFORE)
            held["exp_avg"].copy_(s["m"])
            held["exp_avg_sq"].copy_(s["v"])
            if case["bits"] == 8:
                held["exp_avg_scale"].copy_(s["m_scale"])
                held["exp_avg_sq_scale"].copy_(s["v_scale"])
            s["opt"] = opt
    return s


# ------------------------------------------------------------------ the plain forms
def _rows(v, b):
    """A per-channel [C] or per-sample [B, C] vector as it spreads over [B, T, C]."""
    return v.float() if v.dim() == 1 else v.float()[:, None, :]


def _norm_plain(s):
    case = s["case"]
    x, c, st = s["x"].float(), case["c"], T[case["stream"]]
    if case["kind"] == "pre":
        h, q = x, None
    else:
        d = s["delta"].float()
        rd = torch.rsqrt(d.square().mean(-1, keepdim=True) + EPS)
        dn_ = d * rd
        q = _rows(s["gate"], case["b"]) if "gate" in s else None
        k = s["scale"][:, None, None] if "scale" in s else None
        p = dn_ * s["post"]
        branch = p if q is None else p * q
        h = x + (branch if k is None else branch * k)
    out = {} if case["kind"] == "pre" else {"h": h.to(st)}
    pre = case["kind"] != "post"
    if pre:
        rh = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        hn = h * rh
        out["n"] = (hn * s["pre"]).to(st)
    if not case["train"]:
        return out
    dh = s["dh"].float() if case["kind"] != "pre" else 0.0
    if pre:
        dn = s["dn"].float()
        out["d_pre"] = (dn * hn).sum((0, 1))
        u = dn * s["pre"]
        dh = dh + rh * (u - hn * (u * hn).mean(-1, keepdim=True))
    out["d_x"] = dh.to(st)
    if case["kind"] != "pre":
        e = dh if k is None else dh * k
        if q is not None:
            f = e * p
            out["d_gate"] = f.sum((0, 1)) if s["gate"].dim() == 1 else f.sum(1)
            e = e * q
        out["d_post"] = (e * dn_).sum((0, 1))
        u = e * s["post"]
        out["d_delta"] = (rd * (u - dn_ * (u * dn_).mean(-1, keepdim=True))).to(T[case["delta"]])
    return out


def _act(z, act):
    """The activation and its slope at z."""
    if act == "none":
        return z, None
    if act == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    if act == "silu":
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g))
    cdf = 0.5 * (1 + torch.erf(z * ROOT_HALF))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * INV_ROOT_2PI


def _linear_plain(s):
    case, dt = s["case"], T[s["case"]["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if case["bias"]:
        z = z + s["b"].float()
    y, slope = _act(z, case["act"])
    if case["residual"]:
        y = y + s["r"].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        dz = dy if slope is None else dy * slope
        out["d_x"], out["d_w"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if case["bias"]:
            out["d_b"] = dz.sum(0).to(dt)
        if case["residual"]:
            out["d_r"] = s["dy"]
    return out


def _random20(n, step):
    """Two 20-bit numbers for each of n elements at a step: what the 8-bit states are rounded with."""
    mask = 0xFFFFFFFF
    h = torch.arange(n, device="cuda")
    h = ((h & mask) * 0x9E3779B1 + (h >> 32) * 0x85EBCA6B + step * 0xC2B2AE35) & mask
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & mask
    h = ((h ^ (h >> 15)) * 0x846CA68B) & mask
    h = h ^ (h >> 16)
    return ((h & 0xFFFF) << 4) | 8, ((h >> 16) << 4) | 8


def _hold(v, r, positive):
    """v in 8 bits (e4m3, one f32 scale for BLOCK elements), rounded up where the dropped bits and r in [0, 1) carry."""
    v = v.view(-1, BLOCK)
    top = v.abs().amax(1)
    inv = torch.where(top > TINY, torch.full_like(top, 448.0) / top, torch.zeros_like(top))
    bits = (v.abs() * inv[:, None] * 2.0 ** -120).view(torch.int32)  # exponents of e4m3 in those of f32
    q = ((bits + (r.view(-1, BLOCK) * 2 ** 20).to(torch.int32)) >> 20).clamp(max=126)
    if positive:  # a second moment never falls to zero
        q = torch.where((v > 0) & (inv[:, None] > 0), q.clamp(min=1), q)
    q = q | ((v < 0).to(torch.int32) << 7)
    return q.to(torch.uint8).view(torch.float8_e4m3fn).view(-1), torch.where(top > TINY, top / 448.0, 0.0)


def _adamw_plain(s):
    case = s["case"]
    out = {"param": s["param"]}
    g, p = s["grad"].float(), s["param"].float()
    keep = None
    if case["clip"]:
        norm = g.double().square().sum().sqrt()
        keep = torch.isfinite(norm)
        out["norm"] = norm.float()
        g = g * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0).float()
    eight = case["bits"] == 8
    m, v = s["m"].float(), s["v"].float()
    if eight:
        m = (m.view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (v.view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
    step = s["step"] + 1
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    c1, c2 = 1 - BETA1 ** step.double(), 1 - BETA2 ** step.double()
    denom = v.sqrt() / c2.sqrt().float() + ADAM_EPS
    new = (p * (1 - LR * DECAY) - (LR / c1).float() * (m / denom)).to(s["param"].dtype)
    if eight:
        r1, r2 = _random20(m.numel(), step.to(torch.int64))
        new_m, new_ms = _hold(m, r1.float() / 2 ** 20, False)
        new_v, new_vs = _hold(v, r2.float() / 2 ** 20, True)
        moves = (("param", new), ("step", step), ("m_scale", new_ms), ("v_scale", new_vs))
        held = (("m", new_m), ("v", new_v))
    else:
        moves, held = (("param", new), ("step", step), ("m", m), ("v", v)), ()
    s.update((k, t if keep is None else torch.where(keep, t, s[k])) for k, t in moves)
    s.update((k, t if keep is None else torch.where(keep, t.view(torch.uint8), s[k].view(torch.uint8)).view(t.dtype))
             for k, t in held)
    out.update((k, s[k]) for k in ("param", "m", "v", "m_scale", "v_scale") if k in s)
    return out


# ------------------------------------------------------------------ the framework's calls
def _norm_own(s):
    from omniwave_b200 import norm

    case = s["case"]
    if case["kind"] == "pre":
        res = {"n": norm.rms_norm(s["x"], s["pre"], eps=EPS)}
    else:
        both = norm.norm_residual(s["x"], s["delta"], s["post"], s.get("gate"), sample_scale=s.get("scale"),
                                  next_weight=s["pre"] if case["kind"] == "pair" else None, eps=EPS)
        res = {"h": both[0], "n": both[1]} if case["kind"] == "pair" else {"h": both}
    if case["train"]:
        names = [k for k in ("x", "delta", "post", "gate", "pre") if k in s and (k != "pre" or "n" in res)]
        grads = torch.autograd.grad(list(res.values()), [s[k] for k in names], [s["d" + k] for k in res])
        res = {k: v.detach() for k, v in res.items()}
        res.update(("d_" + k, g) for k, g in zip(names, grads))
    return res


def _linear_own(s):
    from omniwave_b200 import linear

    case = s["case"]
    y = linear.linear(s["x"], s["w"], s.get("b"), activation=case["act"], residual=s.get("r"))
    if not case["train"]:
        return {"y": y}
    names = [k for k in ("x", "w", "b", "r") if k in s]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
    return {"y": y.detach(), **{"d_" + k: g for k, g in zip(names, grads)}}


def _adamw_own(s):
    opt = s["opt"]
    opt.step()
    held = opt.buffers[0]
    out = {"param": s["param"], "m": held["exp_avg"], "v": held["exp_avg_sq"]}
    if s["case"]["bits"] == 8:
        out["m_scale"], out["v_scale"] = held["exp_avg_scale"], held["exp_avg_sq_scale"]
    if s["case"]["clip"]:
        out["norm"] = opt.grad_norm
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return _norm_own(state) if op == "norm" else _linear_own(state) if op == "linear" else _adamw_own(state)
    with torch.no_grad():
        return _norm_plain(state) if op == "norm" else _linear_plain(state) if op == "linear" else _adamw_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    width = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "norm":
        n = case["b"] * case["t"] * case["c"]
        st, dt = width[case["stream"]], width[case["delta"]]
        per = {"pre": 2 * st, "post": 2 * st + dt, "pair": 3 * st + dt}[case["kind"]]
        if case["train"]:  # forward's inputs and both passes' outputs once, and the gradients that come in
            per += {"pre": 2 * st, "post": 2 * st + dt, "pair": 3 * st + dt}[case["kind"]]
        return {"bytes": n * per + 4 * case["c"], "flops": n * (40 if case["train"] else 12)}
    if case["op"] == "linear":
        m, k, n, train = case["m"], case["k"], case["n"], case["train"]
        moved = m * k + n * k + m * n * (2 if case["residual"] else 1)
        if train:  # dy comes in, dx and dw go out
            moved += m * n + m * k + n * k
        return {"bytes": 2 * moved, "flops": 2 * m * k * n * (3 if train else 1)}
    e, p = case["elements"], width[case["dtype"]]
    held = 16 if case["bits"] == 32 else 4 * (1 + 4 / BLOCK)
    return {"bytes": e * (3 * p + held), "flops": e * 15}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_norm(case, s):
    x = s["x"].detach().double()
    b, t, c = x.shape
    leaves = {"x": x}
    for k in ("delta", "post", "gate", "pre"):
        if k in s:
            leaves[k] = s[k].detach().double()
    if case["train"]:
        leaves = {k: v.requires_grad_() for k, v in leaves.items()}

    def rms(v, w):
        return v / (v.pow(2).sum(-1, keepdim=True) / c + EPS) ** 0.5 * w

    h = leaves["x"]
    out = {}
    if case["kind"] != "pre":
        add = rms(leaves["delta"], leaves["post"])
        if "gate" in s:
            gate = leaves["gate"]
            add = add * (gate.reshape(1, 1, c) if gate.dim() == 1 else gate.reshape(b, 1, c))
        if "scale" in s:
            add = add * s["scale"].double().reshape(b, 1, 1)
        h = h + add
        out["h"] = h
    if case["kind"] != "post":
        out["n"] = rms(h, leaves["pre"])
    else:
        leaves.pop("pre")
    if case["train"]:
        loss = sum((out[k] * s["d" + k].double()).sum() for k in out)
        grads = torch.autograd.grad(loss, list(leaves.values()))
        out.update(("d_" + k, g) for k, g in zip(leaves, grads))
    return {k: v.detach() for k, v in out.items()}


def _exact_linear(case, s):
    leaves = {k: s[k].detach().double() for k in ("x", "w", "b", "r") if k in s}
    if case["train"]:
        leaves = {k: v.requires_grad_() for k, v in leaves.items()}
    z = torch.einsum("mk,nk->mn", leaves["x"], leaves["w"])
    if "b" in leaves:
        z = z + leaves["b"]
    y = {"none": lambda v: v, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu}[case["act"]](z)
    if "r" in leaves:
        y = y + leaves["r"]
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, list(leaves.values()), s["dy"].double())
        out.update(("d_" + k, g) for k, g in zip(leaves, grads))
    return out


def _exact_adamw(case, s):
    p, g = s["param"].double(), s["grad"].double()
    out = {}
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        out["norm"] = norm
        g = g * min(1.0, MAX_NORM / (float(norm) + 1e-6))
    m, v = s["m"].double(), s["v"].double()
    if case["bits"] == 8:
        m = m * s["m_scale"].double().repeat_interleave(BLOCK)
        v = v * s["v_scale"].double().repeat_interleave(BLOCK)
    t = STEPS_BEFORE + 1
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    update = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    out["param"] = p - LR * DECAY * p - LR * update
    if case["bits"] == 32:
        out["m"], out["v"] = m, v
        return out
    r1, r2 = _random20(m.numel(), t)
    for k, val, r in (("m", m, r1), ("v", v, r2)):
        top = val.abs().view(-1, BLOCK).amax(1)
        a = torch.where(top > TINY, 448.0 / top, 0.0).repeat_interleave(BLOCK) * val.abs()
        quantum = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
        near = (torch.floor(a / quantum + r.double() / 2 ** 20) * quantum).clamp(max=448.0)
        if k == "v":
            near = torch.where(a > 0, near.clamp(min=2.0 ** -9), near)
        out[k], out[k + "_scale"] = near * torch.sign(val), torch.where(top > TINY, top / 448.0, 0.0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "adamw": _exact_adamw}[case["op"]](case, s)
