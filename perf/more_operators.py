"""A feed-forward sub-block and the loss that trains it, as cases to measure.

Three operators, each in a plain form (elementary torch operations in 32 bits)
and, with ``own``, as a program calls it in ``omniwave_b200``:

* ``ln``      layer norm (``norm.layer_norm``); forward, or forward and backward
  with the gradients of weight and bias;
* ``ffn``     the gated feed-forward block ``(act(x Wg^T + bg) (x Wu^T + bu)) Wd^T + bd + residual``
  (``feed_forward.gated_feed_forward``); forward, or forward and backward;
* ``distill`` the loss of a classifier that learns from a teacher's top logits and
  from labels (``loss.distill_loss``); its value, or its value and the logits' gradient.
"""

import math
import random

import torch

own = False

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5  # of the norm
ROOT_HALF, INV_ROOT_2PI = math.sqrt(0.5), 1.0 / math.sqrt(2.0 * math.pi)


# ------------------------------------------------------------------ cases
def _ln(name, b, t, c, dtype, out, bias, train):
    return {"name": name, "op": "ln", "b": b, "t": t, "c": c, "dtype": dtype, "out": out, "bias": bias, "train": train}


def _ffn(name, m, k, f, n, dtype, act, bias, residual, train):
    return {"name": name, "op": "ffn", "m": m, "k": k, "f": f, "n": n, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "train": train}


def _distill(name, rows, classes, top, dtype, temperature, labels, ragged, train):
    return {"name": name, "op": "distill", "rows": rows, "classes": classes, "top": top, "dtype": dtype,
            "temperature": temperature, "labels": labels, "ragged": ragged, "train": train}


def listed():
    return [
        # One image's single token on its way through a block at inference: latency.
        _ln("ln_one_token", 1, 1, 1024, "bf16", "bf16", True, False),
        # The stage-1 map of the model's training batch: an f32 residual stream, 16-bit compute.
        _ln("ln_stage1_train", 128, 56 * 56, 128, "f32", "bf16", True, True),
        # A 14 x 14 map of 1024 channels in a 16-bit model, trained.
        _ln("ln_wide_train", 256, 14 * 14, 1024, "bf16", "bf16", True, True),
        # A ragged map without a bias: 7 x 7 tokens of 777 channels.
        _ln("ln_ragged_train", 33, 7 * 7, 777, "f16", "f16", False, True),
        # One token through the block at inference: latency.
        _ffn("ffn_one_token", 1, 1024, 2048, 1024, "bf16", "silu", False, True, False),
        # Stage-4 tokens of the inference batch, with biases, into the residual stream.
        _ffn("ffn_stage4_infer", 256 * 49, 1024, 2048, 1024, "f16", "silu", True, True, False),
        # Stage-3 tokens of the training batch.
        _ffn("ffn_stage3_train", 128 * 196, 512, 1024, 512, "bf16", "gelu", True, True, True),
        # A wide model's block in training, the largest product.
        _ffn("ffn_wide_train", 16384, 4096, 8192, 4096, "bf16", "silu", False, True, True),
        # Fine-tuning a classifier with a few images: latency.
        _distill("distill_few", 8, 1000, 10, "f32", 1.0, True, False, True),
        # The model's training batch, a softened teacher.
        _distill("distill_batch", 128, 1000, 32, "bf16", 2.0, True, True, True),
        # Token-sized batches over a large set of classes, the largest loss; some rows have no teacher, some no label.
        _distill("distill_wide", 4096, 32000, 64, "bf16", 2.0, True, True, True),
        # Validation over an odd set of classes, from the teacher alone.
        _distill("distill_odd_valid", 1531, 40009, 100, "f16", 1.0, False, True, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 else max(lo, n // 8 * 8) if n >= 8 else n


def draw(rng):
    op = rng.choice(("ln", "ffn", "distill"))
    if op == "ln":
        c = _size(rng, 16, 8192)
        b = _log(rng, 1, 256)
        t = _log(rng, 1, max(1, min(3136, 50_000_000 // (b * c))))
        dtype = rng.choice(("f32", "bf16", "f16"))
        out = rng.choice(("f32", "bf16", "f16")) if dtype == "f32" else dtype
        c_ = _ln("", b, t, c, dtype, out, rng.random() < 0.7, rng.random() < 0.6)
    elif op == "ffn":
        m, k, f = _log(rng, 1, 16384), _size(rng, 16, 4096), _size(rng, 16, 8192)
        n = k if rng.random() < 0.7 else _size(rng, 16, 4096)
        c_ = _ffn("", m, k, f, n, rng.choice(("bf16", "f16")), rng.choice(("silu", "silu", "gelu", "relu", "none")),
                  rng.random() < 0.4, n == k and rng.random() < 0.6, rng.random() < 0.6)
    else:
        classes = _log(rng, 10, 131072)
        rows = _log(rng, 1, max(1, min(16384, 131_072_000 // classes)))
        top = _log(rng, 1, min(classes, 256))
        c_ = _distill("", rows, classes, top, rng.choice(("f32", "bf16", "f16")), rng.choice((1.0, 2.0, 0.7, 4.0)),
                      rng.random() < 0.7, rng.random() < 0.6, rng.random() < 0.7)
    del c_["name"]
    return c_


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(g, shape, dtype, scale=1.0, shift=0.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    train = case["train"]
    if case["op"] == "ln":
        b, t, c = case["b"], case["t"], case["c"]
        # activations sit beside zero, as a residual stream's channels do
        s["x"] = _randn(g, (b, t, c), T[case["dtype"]], 1.0, 0.3).requires_grad_(train)
        s["w"] = _randn(g, (c,), torch.float32, 0.1, 1.0).requires_grad_(train)
        if case["bias"]:
            s["b"] = _randn(g, (c,), torch.float32, 0.1).requires_grad_(train)
        if train:
            s["dn"] = _randn(g, (b, t, c), T[case["out"]], 1e-2)
    elif case["op"] == "ffn":
        m, k, f, n, dt = case["m"], case["k"], case["f"], case["n"], T[case["dtype"]]
        s["x"] = _randn(g, (m, k), dt).requires_grad_(train)
        for name, shape in (("wg", (f, k)), ("wu", (f, k)), ("wd", (n, f))):
            s[name] = _randn(g, shape, dt, shape[1] ** -0.5).requires_grad_(train)
        if case["bias"]:
            for name, width in (("bg", f), ("bu", f), ("bd", n)):
                s[name] = _randn(g, (width,), dt, 0.1).requires_grad_(train)
        if case["residual"]:
            s["r"] = _randn(g, (m, n), dt).requires_grad_(train)
        if train:
            s["dy"] = _randn(g, (m, n), dt, 1e-2)
    else:
        rows, v, top = case["rows"], case["classes"], case["top"]
        z = torch.randn((rows, v), generator=g, device="cuda").mul_(2.0)
        # the teacher knows some of what the student knows; a program has its top logits stored, in 16 bits
        best = (z * 0.7 + torch.randn((rows, v), generator=g, device="cuda").mul_(2.0)).topk(top, dim=1)
        s["top"], s["cls"] = best.values.to(torch.float16), best.indices.to(torch.int32)
        s["z"] = z.to(T[case["dtype"]]).requires_grad_(train)
        if case["ragged"]:  # fewer entries than there is room for, in some rows none
            kept = (torch.rand((rows,), generator=g, device="cuda") * 1.5 * (top + 1)).long()
            s["cls"].masked_fill_(torch.arange(top, device="cuda") >= kept[:, None], -1)
        if case["labels"]:
            s["y"] = torch.randint(v, (rows,), generator=g, device="cuda")
            if case["ragged"]:
                s["y"].masked_fill_(torch.rand((rows,), generator=g, device="cuda") < 0.1, -100)
        s["weight"] = 0.6 if case["labels"] else 1.0
    return s


# ------------------------------------------------------------------ the plain forms
def _ln_plain(s):
    case = s["case"]
    x, w, out = s["x"].float(), s["w"].float(), T[case["out"]]
    x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    hat = x * r
    n = hat * w
    if case["bias"]:
        n = n + s["b"].float()
    res = {"n": n.to(out)}
    if case["train"]:
        dn = s["dn"].float()
        u = dn * w
        res["d_x"] = (r * (u - u.mean(-1, keepdim=True) - hat * (u * hat).mean(-1, keepdim=True))).to(T[case["dtype"]])
        res["d_w"] = (dn * hat).sum((0, 1))
        if case["bias"]:
            res["d_b"] = dn.sum((0, 1))
    return res


def _act(z, act):
    """The activation and its slope at z."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    if act == "silu":
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g))
    cdf = 0.5 * (1 + torch.erf(z * ROOT_HALF))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * INV_ROOT_2PI


def _ffn_plain(s):
    case, dt = s["case"], T[s["case"]["dtype"]]
    x, wg, wu, wd = (s[k].float() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + s["bg"].float(), u + s["bu"].float()
    a, slope = _act(g, case["act"])
    h = a * u
    y = h @ wd.t()
    if case["bias"]:
        y = y + s["bd"].float()
    if case["residual"]:
        y = y + s["r"].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * slope, dh * a
        out["d_x"] = (dg @ wg + du @ wu).to(dt)
        out["d_wg"], out["d_wu"], out["d_wd"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ h).to(dt)
        if case["bias"]:
            out["d_bg"], out["d_bu"], out["d_bd"] = dg.sum(0).to(dt), du.sum(0).to(dt), dy.sum(0).to(dt)
        if case["residual"]:
            out["d_r"] = s["dy"]
    return out


def _softmax(z):
    """Softmax over the last dimension, and the logarithm of its sum."""
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    return e / total, top + torch.log(total)


def _distill_plain(s):
    case, temp, weight = s["case"], s["case"]["temperature"], s["weight"]
    z = s["z"].float()
    rows = torch.arange(z.shape[0], device=z.device)
    on = s["cls"] >= 0
    cls = torch.where(on, s["cls"], 0).long()
    some = on.any(1)
    t = torch.where(on, s["top"].float() / temp, float("-inf"))
    t = torch.where(some[:, None], t, 0.0)
    p, lse_t = _softmax(t)
    p, log_p = torch.where(on, p, 0.0), t - lse_t
    q, lse = _softmax(z / temp)
    log_q = z[rows[:, None], cls] / temp - lse
    n_soft = torch.clamp(some.sum(), min=1).float()
    soft = torch.where(on, p * (log_p - log_q), 0.0).sum() * (temp * temp)
    loss = weight * soft / n_soft
    if case["labels"]:
        known = s["y"] >= 0
        y = torch.where(known, s["y"], 0)
        q1, lse1 = _softmax(z)
        n_hard = torch.clamp(known.sum(), min=1).float()
        loss = loss + (1 - weight) * torch.where(known, lse1[:, 0] - z[rows, y], 0.0).sum() / n_hard
    out = {"loss": loss}
    if case["train"]:
        ks = weight * temp / n_soft * some.float()[:, None]
        dz = q * ks
        dz.scatter_add_(1, cls, -p * ks)
        if case["labels"]:
            kh = ((1 - weight) / n_hard * known.float())[:, None]
            dz = dz + q1 * kh
            dz.scatter_add_(1, y[:, None], -kh)
        out["d_z"] = dz.to(T[case["dtype"]])
    return out


# ------------------------------------------------------------------ the framework's calls
def _grads(out, s, names, given):
    grads = torch.autograd.grad(out, [s[k] for k in names], given)
    return {"d_" + k: g for k, g in zip(names, grads)}


def _ln_own(s):
    from omniwave_b200 import norm

    n = norm.layer_norm(s["x"], s["w"], s.get("b"), eps=EPS, out_dtype=T[s["case"]["out"]])
    if not s["case"]["train"]:
        return {"n": n}
    return {"n": n.detach(), **_grads(n, s, [k for k in ("x", "w", "b") if k in s], s["dn"])}


def _ffn_own(s):
    from omniwave_b200 import feed_forward

    y = feed_forward.gated_feed_forward(s["x"], s["wg"], s["wu"], s["wd"], gate_bias=s.get("bg"), up_bias=s.get("bu"),
                                        down_bias=s.get("bd"), activation=s["case"]["act"], residual=s.get("r"))
    if not s["case"]["train"]:
        return {"y": y}
    names = [k for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd", "r") if k in s]
    return {"y": y.detach(), **_grads(y, s, names, s["dy"])}


def _distill_own(s):
    from omniwave_b200 import loss

    value = loss.distill_loss(s["z"], s["top"], s["cls"], s.get("y"), temperature=s["case"]["temperature"],
                              weight=s["weight"])
    if not s["case"]["train"]:
        return {"loss": value}
    return {"loss": value.detach(), **_grads(value, s, ["z"], None)}


def run(state):
    op = state["case"]["op"]
    if own:
        return _ln_own(state) if op == "ln" else _ffn_own(state) if op == "ffn" else _distill_own(state)
    with torch.no_grad():
        return _ln_plain(state) if op == "ln" else _ffn_plain(state) if op == "ffn" else _distill_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    width = {"f32": 4, "bf16": 2, "f16": 2}
    train = case["train"]
    if case["op"] == "ln":
        n = case["b"] * case["t"] * case["c"]
        per = width[case["dtype"]] + width[case["out"]]
        return {"bytes": n * per * (2 if train else 1) + 8 * case["c"], "flops": n * (24 if train else 8)}
    if case["op"] == "ffn":
        m, k, f, n = case["m"], case["k"], case["f"], case["n"]
        weights = f * (2 * k + n)
        moved = m * k + weights + m * n * (2 if case["residual"] else 1)
        if train:  # dy comes in, dx and the weights' gradients go out
            moved += m * n + m * k + weights
        return {"bytes": 2 * moved, "flops": 2 * m * f * (2 * k + n) * (3 if train else 1)}
    e = case["rows"] * case["classes"]
    return {"bytes": e * width[case["dtype"]] * (2 if train else 1) + case["rows"] * (6 * case["top"] + 8),
            "flops": e * (10 if train else 4)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _leaves(case, s, names):
    leaves = {k: s[k].detach().double() for k in names if k in s}
    return {k: v.requires_grad_() for k, v in leaves.items()} if case["train"] else leaves


def _exact_ln(case, s):
    leaves = _leaves(case, s, ("x", "w", "b"))
    x = leaves["x"]
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    n = (x - mean) / torch.sqrt(var + EPS) * leaves["w"]
    if "b" in leaves:
        n = n + leaves["b"]
    out = {"n": n.detach()}
    if case["train"]:
        grads = torch.autograd.grad(n, list(leaves.values()), s["dn"].double())
        out.update(("d_" + k, g) for k, g in zip(leaves, grads))
    return out


def _exact_ffn(case, s):
    leaves = _leaves(case, s, ("x", "wg", "wu", "wd", "bg", "bu", "bd", "r"))
    linear = torch.nn.functional.linear
    act = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu}[case["act"]]
    h = act(linear(leaves["x"], leaves["wg"], leaves.get("bg"))) * linear(leaves["x"], leaves["wu"], leaves.get("bu"))
    y = linear(h, leaves["wd"], leaves.get("bd"))
    if "r" in leaves:
        y = y + leaves["r"]
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, list(leaves.values()), s["dy"].double())
        out.update(("d_" + k, g) for k, g in zip(leaves, grads))
    return out


def _exact_distill(case, s):
    z = s["z"].detach().double().requires_grad_(case["train"])
    temp, weight = case["temperature"], s["weight"]
    held = s["cls"] >= 0
    taught = held.any(dim=1)
    teacher = s["top"].double().div(temp).masked_fill(~held, float("-inf"))[taught].log_softmax(dim=1)
    student = z.div(temp).log_softmax(dim=1)[taught].gather(1, s["cls"][taught].clamp(min=0).long())
    terms = torch.where(held[taught], teacher.exp() * (teacher - student), 0.0)
    loss = weight * temp ** 2 * terms.sum() / max(1, int(taught.sum()))
    if case["labels"]:
        known = s["y"] >= 0
        nll = -z.log_softmax(dim=1)[known].gather(1, s["y"][known, None])
        loss = loss + (1 - weight) * nll.sum() / max(1, int(known.sum()))
    out = {"loss": loss.detach()}
    if case["train"]:
        out["d_z"] = torch.autograd.grad(loss, z)[0]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"ln": _exact_ln, "ffn": _exact_ffn, "distill": _exact_distill}[case["op"]](case, s)
