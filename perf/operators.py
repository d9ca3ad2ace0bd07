"""Measured cases of the operators that a training step runs behind the model's body, and of their forward-only forms:

  norm   RMS norm with the residual's addition (forward, backward, and output in 8 bits with scales)
  xent   softmax cross entropy of a linear output layer, logits not kept (loss alone, and loss with both gradients)
  clip   global norm over many gradient tensors, and the scaled gradients

`run` computes them in plain torch operations in 32 bits (`own` false) or by the package's entry points (`own` true).
"""
import math

import torch

own = False

EPS = 1e-6
IGNORE = -100
E4M3_MAX = 448.0
SCALE_FLOOR = 2.0 ** -126     # scale of a group whose values are all (nearly) zero
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

_handle = None


def _context():
    """The process's library context on cuda:0, made once, as a program would."""
    global _handle
    if _handle is None:
        from gern_b200 import api
        _handle = api.Context(0)
    return _handle


# ---- cases ----------------------------------------------------------------------------------------

def listed():
    return [
        # one generated token passing the norm in front of a layer: latency
        {"name": "norm_token", "op": "norm", "way": "forward", "type": "bf16", "rows": 1, "cols": 4096, "group": 0},
        # a training batch's activations through the same norm
        {"name": "norm_batch", "op": "norm", "way": "forward", "type": "bf16", "rows": 16384, "cols": 4096, "group": 0},
        # the gradient of that batch, with the gradient that arrives along the residual
        {"name": "norm_batch_back", "op": "norm", "way": "backward", "type": "bf16", "rows": 16384, "cols": 4096, "group": 0},
        # an fp32 model of odd width, forward and backward: rows that no vector load fits
        {"name": "norm_odd_back", "op": "norm", "way": "backward", "type": "f32", "rows": 2051, "cols": 1021, "group": 0},
        # activations handed to an 8-bit product, a scale for each 128 columns
        {"name": "norm_e4m3", "op": "norm", "way": "e4m3", "type": "bf16", "rows": 4096, "cols": 8192, "group": 128},
        # scoring one token: the whole output matrix is read for one row
        {"name": "xent_token", "op": "xent", "way": "forward", "tokens": 1, "vocab": 65536, "dim": 4096, "ignored": 0.0, "weights": "mean"},
        # evaluation loss of a held-out batch
        {"name": "xent_eval", "op": "xent", "way": "forward", "tokens": 4096, "vocab": 50001, "dim": 2048, "ignored": 0.0, "weights": "mean"},
        # a small model's step, each token with a weight of its own
        {"name": "xent_small_step", "op": "xent", "way": "step", "tokens": 300, "vocab": 1021, "dim": 256, "ignored": 0.1, "weights": "token"},
        # fine-tuning on answers only: most prompt tokens are not counted
        {"name": "xent_answers_step", "op": "xent", "way": "step", "tokens": 5000, "vocab": 32768, "dim": 2048, "ignored": 0.6, "weights": "mean"},
        # a pre-training micro-batch over a large vocabulary
        {"name": "xent_large_step", "op": "xent", "way": "step", "tokens": 8192, "vocab": 131072, "dim": 4096, "ignored": 0.0, "weights": "mean"},
        # a small model's gradients, odd sizes, a dozen tensors
        {"name": "clip_small", "op": "clip", "type": "f32", "out": "f32", "tensors": 12, "numel": 200003},
        # a model of half a billion parameters, hundreds of bf16 gradients
        {"name": "clip_large", "op": "clip", "type": "bf16", "out": "bf16", "tensors": 292, "numel": 536870912},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "xent", "clip"])
    if op == "norm":
        cols = rng.choice([_log(rng, 64, 16384), 8 * _log(rng, 8, 2048), 128 * _log(rng, 1, 128)])
        rows = _log(rng, 1, max(2, min(32768, 67108864 // cols)))
        way = rng.choice(["forward", "backward", "e4m3"])
        group = rng.choice([0, 128]) if way == "e4m3" else 0
        return {"op": "norm", "way": way, "type": rng.choice(["bf16", "bf16", "f32"]), "rows": rows, "cols": cols, "group": group}
    if op == "xent":
        vocab = rng.choice([_log(rng, 500, 131072), 256 * _log(rng, 2, 512)])
        dim = rng.choice([64 * _log(rng, 1, 64), 8 * _log(rng, 16, 512), _log(rng, 100, 4096)])
        tokens = _log(rng, 1, 8192)
        return {"op": "xent", "way": rng.choice(["forward", "step", "step"]), "tokens": tokens, "vocab": vocab, "dim": dim,
                "ignored": round(rng.choice([0.0, rng.uniform(0.05, 0.8)]), 3), "weights": rng.choice(["mean", "token"])}
    kind = rng.choice(["f32", "bf16", "bf16_f32"])
    tensors = _log(rng, 1, 400)
    return {"op": "clip", "type": "f32" if kind == "f32" else "bf16", "out": "bf16" if kind == "bf16" else "f32", "tensors": tensors,
            "numel": _log(rng, max(1000, 2 * tensors), 134217728)}


def _counted(case):
    return case["tokens"] - int(case["tokens"] * case["ignored"])


def _cuts(case):
    """Sizes of a gradient list: one large tensor to four small ones, as matrices and their norms' weights, odd sizes among them."""
    n, total = case["tensors"], case["numel"]
    share = [1.0 if i % 5 == 0 else 0.002 + 0.01 * (i % 3) for i in range(n)]
    whole = sum(share)
    sizes = [max(1, int(total * s / whole)) for s in share]
    sizes[0] = max(1, sizes[0] + total - sum(sizes))
    return sizes


# ---- inputs ---------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": dict(case)}
    if case["op"] == "norm":
        t, shape = TYPES[case["type"]], (case["rows"], case["cols"])
        # activations whose size differs from row to row, a weight near one
        s["x"] = (torch.randn(shape, generator=g, device="cuda") * torch.exp(torch.randn((shape[0], 1), generator=g, device="cuda"))).to(t)
        s["residual"] = torch.randn(shape, generator=g, device="cuda").to(t)
        s["weight"] = (1.0 + 0.1 * torch.randn(shape[1], generator=g, device="cuda")).to(t)
        if case["way"] == "backward":
            s["dy"] = (0.01 * torch.randn(shape, generator=g, device="cuda")).to(t)
    elif case["op"] == "xent":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        # a layer's weights, and activations that lean towards their target's row as a trained model's do
        s["w"] = (0.02 * torch.randn((v, d), generator=g, device="cuda")).to(torch.bfloat16)
        s["targets"] = torch.randint(0, v, (n,), generator=g, device="cuda")
        lean = 6.0 / (0.0004 * d) * torch.rand((n, 1), generator=g, device="cuda")
        s["h"] = (torch.randn((n, d), generator=g, device="cuda") + lean * s["w"][s["targets"]].float()).to(torch.bfloat16)
        left_out = torch.randperm(n, generator=g, device="cuda")[: n - _counted(case)]
        s["targets"][left_out] = IGNORE
        s["dloss"] = (torch.rand(n, generator=g, device="cuda") + 0.5) / n if case["weights"] == "token" else None
    else:
        sizes = _cuts(case)
        flat = 1e-3 * torch.randn(sum(sizes), generator=g, device="cuda")
        s["flat"] = flat.to(TYPES[case["type"]])
        s["grads"] = list(s["flat"].split(sizes))
        s["scaled"] = torch.empty(sum(sizes), device="cuda", dtype=TYPES[case["out"]])
        s["outs"] = list(s["scaled"].split(sizes))
        s["norm"] = torch.empty(1, device="cuda")
        # about a third of the norm that these gradients have: the clipping is at work
        s["max_norm"] = 0.37e-3 * math.sqrt(sum(sizes))
    return s


# ---- one pass -------------------------------------------------------------------------------------

def _norm_plain(s):
    case = s["case"]
    t, cols = TYPES[case["type"]], case["cols"]
    w = s["weight"].float()
    if case["way"] == "backward":
        h, dy = s["x"].float(), s["dy"].float()
        r = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
        wdy = w * dy
        dx = r * wdy - h * (r * r * r * (wdy * h).mean(dim=1, keepdim=True)) + s["residual"].float()
        dw = (dy * h * r).sum(dim=0)
        return {"dx": dx.to(t), "dweight": dw}
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * w
    if case["way"] == "forward":
        return {"y": y.to(t), "h": h.to(t)}
    width = case["group"] or cols
    groups = -(-cols // width)
    padded = torch.zeros((case["rows"], groups * width), device=y.device)
    padded[:, :cols] = y
    parts = padded.view(case["rows"], groups, width)
    scales = torch.clamp(parts.abs().amax(dim=2) / E4M3_MAX, min=SCALE_FLOOR)
    q = torch.clamp(parts / scales[:, :, None], -E4M3_MAX, E4M3_MAX).reshape(case["rows"], groups * width)[:, :cols]
    return {"q": q.to(torch.float8_e4m3fn), "scales": scales, "h": h.to(t)}


def _norm_own(s):
    case, ctx = s["case"], _context()
    x, residual, weight = s["x"], s["residual"], s["weight"]
    if case["way"] == "backward":
        dx = torch.empty_like(x)
        dweight = torch.empty(case["cols"], device="cuda")
        ctx.rmsnorm_backward(s["dy"], x, weight, dx, dweight, EPS, dresidual=residual)
        return {"dx": dx, "dweight": dweight}
    h = torch.empty_like(x)
    if case["way"] == "forward":
        y = torch.empty_like(x)
        ctx.rmsnorm(x, weight, y, EPS, residual=residual, residual_out=h)
        return {"y": y, "h": h}
    groups = -(-case["cols"] // case["group"]) if case["group"] else 1
    q = torch.empty(x.shape, device="cuda", dtype=torch.float8_e4m3fn)
    scales = torch.empty((case["rows"], groups), device="cuda")
    ctx.rmsnorm_e4m3(x, weight, q, scales, EPS, group=case["group"], residual=residual, residual_out=h)
    return {"q": q, "scales": scales, "h": h}


def _xent_plain(s):
    case, targets = s["case"], s["targets"]
    h, w = s["h"].float(), s["w"].float()
    counted = targets != IGNORE
    at = torch.where(counted, targets, 0)[:, None]
    logits = h @ w.T
    top = logits.amax(dim=1, keepdim=True)
    lse = top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True))
    loss = torch.where(counted, (lse - logits.gather(1, at))[:, 0], 0.0)
    total = torch.stack([loss.double().sum(), counted.sum().double()]).float()
    if case["way"] == "forward":
        return {"loss": loss, "total": total}
    weights = s["dloss"] if s["dloss"] is not None else (1.0 / total[1]).expand(case["tokens"])
    weights = torch.where(counted, weights, 0.0)[:, None]
    dlogits = torch.exp(logits - lse) * weights
    dlogits.scatter_add_(1, at, -weights)
    return {"loss": loss, "total": total, "dh": (dlogits @ w).to(torch.bfloat16), "dw": (dlogits.T @ h).to(torch.bfloat16)}


def _xent_own(s):
    case, ctx = s["case"], _context()
    h, w, targets = s["h"], s["w"], s["targets"]
    loss = torch.empty(case["tokens"], device="cuda")
    lse = torch.empty(case["tokens"], device="cuda")
    total = torch.empty(2, device="cuda")
    ctx.linear_xent(h, w, targets, loss, lse, total, ignore_index=IGNORE)
    if case["way"] == "forward":
        return {"loss": loss, "total": total}
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    if s["dloss"] is not None:
        ctx.linear_xent_backward(h, w, targets, lse, dh, dw, dloss=s["dloss"], ignore_index=IGNORE)
    else:
        ctx.linear_xent_backward(h, w, targets, lse, dh, dw, total=total, ignore_index=IGNORE)
    return {"loss": loss, "total": total, "dh": dh, "dw": dw}


def _clip_plain(s):
    squares = torch.stack([x.float().square().sum(dtype=torch.float64) for x in s["grads"]])
    norm = squares.sum().sqrt()
    coefficient = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).float()
    # the result is kept as one buffer cut into the gradients' sizes, as the inputs are
    s["scaled"].copy_(torch.cat([x.float() * coefficient for x in s["grads"]]))
    return {"norm": norm.float().reshape(1), "scaled": s["scaled"]}


def _clip_own(s):
    _context().grad_clip(s["grads"], s["max_norm"], s["norm"], outs=s["outs"])
    return {"norm": s["norm"], "scaled": s["scaled"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return _norm_own(state) if op == "norm" else _xent_own(state) if op == "xent" else _clip_own(state)
    return _norm_plain(state) if op == "norm" else _xent_plain(state) if op == "xent" else _clip_plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    if case["op"] == "norm":
        size, n = TYPES[case["type"]].itemsize, case["rows"] * case["cols"]
        if case["way"] == "forward":       # x, residual -> y, h
            return {"bytes": 4 * n * size + case["cols"] * size, "flops": 5 * n}
        if case["way"] == "backward":      # dy, h, dresidual -> dx, dweight
            return {"bytes": 4 * n * size + case["cols"] * (size + 4), "flops": 10 * n}
        scales = case["rows"] * (-(-case["cols"] // case["group"]) if case["group"] else 1)
        return {"bytes": 3 * n * size + n + 4 * scales + case["cols"] * size, "flops": 7 * n}
    if case["op"] == "xent":
        n, v, d, kept = case["tokens"], case["vocab"], case["dim"], _counted(case)
        read = 2 * v * d + 2 * kept * d + 8 * n
        if case["way"] == "forward":
            return {"bytes": read + 4 * n, "flops": 2 * kept * v * d}
        # the logits are not kept from the loss for the gradient: their product is formed twice
        return {"bytes": read + 4 * n + 2 * v * d + 2 * n * d, "flops": 8 * kept * v * d}
    n = case["numel"]
    return {"bytes": n * (TYPES[case["type"]].itemsize + TYPES[case["out"]].itemsize), "flops": 3 * n}


# ---- 64 bits --------------------------------------------------------------------------------------

def _norm_exact(s):
    case = s["case"]
    x, residual, w = (s[k].to(torch.float64) for k in ("x", "residual", "weight"))
    if case["way"] == "backward":
        dy = s["dy"].to(torch.float64)
        scale = 1.0 / torch.sqrt(torch.sum(x ** 2, dim=1) / case["cols"] + EPS)
        along = torch.sum(dy * w * x, dim=1) * scale ** 2 / case["cols"]
        dx = scale[:, None] * (dy * w - x * along[:, None]) + residual
        return {"dx": dx, "dweight": torch.sum(dy * x * scale[:, None], dim=0)}
    h = x + residual
    y = h / torch.sqrt(torch.sum(h ** 2, dim=1) / case["cols"] + EPS)[:, None] * w[None, :]
    if case["way"] == "forward":
        return {"y": y, "h": h}
    q, scales = torch.empty_like(y), []
    width = case["group"] or case["cols"]
    for first in range(0, case["cols"], width):
        part = y[:, first:first + width]
        scale = torch.clamp(torch.max(torch.abs(part), dim=1).values / E4M3_MAX, min=SCALE_FLOOR)
        q[:, first:first + width] = part / scale[:, None]
        scales.append(scale)
    return {"q": q, "scales": torch.stack(scales, dim=1), "h": h}


def _xent_exact(s):
    case = s["case"]
    n, d = case["tokens"], case["dim"]
    w = s["w"].to(torch.float64)
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    dh = torch.zeros((n, d), dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w) if case["way"] == "step" else None
    places = torch.nonzero(s["targets"] != IGNORE)[:, 0]
    for first in range(0, len(places), 2048):
        rows = places[first:first + 2048]
        h, t = s["h"][rows].to(torch.float64), s["targets"][rows]
        logits = torch.matmul(h, w.T)
        log_p = torch.log_softmax(logits, dim=1)
        del logits
        picked = torch.arange(len(rows), device="cuda")
        loss[rows] = -log_p[picked, t]
        if case["way"] == "step":
            p = log_p.exp_()
            p[picked, t] -= 1.0
            p *= (s["dloss"][rows].to(torch.float64) if s["dloss"] is not None else torch.full((len(rows),), 1.0 / len(places), dtype=torch.float64, device="cuda"))[:, None]
            dh[rows] = torch.matmul(p, w)
            dw += torch.matmul(p.T, h)
    total = torch.tensor([float(loss.sum()), float(len(places))], dtype=torch.float64)
    if case["way"] == "forward":
        return {"loss": loss, "total": total}
    return {"loss": loss, "total": total, "dh": dh, "dw": dw}


def _clip_exact(s):
    norm = math.sqrt(math.fsum(float(torch.sum(x.to(torch.float64) ** 2)) for x in s["grads"]))
    scaled = s["flat"].to(torch.float64) * min(1.0, s["max_norm"] / norm)
    return {"norm": torch.tensor([norm], dtype=torch.float64), "scaled": scaled}


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _norm_exact, "xent": _xent_exact, "clip": _clip_exact}[case["op"]](state)
