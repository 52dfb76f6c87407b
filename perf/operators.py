"""The training-step operators around the attention layer, as measured: layer norm with its residual
add, the vocabulary loss, and the gradient norm with clipping, in plain torch and through this package.

Layer norm      h = x + residual (stored in x's type; h = x without a residual), y = norm of the stored
                h times weight plus bias; its backward gives the gradient of x (and of the residual, the
                same), including what reaches h directly, and of weight and bias.
Vocabulary loss z = hidden @ weight^T, loss_t = logsumexp_v(z_tv) - z_t,target; ignored targets count
                nothing; "mean" divides by the kept targets (by one if none is kept).
Clipping        norm = 2-norm over all gradients after removing the loss scale; every gradient times
                min(1, max_norm / (norm + 1e-6)) / loss_scale, written to flat storage.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
IGNORE = -100
EPS = 1e-5

# the most a drawn case may cost: the largest listed ones
MOST_NORM = 65536 * 2048 * 2  # bytes of one tensor
MOST_LOSS = 16384 * 65536 * 1024


def listed():
    return [
        # one new token through a norm with its residual: latency
        {"name": "norm_one_token", "op": "norm", "rows": 1, "dim": 512, "type": "fp16", "train": False, "residual": True},
        # odd rows and width in 32 bits, no residual: nothing aligns
        {"name": "norm_odd_fp32", "op": "norm", "rows": 333, "dim": 1001, "type": "fp32", "train": True, "residual": False},
        # the 64 x 197 token batch of the image encoder, forward and backward
        {"name": "norm_encoder", "op": "norm", "rows": 64 * 197, "dim": 768, "type": "fp16", "train": True, "residual": True},
        # the longest configuration's batch, 8 x 8192 tokens, width 2048
        {"name": "norm_long", "op": "norm", "rows": 8 * 8192, "dim": 2048, "type": "bf16", "train": True, "residual": True},
        # scoring one token against a large vocabulary: the weight is read once
        {"name": "loss_one_token", "op": "loss", "tokens": 1, "vocab": 32768, "dim": 1024, "type": "bf16", "train": False, "reduction": "none", "ignored": 0.0},
        # a small training batch: 2 x 128 tokens, small vocabulary
        {"name": "loss_small", "op": "loss", "tokens": 256, "vocab": 1000, "dim": 256, "type": "fp16", "train": True, "reduction": "mean", "ignored": 0.1},
        # ragged: 8 x 197 tokens, odd vocabulary, per-token gradients, much padding
        {"name": "loss_ragged", "op": "loss", "tokens": 8 * 197, "vocab": 50001, "dim": 768, "type": "fp16", "train": True, "reduction": "none", "ignored": 0.4},
        # the causal configuration's batch, 8 x 1024 tokens, width 512
        {"name": "loss_causal", "op": "loss", "tokens": 8 * 1024, "vocab": 32768, "dim": 512, "type": "fp16", "train": True, "reduction": "mean", "ignored": 0.05},
        # the long configuration's batch, 4 x 4096 tokens, width 1024
        {"name": "loss_long", "op": "loss", "tokens": 4 * 4096, "vocab": 65536, "dim": 1024, "type": "bf16", "train": True, "reduction": "mean", "ignored": 0.05},
        # the gradients of one small layer, nothing to clip but the scale to remove
        {"name": "clip_layer", "op": "clip", "blocks": 1, "dim": 256, "odd": 0, "type": "fp16", "out": "fp32", "scale": 1024.0, "share": 2.0},
        # a twelve-block encoder of width 768, fp16 gradients to 32-bit ones
        {"name": "clip_encoder", "op": "clip", "blocks": 12, "dim": 768, "odd": 0, "type": "fp16", "out": "fp32", "scale": 1024.0, "share": 0.25},
        # tensors of odd lengths packed without gaps, gradients kept in their type
        {"name": "clip_ragged", "op": "clip", "blocks": 3, "dim": 512, "odd": 7, "type": "bf16", "out": "bf16", "scale": 1.0, "share": 0.1},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "loss", "loss", "clip"])
    if op == "norm":
        dim = _log(rng, 64, 4096) if rng.random() < 0.5 else 8 * _log(rng, 8, 512)
        kind = rng.choice(sorted(TYPES))
        rows = min(_log(rng, 1, 65536), MOST_NORM // (dim * (4 if kind == "fp32" else 2)))
        return {"op": op, "rows": rows, "dim": dim, "type": kind, "train": rng.random() < 0.7,
                "residual": rng.random() < 0.6}
    if op == "loss":
        dim, vocab = 8 * _log(rng, 32, 256), _log(rng, 1000, 131072)
        tokens = max(1, min(_log(rng, 1, 16384), MOST_LOSS // (dim * vocab)))
        return {"op": op, "tokens": tokens, "vocab": vocab, "dim": dim, "type": rng.choice(["fp16", "bf16"]),
                "train": rng.random() < 0.7, "reduction": rng.choice(["mean", "sum", "none"]),
                "ignored": round(rng.uniform(0.0, 0.5), 3)}
    kind = rng.choice(sorted(TYPES))
    return {"op": op, "blocks": _log(rng, 1, 9 if kind == "fp32" else 12), "dim": 8 * _log(rng, 8, 96), "odd": rng.choice([0, 0, 1, 3, 7]),
            "type": kind, "out": rng.choice([kind, "fp32"]), "scale": rng.choice([1.0, 256.0, 1024.0]),
            "share": round(rng.uniform(0.05, 3.0), 3)}


def _sizes(case):
    """Element counts of the gradients of `blocks` pre-norm encoder blocks of width `dim` (8 attention
    heads' gates of 16, a four times wider MLP); `odd` lengthens every tensor, so that none aligns."""
    d = case["dim"]
    block = [d, d, d * 128, 128, 128, d * d, d, d, 4 * d * d, 4 * d, 4 * d * d, d]
    return [n + case["odd"] for n in block * case["blocks"]]


def _seed(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _normal(g, *size):
    return torch.randn(*size, generator=g, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    g = _seed(seed)
    kind = TYPES[case["type"]]
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        # a residual stream: a few wide channels and an offset beside unit noise
        wide = 1.0 + 8.0 * (torch.rand(dim, generator=g, device="cuda") < 0.01)
        s = {"op": "norm", "train": case["train"], "x": (_normal(g, rows, dim) * wide + 0.3).to(kind),
             "residual": (0.5 * _normal(g, rows, dim)).to(kind) if case["residual"] else None,
             "weight": (1.0 + 0.1 * _normal(g, dim)).to(kind), "bias": (0.1 * _normal(g, dim)).to(kind)}
        if case["train"]:
            s["grad_y"] = _normal(g, rows, dim).to(kind)
            s["grad_h"] = _normal(g, rows, dim).to(kind) if case["residual"] else None
        return s
    if case["op"] == "loss":
        T, V, D = case["tokens"], case["vocab"], case["dim"]
        weight = (2.0 * D ** -0.5 * _normal(g, V, D)).to(kind)
        target = torch.randint(0, V, (T,), generator=g, device="cuda")
        # a partly trained model: hidden states lean towards their target's row
        hidden = (_normal(g, T, D) + 2.0 * weight[target].float()).to(kind)
        target[torch.rand(T, generator=g, device="cuda") < case["ignored"]] = IGNORE
        s = {"op": "loss", "train": case["train"], "reduction": case["reduction"], "hidden": hidden, "weight": weight,
             "target": target}
        if case["train"]:
            # fp16 gradients come with a loss scale, without which they would underflow
            scale = 1024.0 if case["type"] == "fp16" and case["reduction"] == "mean" else 1.0
            s["grad"] = (torch.rand(T, generator=g, device="cuda") + 0.5 if case["reduction"] == "none" else
                         torch.full((), scale, device="cuda"))
        return s
    sizes = _sizes(case)
    # layers' gradients differ in size by orders of magnitude
    grads = [(_normal(g, n) * (case["scale"] * 10.0 ** (-1.0 - i % 3))).to(kind) for i, n in enumerate(sizes)]
    flat = torch.empty(sum(sizes), device="cuda", dtype=TYPES[case["out"]])
    expected = math.sqrt(sum(n * 10.0 ** (-2.0 - 2 * (i % 3)) for i, n in enumerate(sizes)))
    return {"op": "clip", "grads": grads, "flat": flat, "out": list(flat.split(sizes)), "scale": case["scale"],
            "max_norm": case["share"] * expected}


def _plain_norm(s):
    x = s["x"]
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    hf, w, b = h.float(), s["weight"].float(), s["bias"].float()
    c = hf - hf.mean(-1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    n = c * rstd
    out = {"y": (n * w + b).to(x.dtype)}
    if s["residual"] is not None:
        out["h"] = h
    if s["train"]:
        dy = s["grad_y"].float()
        d = dy * w
        dx = rstd * (d - d.mean(-1, keepdim=True) - n * (d * n).mean(-1, keepdim=True))
        if s["grad_h"] is not None:
            dx = dx + s["grad_h"].float()
        out.update(dx=dx.to(x.dtype), dweight=(dy * n).sum(0).to(x.dtype), dbias=dy.sum(0).to(x.dtype))
    return out


def _plain_loss(s):
    h, w, target = s["hidden"].float(), s["weight"].float(), s["target"]
    keep = target != IGNORE
    at = target.clamp(min=0)[:, None]
    z = h @ w.T
    top = z.amax(-1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(-1, keepdim=True)
    each = torch.where(keep, (top + total.log() - z.gather(1, at))[:, 0], 0.0)
    kept = keep.sum().clamp(min=1).float()
    reduction = s["reduction"]
    out = {"loss": each if reduction == "none" else each.sum() if reduction == "sum" else each.sum() / kept,
           "lse": (top + total.log())[:, 0]}
    if s["train"]:
        g = s["grad"] / kept if reduction == "mean" else s["grad"]
        g = torch.where(keep, g, 0.0)[:, None]
        dz = e / total
        dz.scatter_add_(1, at, torch.full_like(total, -1.0))
        dz = dz * g
        out.update(dhidden=(dz @ w).to(s["hidden"].dtype), dweight=(dz.T @ h).to(s["weight"].dtype))
    return out


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt() / s["scale"]
    by = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0) / s["scale"]
    flat = torch.cat([(g.float() * by).to(s["flat"].dtype) for g in s["grads"]])
    return {"norm": norm, "flat": flat}


def run(s):
    if not own:
        return {"norm": _plain_norm, "loss": _plain_loss, "clip": _plain_clip}[s["op"]](s)
    import morphottention_b200 as mo
    if s["op"] == "norm":
        y, mean, rstd, *h = mo.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS, s["residual"])
        out = {"y": y}
        if h:
            out["h"] = h[0]
        if s["train"]:
            out["dx"], out["dweight"], out["dbias"] = mo.layer_norm_backward(
                s["grad_y"], h[0] if h else s["x"], s["weight"], mean, rstd, s["grad_h"])
        return out
    if s["op"] == "loss":
        loss, lse = mo.linear_cross_entropy_forward(s["hidden"], s["weight"], s["target"], IGNORE, s["reduction"])
        out = {"loss": loss, "lse": lse}
        if s["train"]:
            out["dhidden"], out["dweight"] = mo.linear_cross_entropy_backward(
                s["grad"], s["hidden"], s["weight"], s["target"], lse, IGNORE, s["reduction"])
        return out
    norm = mo.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"], loss_scale=s["scale"])
    return {"norm": norm, "flat": s["flat"]}


def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    if case["op"] == "norm":
        one = case["rows"] * case["dim"]
        forward, backward = (4, 4) if case["residual"] else (2, 3)  # tensors read and written
        tensors = forward + (backward if case["train"] else 0)
        rows = case["rows"] * 8 * (2 if case["train"] else 1)
        return {"bytes": tensors * one * size[case["type"]] + rows + 4 * case["dim"] * size[case["type"]],
                "flops": one * (22 if case["train"] else 9)}
    if case["op"] == "loss":
        T, V, D = case["tokens"], case["vocab"], case["dim"]
        passes = 2 if case["train"] else 1  # hidden and weight read, their gradients written
        return {"bytes": passes * 2 * (T * D + V * D) + 16 * T, "flops": (6 if case["train"] else 2) * T * V * D}
    n = sum(_sizes(case))
    return {"bytes": n * (size[case["type"]] + size[case["out"]]), "flops": 4 * n}


def _exact_norm(s):
    x = s["x"].double()
    # h is stored in x's type, and the norm is of what is stored
    h = x if s["residual"] is None else (x + s["residual"].double()).to(s["x"].dtype).double()
    mu = h.mean(-1, keepdim=True)
    sigma = ((h - mu).pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    n = (h - mu) / sigma
    w = s["weight"].double()
    out = {"y": torch.addcmul(s["bias"].double(), n, w)}
    if s["residual"] is not None:
        out["h"] = x + s["residual"].double()
    if s["train"]:
        dy = s["grad_y"].double()
        out["dweight"] = torch.einsum("rd,rd->d", dy, n)
        out["dbias"] = dy.sum(0)
        dy = dy * w
        # project out the constant and the normalised row, the directions the norm does not see
        dx = (dy - dy.mean(-1, keepdim=True) - n * torch.einsum("rd,rd->r", dy, n)[:, None] / n.shape[1]) / sigma
        out["dx"] = dx if s["grad_h"] is None else dx + s["grad_h"].double()
    return out


def _exact_loss(s):
    h, w, target = s["hidden"].double(), s["weight"].double(), s["target"]
    T = target.numel()
    live = (target != IGNORE).double()
    rows = torch.arange(T, device=target.device)
    label = torch.where(target == IGNORE, torch.zeros_like(target), target)
    z = torch.einsum("td,vd->tv", h, w)
    own_z = z[rows, label]
    lse = torch.logsumexp(z, 1)
    each = (lse - own_z) * live
    share = 1.0 / max(1.0, float(live.sum())) if s["reduction"] == "mean" else 1.0
    out = {"loss": each if s["reduction"] == "none" else each.sum() * share, "lse": lse}
    if s["train"]:
        g = live * share * s["grad"].double()
        z.sub_(lse[:, None]).exp_()
        z[rows, label] -= 1.0
        z.mul_(g[:, None])
        out["dhidden"] = torch.einsum("tv,vd->td", z, w)
        out["dweight"] = torch.einsum("tv,td->vd", z, h)
    return out


def _exact_clip(s):
    every = torch.cat([g.double() for g in s["grads"]]) / s["scale"]
    norm = torch.linalg.vector_norm(every)
    return {"norm": norm, "flat": every * min(1.0, float(s["max_norm"] / (norm + 1e-6)))}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "loss": _exact_loss, "clip": _exact_clip}[case["op"]](s)
