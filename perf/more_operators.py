"""Performance cases of what a mixture-of-experts layer needs around its
products: the choice of each token's experts from the router's logits, matrix
products in 8-bit integers with a scale for each token and each channel, dense
and by experts, and the weighted sum of the experts' rows.

Activations are f32; a product quantizes its tokens in the call, or takes them
as 8-bit integers with their scales.  `run` computes either the plain form
(elementary torch operations) or, with `own`, calls the framework.  `exact`
evaluates the definitions in f64.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"


def listed():
    return [
        # ---- experts of each token
        # One token of a decode step, 128 experts: latency.
        {"name": "route_token", "op": "route", "tokens": 1, "experts": 128, "k": 8, "gating": "softmax", "bias": False,
         "groups": 1, "keep": 1, "top": 1, "renorm": True, "scale": 1.0},
        # A step of 61 sequences; 256 experts in groups, balanced by a bias.
        {"name": "route_step", "op": "route", "tokens": 61, "experts": 256, "k": 8, "gating": "sigmoid", "bias": True,
         "groups": 8, "keep": 4, "top": 2, "renorm": True, "scale": 2.5},
        # A prompt batch of 8192 tokens with the same router.
        {"name": "route_prompt", "op": "route", "tokens": 8192, "experts": 256, "k": 8, "gating": "sigmoid",
         "bias": True, "groups": 8, "keep": 4, "top": 2, "renorm": True, "scale": 2.5},
        # ---- dense products
        # One token through a 4096 x 14336 projection.
        {"name": "product_token", "op": "product", "tokens": 1, "rows": 4096, "inner": 14336, "x": "f32"},
        # A decode step of 24 sequences through a 14336 x 4096 projection.
        {"name": "product_step", "op": "product", "tokens": 24, "rows": 14336, "inner": 4096, "x": "f32"},
        # Odd sizes: a ragged prompt batch of 333 tokens.
        {"name": "product_odd", "op": "product", "tokens": 333, "rows": 5003, "inner": 2720, "x": "f32"},
        # A prompt of 4096 tokens, quantized before (several projections share their input).
        {"name": "product_prompt", "op": "product", "tokens": 4096, "rows": 14336, "inner": 4096, "x": "i8"},
        # ---- products by experts
        # One token through the gate and up projections of 8 of 128 experts.
        {"name": "experts_token", "op": "experts", "tokens": 1, "experts": 128, "k": 8, "rows": 1536, "inner": 2048,
         "slots": False, "x": "f32"},
        # A decode step of 48 sequences through the experts' down projections.
        {"name": "experts_step", "op": "experts", "tokens": 48, "experts": 128, "k": 8, "rows": 2048, "inner": 768,
         "slots": True, "x": "f32"},
        # A prompt of 4096 tokens through the gate and up projections.
        {"name": "experts_prompt", "op": "experts", "tokens": 4096, "experts": 128, "k": 8, "rows": 1536,
         "inner": 2048, "slots": False, "x": "f32"},
        # ---- weighted sums
        # A decode step of 7 sequences, added to the shared expert's rows.
        {"name": "combine_step", "op": "combine", "tokens": 7, "k": 8, "rows": 2048, "add": True},
        # A prompt of 4096 tokens.
        {"name": "combine_prompt", "op": "combine", "tokens": 4096, "k": 8, "rows": 2048, "add": False},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    op = rng.choice(("route", "product", "product", "experts", "experts", "combine"))
    if op == "route":
        groups = rng.choice((1, 1, 4, 8))
        experts = groups * log_int(max(1, 8 // groups), 512 // groups)
        keep = rng.randint(1, groups)
        return {"op": op, "tokens": log_int(1, 8192 * 256 // experts), "experts": experts,
                "k": rng.randint(1, min(16, experts // groups * keep)),
                "gating": rng.choice(("softmax", "sigmoid", "softmax_chosen")), "bias": rng.random() < 0.5,
                "groups": groups, "keep": keep, "top": rng.choice((1, 2)), "renorm": rng.random() < 0.7,
                "scale": rng.choice((1.0, 2.5))}
    if op == "product":
        rows, inner = log_int(256, 16384), log_int(256, 16384)
        tokens = log_int(1, min(8192, 4096 * 14336 * 4096 // (rows * inner), 2 ** 28 // (4 * (rows + inner))))
        return {"op": op, "tokens": tokens, "rows": rows, "inner": inner, "x": rng.choice(("f32", "f32", "i8"))}
    if op == "combine":
        k, rows = rng.randint(1, 16), log_int(256, 8192)
        return {"op": op, "tokens": log_int(1, 4096 * 8 * 2048 // (k * rows)), "k": k, "rows": rows,
                "add": rng.random() < 0.5}
    experts, k, rows, inner = log_int(8, 256), rng.randint(1, 8), log_int(256, 4096), log_int(256, 4096)
    experts = min(experts, max(8, 128 * 1536 * 2048 // (rows * inner)))
    slots = rng.random() < 0.5
    most = min(8192, 4096 * 8 * 1536 * 2048 // (k * rows * inner), 2 ** 27 // (2 * k * (rows + slots * inner)))
    return {"op": op, "tokens": log_int(1, most), "experts": experts, "k": min(k, experts), "rows": rows,
            "inner": inner, "slots": slots, "x": rng.choice(("f32", "f32", "i8"))}


# ---------------------------------------------------------------- inputs


def _padded(rows, inner):
    """8-bit rows as the framework's quantizer lays them: 16-byte aligned, the padding zeros."""
    q = torch.zeros(*rows, -(-inner // 16) * 16, dtype=torch.int8, device=DEV)
    return q[..., :inner]


def _weights(gen, *shape):
    """8-bit weights with a scale for each channel, as quantizing near normal ones leaves them."""
    w = _padded(shape[:-1], shape[-1])
    w.view(-1, *shape[-2:]).copy_(torch.randn(shape, generator=gen, device=DEV, dtype=torch.bfloat16)
                                  .mul_(32).round_().clamp_(-127, 127).view(-1, *shape[-2:]))
    scale = (0.5 + torch.rand(shape[:-1], generator=gen, device=DEV)) * (2.0 / 127 / math.sqrt(shape[-1]))
    return w, scale


def _tokens(gen, kind, *shape):
    """Activations with a few channels far above the others, and their scales where they are 8-bit."""
    far = 1 + 15 * (torch.rand(shape[-1], generator=gen, device=DEV) < 0.005).float()
    x = torch.randn(shape, generator=gen, device=DEV) * far * (0.2 + torch.rand(shape[:-1], generator=gen, device=DEV)[..., None])
    if kind == "f32":
        return x, None
    scale = x.abs().amax(-1) / 127
    q = _padded(shape[:-1], shape[-1])
    q.copy_((x / scale[..., None]).round())
    return q, scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s, n, op = {"case": case}, case["tokens"], case["op"]
    if op == "route":
        s["logits"] = torch.randn(n, case["experts"], generator=gen, device=DEV) * 1.7
        s["bias"] = torch.randn(case["experts"], generator=gen, device=DEV) * 0.1 if case["bias"] else None
    elif op == "product":
        s["w"], s["w_scale"] = _weights(gen, case["rows"], case["inner"])
        s["x"], s["x_scale"] = _tokens(gen, case["x"], n, case["inner"])
    elif op == "experts":
        s["w"], s["w_scale"] = _weights(gen, case["experts"], case["rows"], case["inner"])
        s["x"], s["x_scale"] = _tokens(gen, case["x"], n, case["k"] if case["slots"] else 1, case["inner"])
        # Some experts are asked for more often than others.
        liked = torch.randn(case["experts"], generator=gen, device=DEV) * 0.4
        logits = torch.randn(n, case["experts"], generator=gen, device=DEV) + liked
        s["ids"] = torch.topk(logits, case["k"]).indices.int().contiguous()
    else:
        s["y"] = torch.randn(n, case["k"], case["rows"], generator=gen, device=DEV)
        s["weights"] = torch.softmax(torch.randn(n, case["k"], generator=gen, device=DEV), -1)
        s["add"] = torch.randn(n, case["rows"], generator=gen, device=DEV) if case["add"] else None
    return s


# ---------------------------------------------------------------- plain forms


def _plain_route(s):
    c, logits = s["case"], s["logits"]
    n, e = logits.shape
    # The order in f64: scores closer than f32 tells apart would swap their experts.
    wide = logits.double()
    if c["gating"] == "softmax":
        score = (wide - wide.amax(-1, keepdim=True)).exp()
        score = score / score.sum(-1, keepdim=True)
    elif c["gating"] == "sigmoid":
        score = 1 / (1 + (-wide).exp())
    else:
        score = wide
    p = score.float()
    if s["bias"] is not None:
        score = score + s["bias"].double()
    if c["groups"] > 1:
        grouped = score.view(n, c["groups"], -1)
        best = grouped.sort(dim=-1, descending=True).values[..., :c["top"]].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :c["keep"]]
        seen = (kept[:, :, None] == torch.arange(c["groups"], device=DEV)).any(1)
        score = torch.where(seen[..., None], grouped, -math.inf).view(n, e)
    ids = score.sort(dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    w = p.gather(1, ids)
    if c["gating"] == "softmax_chosen":
        w = (w - w.amax(-1, keepdim=True)).exp()
        w = w / w.sum(-1, keepdim=True)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=2.0 ** -14)
    return {"ids": ids.int(), "weights": w * c["scale"]}


def _plain_tokens(s):
    """The 8-bit values, as f32, and the scales."""
    x, scale = s["x"], s["x_scale"]
    if scale is not None:
        return x.float(), scale
    scale = x.abs().amax(-1) / 127
    return (x / scale[..., None]).round(), scale


def _plain_experts(s):
    c, ids = s["case"], s["ids"].long()
    q, scale = _plain_tokens(s)
    n, k, e = c["tokens"], c["k"], c["experts"]
    q, scale = (t.expand(n, k, *t.shape[2:]).flatten(0, 1) for t in (q, scale))
    # The pairs of an expert side by side, as many places for each as the fullest needs.
    flat = ids.flatten()
    if n * k <= e:
        # Few pairs: each with a copy of its expert's weights.
        out = (s["w"][flat].float() @ q[:, :, None])[..., 0] * scale[:, None] * s["w_scale"][flat]
        return out.view(n, k, -1)
    order = flat.sort(stable=True).indices
    count = torch.zeros(e, dtype=torch.long, device=DEV).index_add_(0, flat, torch.ones_like(flat))
    place = torch.empty_like(flat)
    place[order] = torch.arange(n * k, device=DEV) - (count.cumsum(0) - count)[flat[order]]
    most = int(count.max())
    at = flat * most + place
    rows = torch.zeros(e * most, c["inner"], device=DEV)
    rows[at] = q
    out = rows.view(e, most, -1) @ s["w"].float().transpose(1, 2).contiguous()
    out = out.flatten(0, 1)[at] * scale[:, None] * s["w_scale"][flat]
    return out.view(n, k, -1)


def _plain(s):
    op = s["case"]["op"]
    if op == "route":
        return _plain_route(s)
    if op == "product":
        q, scale = _plain_tokens(s)
        return q @ s["w"].float().T.contiguous() * scale[:, None] * s["w_scale"]
    if op == "experts":
        return _plain_experts(s)
    out = (s["y"] * s["weights"][..., None]).sum(1)
    return out if s["add"] is None else out + s["add"]


# ---------------------------------------------------------------- the framework


def _framework():
    path = os.path.join(os.getcwd(), "llama.zig_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ggml_hip
    return ggml_hip


def _own(s):
    G, c = _framework(), s["case"]
    if c["op"] == "route":
        ids, weights = G.route(s["logits"], c["k"], gating=c["gating"], bias=s["bias"], groups=c["groups"],
                               keep=c["keep"], top=c["top"], renormalize=c["renorm"], scale=c["scale"])
        return {"ids": ids, "weights": weights}
    if c["op"] == "product":
        return G.mul_mat_i8(s["w"], s["w_scale"], s["x"], s["x_scale"])
    if c["op"] == "experts":
        return G.mul_mat_id_i8(s["w"], s["w_scale"], s["x"], s["ids"], s["x_scale"])
    return G.combine(s["y"], s["weights"], add=s["add"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- floors


def work(case):
    n, op = case["tokens"], case["op"]
    if op == "route":
        e = case["experts"]
        return {"bytes": 4 * n * e + 8 * n * case["k"] + (4 * e if case["bias"] else 0), "flops": n * e * (2 + case["k"])}
    if op == "combine":
        k, m = case["k"], case["rows"]
        return {"bytes": 4 * n * (k * m + k + m * (2 if case["add"] else 1)), "flops": 2 * n * k * m}
    m, inner, size = case["rows"], case["inner"], 4 if case["x"] == "f32" else 1
    scales = 4 if case["x"] == "i8" else 0
    if op == "product":
        return {"bytes": m * (inner + 4) + n * (inner * size + scales) + 4 * n * m, "flops": 2 * n * m * inner}
    e, k = case["experts"], case["k"]
    asked = e * (1 - (1 - k / e) ** n)  # experts that some token asks for, were they all liked the same
    return {"bytes": int(asked * m * (inner + 4)) + n * (k if case["slots"] else 1) * (inner * size + scales) + 4 * n * k * (m + 1),
            "flops": 2 * n * k * m * inner}


# ---------------------------------------------------------------- definitions


def _exact_route(case, s):
    """Row by row over sets of experts, from the definition."""
    if case["tokens"] * case["experts"] > 1 << 19:
        return None  # Python's loops would take too long
    import numpy as np
    logits = s["logits"].cpu().numpy().astype(np.float64)
    bias = np.zeros(case["experts"]) if s["bias"] is None else s["bias"].cpu().numpy().astype(np.float64)
    size, k = case["experts"] // case["groups"], case["k"]
    ids, weights = np.zeros((len(logits), k), np.int32), np.zeros((len(logits), k))
    for t, row in enumerate(logits):
        if case["gating"] == "softmax":
            p = np.exp(row - row.max())
            p = p / math.fsum(p)
        else:
            p = 1 / (1 + np.exp(-row)) if case["gating"] == "sigmoid" else row
        score = p + bias
        of_group = [sum(sorted(score[g * size:(g + 1) * size])[::-1][:case["top"]]) for g in range(case["groups"])]
        kept = sorted(range(case["groups"]), key=lambda g: (-of_group[g], g))[:case["keep"]]
        open_ = [e for g in kept for e in range(g * size, (g + 1) * size)]
        ids[t] = sorted(open_, key=lambda e: (-score[e], e))[:k]
        w = p[ids[t]]
        if case["gating"] == "softmax_chosen":
            w = np.exp(w - w.max())
            w = w / math.fsum(w)
        if case["renorm"]:
            w = w / max(math.fsum(w), 2.0 ** -14)
        weights[t] = w * case["scale"]
    return {"ids": torch.from_numpy(ids), "weights": torch.from_numpy(weights)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, s)
    if case["op"] == "combine":
        out = torch.bmm(s["weights"].double()[:, None], s["y"].double())[:, 0]
        return out if s["add"] is None else out + s["add"].double()
    x = s["x"].double()
    if s["x_scale"] is None:
        # The quantizer's divisions are f32 ones: those of f64, rounded once more, are the same.
        scale = (x.abs().amax(-1) / 127).float().double()
        x = (x / scale[..., None]).float().double().round()
    else:
        scale = s["x_scale"].double()
    if case["op"] == "product":
        return torch.mm(x * scale[:, None], s["w"].double().t().contiguous()) * s["w_scale"].double()
    n, k = case["tokens"], case["k"]
    x = (x * scale[..., None]).expand(n, k, -1)
    out = torch.zeros(n, k, case["rows"], dtype=torch.float64, device=DEV)
    for e in range(case["experts"]):
        t, j = (s["ids"] == e).nonzero(as_tuple=True)
        out[t, j] = torch.mm(x[t, j], s["w"][e].double().t().contiguous()) * s["w_scale"][e].double()
    return out
