"""Performance cases of the attention half of a decoder layer: rotary positions
with the store into a paged key-value cache, attention over that cache (one new
token per sequence, and many, with a window and first tokens that stay
visible), and the upkeep of its pages.

The cache of a layer is two f16 or bf16 tensors [pages, kv heads, page size,
head dim]; a sequence's tokens are found through its row of a page table.
Activations are f32.  `run` computes either the plain form (elementary torch
operations in f32) or, with `own`, calls the framework.  `exact` evaluates the
definitions in f64.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # ---- rotary positions, and the store of keys and values into the cache
        # One token of one sequence: a decode step, where the call's latency counts.
        {"name": "rope_step", "op": "rope", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "layout": "half", "stretch": 1.0, "ctx": 8192, "page": 64, "type": "f16"},
        # A step of 200 sequences far into stretched contexts, part of each head rotated.
        {"name": "rope_batch", "op": "rope", "tokens": 200, "heads": 32, "kv_heads": 32, "dim": 80, "rot": 32,
         "layout": "interleaved", "stretch": 8.0, "ctx": 131072, "page": 16, "type": "bf16"},
        # A prompt batch of 8192 tokens.
        {"name": "rope_prompt", "op": "rope", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "layout": "half", "stretch": 4.0, "ctx": 32768, "page": 64, "type": "f16"},
        # ---- attention of one new token per sequence
        # One sequence, an ordinary chat's length.
        {"name": "step_short", "op": "step", "seqs": 1, "kv": 333, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "window": 0, "sinks": 0, "type": "f16"},
        # One sequence over a long document.
        {"name": "step_long", "op": "step", "seqs": 1, "kv": 131072, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "sinks": 0, "type": "f16"},
        # 48 sequences of ragged lengths served together.
        {"name": "step_batch", "op": "step", "seqs": 48, "kv": 8191, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 32, "window": 0, "sinks": 0, "type": "bf16"},
        # 100 streams in a window of 1024 tokens behind four first ones, a head of keys for each of queries.
        {"name": "step_window", "op": "step", "seqs": 100, "kv": 5000, "heads": 32, "kv_heads": 32, "dim": 64,
         "page": 16, "window": 1024, "sinks": 4, "type": "f16"},
        # ---- attention of many new tokens
        # A whole prompt of 4096 tokens.
        {"name": "prompt", "op": "many", "seqs": 1, "new": 4096, "kv": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "sinks": 0, "type": "f16"},
        # Three ragged prompts in a window behind four first tokens.
        {"name": "prompt_window", "op": "many", "seqs": 3, "new": 2500, "kv": 2500, "heads": 32, "kv_heads": 4,
         "dim": 128, "page": 32, "window": 1024, "sinks": 4, "type": "bf16"},
        # Drafts of 13 tokens verified at once for two sequences with long contexts.
        {"name": "verify", "op": "many", "seqs": 2, "new": 13, "kv": 20000, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "window": 0, "sinks": 0, "type": "f16"},
        # ---- pages
        # 64 sequences forked: the partly filled last page of each is copied.
        {"name": "fork", "op": "copy", "pages": 1024, "copies": 64, "kv_heads": 8, "dim": 128, "page": 16,
         "type": "f16"},
        # A pool whose pages are half in use, scattered, moved together.
        {"name": "compact", "op": "compact", "pages": 4096, "seqs": 64, "held": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "type": "f16"},
    ]


def draw(rng):
    def log_int(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return n + (n == 3 << 10)

    op = rng.choice(("rope", "step", "step", "many", "many", "copy", "compact"))
    heads, kv_heads = rng.choice(((32, 8), (32, 8), (32, 4), (32, 32), (40, 8), (14, 2), (16, 1)))
    case = {"op": op, "kv_heads": kv_heads, "dim": rng.choice((64, 80, 128, 128, 256)), "page": 2 ** rng.randint(4, 7),
            "type": rng.choice(("f16", "bf16"))}
    if op == "rope":
        rot = rng.choice((case["dim"], case["dim"], 32, case["dim"] // 2))
        return dict(case, heads=heads, tokens=log_int(1, 8192 * 48 * 128 // ((heads + 2 * kv_heads) * case["dim"])),
                    rot=rot, layout=rng.choice(("half", "interleaved")), stretch=rng.choice((1.0, 1.0, 4.0, 8.0)),
                    ctx=rng.choice((8192, 32768, 131072)))
    if op == "copy":
        pages = log_int(128, 2 ** 26 // (kv_heads * case["dim"] * case["page"]) + 256)
        return dict(case, pages=pages, copies=log_int(1, pages // 2))
    if op == "compact":
        pages = log_int(128, 2 ** 26 // (kv_heads * case["dim"] * case["page"]) + 256)
        seqs = log_int(1, 64)
        return dict(case, pages=pages, seqs=seqs, held=max(1, int(pages * rng.uniform(0.1, 0.9)) // seqs))
    window, sinks = rng.choice(((0, 0), (0, 0), (1024, 4), (log_int(1, 4096), rng.randint(0, 40))))
    case = dict(case, heads=heads, window=window, sinks=sinks)
    if op == "step":
        seqs = log_int(1, 128)
        return dict(case, seqs=seqs, kv=log_int(1, 2 ** 27 // (seqs * max(kv_heads, 4) * case["dim"])))
    seqs = rng.choice((1, 1, 2, 3, 8))
    new = log_int(2, 4096 // seqs)
    most = min(2 ** 27 // (seqs * max(kv_heads, 4) * case["dim"]), 2 ** 36 // (new * seqs * heads * case["dim"]))
    return dict(case, seqs=seqs, new=new, kv=log_int(new, max(new, most)))


# ---------------------------------------------------------------- inputs


def _lengths(case):
    """Ragged cache lengths, the longest case["kv"], and new tokens of each sequence, at most its length."""
    n = case["seqs"]
    share = [1.0 if i == 0 else 0.1 + 0.9 * ((i * 0.6180339887) % 1.0) for i in range(n)]
    lens = [max(1, round(case["kv"] * s)) for s in share]
    if case["op"] == "step":
        return lens, [1] * n
    return lens, [min(k, max(1, round(case["new"] * s))) for k, s in zip(lens, share)]


def _steps(rot, stretch, base=500000.0, ctx=8192):
    """Per rotated pair, the turn that one position adds, as a whole number of
    2^-64 turns (wrapping), and the magnitude that goes with the stretch: the
    low frequencies interpolated by it, the high ones kept, a ramp between
    those that turn 32 times and once over ctx positions (YaRN)."""
    def pair_of(turns):
        return rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(0, math.floor(pair_of(32.0))), min(rot - 1, math.ceil(pair_of(1.0)))
    steps = []
    for i in range(rot // 2):
        keep = 1.0 - min(1.0, max(0.0, (i - low) / max(0.001, high - low))) if stretch != 1.0 else 1.0
        turns = base ** (-2.0 * i / rot) / (2 * math.pi) * (keep + (1.0 - keep) / stretch)
        whole = round(turns * 2.0 ** 64) % 2 ** 64
        steps.append(whole - 2 ** 64 if whole >= 2 ** 63 else whole)
    return steps, 1.0 + 0.1 * math.log(stretch)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _cache(gen, case, pages):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    return [_normal(gen, *shape).to(TYPES[case["type"]]) for _ in range(2)]


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    perm = lambda n: torch.randperm(n, generator=gen, device=DEV)  # noqa: E731
    op, page = case["op"], case["page"]
    if op == "rope":
        n = case["tokens"]
        pages = -(-n // page) + 3
        steps, scale = _steps(case["rot"], case["stretch"])
        k_cache, v_cache = _cache(gen, case, pages)
        rows = [_normal(gen, n, h, case["dim"]) for h in (case["heads"], case["kv_heads"], case["kv_heads"])]
        first = torch.randint(0, max(1, case["ctx"] - n), (1,), generator=gen, device=DEV)
        pos = first + torch.arange(n, device=DEV) if n > 256 else torch.randint(0, case["ctx"], (n,), generator=gen, device=DEV)
        return dict(case=case, q=rows[0], k=rows[1], v=rows[2], pos=pos.int(), k_cache=k_cache, v_cache=v_cache,
                    steps=torch.tensor(steps, dtype=torch.int64, device=DEV), scale=scale,
                    slots=perm(pages * page)[:n].int())
    if op == "copy":
        k_cache, v_cache = _cache(gen, case, case["pages"])
        order = perm(case["pages"]).int()
        return dict(case=case, k_cache=k_cache, v_cache=v_cache, src=order[:case["copies"]].contiguous(),
                    dst=order[case["copies"]:2 * case["copies"]].contiguous(),
                    tokens=torch.randint(1, page + 1, (case["copies"],), generator=gen, device=DEV).int())
    if op == "compact":
        k_cache, v_cache = _cache(gen, case, case["pages"])
        seqs, held = case["seqs"], case["held"]
        # Every sequence but the first has the first one's first two pages (a prompt that they share) before its own.
        table = perm(case["pages"])[:seqs * held].view(seqs, held).int()
        if held > 2:
            table[1:, :2] = table[0, :2]
        lens = torch.randint((held - 1) * page + 1, held * page + 1, (seqs,), generator=gen, device=DEV).int()
        return dict(case=case, k_cache=k_cache, v_cache=v_cache, table=table, lens=lens)
    lens, new = _lengths(case)
    width = -(-max(lens) // page)
    used = sum(-(-n // page) for n in lens)
    k_cache, v_cache = _cache(gen, case, used + 2)
    order, at = perm(used + 2).int(), 0
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
    for i, n in enumerate(lens):
        m = -(-n // page)
        table[i, :m] = order[at:at + m]
        at += m
    starts = [0]
    for m in new:
        starts.append(starts[-1] + m)
    return dict(case=case, q=_normal(gen, starts[-1], case["heads"], case["dim"]), k_cache=k_cache, v_cache=v_cache,
                table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), most=max(new),
                starts=torch.tensor(starts, dtype=torch.int32, device=DEV))


# ---------------------------------------------------------------- the plain form


def _rotate(x, cos, sin, rot, layout):
    """x f32 [tokens, heads, dim], cos / sin [tokens, 1, rot / 2]."""
    y = x.clone()
    if layout == "half":
        a, b = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        a, b = slice(0, rot, 2), slice(1, rot, 2)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _plain_rope(s):
    case = s["case"]
    phase = s["pos"].long()[:, None] * s["steps"]  # turns in units of 2^-64, whole turns dropped by the wrap
    angle = (phase.float() * (2.0 * math.pi * 2.0 ** -64))[:, None, :]
    cos, sin = angle.cos() * s["scale"], angle.sin() * s["scale"]
    q = _rotate(s["q"], cos, sin, case["rot"], case["layout"])
    k = _rotate(s["k"], cos, sin, case["rot"], case["layout"])
    slots = s["slots"].long()
    at, off = slots // case["page"], slots % case["page"]
    s["k_cache"][at, :, off] = k.to(s["k_cache"].dtype)
    s["v_cache"][at, :, off] = s["v"].to(s["v_cache"].dtype)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s, window, sinks):
    q, table, lens, starts, most = s["q"], s["table"].long(), s["lens"].long(), s["starts"].long(), s["most"]
    (total, heads, dim), (n, width) = q.shape, table.shape
    kv_heads, page = s["k_cache"].shape[1:3]
    span = width * page
    gather = lambda c: c[table.clamp(min=0)].float().transpose(1, 2).reshape(n, kv_heads, span, dim)  # noqa: E731
    k, v = gather(s["k_cache"]), gather(s["v_cache"])
    new = starts[1:] - starts[:-1]
    i = torch.arange(most, device=q.device)
    at = torch.where(i < new[:, None], starts[:-1, None] + i, total)  # [n, most], past a sequence's end the spare row
    rows = torch.cat([q, q.new_zeros(1, heads, dim)])[at].view(n, most, kv_heads, heads // kv_heads, dim)
    rows = rows.permute(0, 2, 3, 1, 4).reshape(n, kv_heads, -1, dim)
    p = torch.matmul(rows, k.transpose(2, 3)).mul_(dim ** -0.5).view(n, kv_heads, -1, most, span)
    pos = ((lens - new)[:, None] + i)[:, :, None]
    j = torch.arange(span, device=q.device)
    seen = (j <= pos) & (j < lens[:, None, None])
    if window:
        seen &= (pos - j < window) | (j < sinks)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True).clamp(min=-1e30)
    p = p.sub_(top).exp_()
    o = torch.matmul(p.view(n, kv_heads, -1, span), v) / p.sum(-1).view(n, kv_heads, -1, 1).clamp(min=1e-30)
    o = o.view(n, kv_heads, -1, most, dim).permute(0, 3, 1, 2, 4).reshape(n, most, heads, dim)
    out = q.new_empty(total + 1, heads, dim)
    out[at] = o
    return out[:total]


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    filled = (torch.arange(s["case"]["page"], device=src.device) < s["tokens"][:, None])[:, None, :, None]
    for c in (s["k_cache"], s["v_cache"]):
        c[dst] = torch.where(filled, c[src], c[dst])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_compact(s):
    """The k-th page in use at or above their count moves into the k-th unused page below it."""
    table, pages = s["table"].long(), s["case"]["pages"]
    i = torch.arange(table.shape[1], device=table.device)
    valid = (i * s["case"]["page"] < s["lens"][:, None]) & (table >= 0) & (table < pages)
    used = torch.zeros(pages + 1, dtype=torch.bool, device=table.device)
    used[torch.where(valid, table, pages)] = True
    used = used[:pages]
    live = used.sum()
    number = torch.arange(pages, device=table.device)
    src, dst = (used & (number >= live)).nonzero()[:, 0], (~used & (number < live)).nonzero()[:, 0]
    to = number.clone()
    to[src] = dst
    for c in (s["k_cache"], s["v_cache"]):
        c[dst] = c[src]
    new = torch.where(valid, to[table.clamp(0, pages - 1)], -1).int()
    return {"table": new, "live": live.int().view(1), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


# ---------------------------------------------------------------- the framework's operators


def _framework():
    path = os.path.join(os.getcwd(), "llama.zig_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ggml_hip
    return ggml_hip


def _own(s):
    G, case = _framework(), s["case"]
    op = case["op"]
    if "kv" not in s:
        s["kv"] = G.PagedKV(s["k_cache"], s["v_cache"])  # the cache's handle, which a program keeps
    kv = s["kv"]
    caches = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "rope":
        return dict(caches, q=G.rope_kv_store(s["q"], s["k"], s["v"], s["pos"], s["steps"], kv, s["slots"],
                                              layout=case["layout"], mscale=s["scale"]))
    if op == "copy":
        G.copy_pages(kv, s["src"], s["dst"], s["tokens"])
        return caches
    if op == "compact":
        table, live = G.compact_pages(kv, s["table"], s["lens"])
        return dict(caches, table=table, live=live)
    return G.attn_paged(s["q"], kv, s["table"], s["lens"], q_starts=None if op == "step" else s["starts"],
                        max_q=s["most"], max_kv=case["kv"], window=case["window"], sinks=case["sinks"])


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "rope":
        return _plain_rope(state)
    if case["op"] == "copy":
        return _plain_copy(state)
    if case["op"] == "compact":
        return _plain_compact(state)
    return _plain_attention(state, case["window"], case["sinks"])


# ---------------------------------------------------------------- work and the definition in 64 bits


def _seen(p, window, sinks):
    """How many keys a token at position p sees."""
    if not window or p + 1 <= window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(case):
    op, size = case["op"], 2 * case["kv_heads"] * case["dim"]  # cache bytes of one token's keys, or values
    if op == "rope":
        n = case["tokens"]
        return {"bytes": n * (4 * case["dim"] * (2 * case["heads"] + 2 * case["kv_heads"]) + 2 * size + 8)
                + 8 * (case["rot"] // 2), "flops": n * (case["heads"] + case["kv_heads"]) * case["rot"] * 3}
    if op == "copy":
        return {"bytes": case["copies"] * ((case["page"] + 1) * 2 * size + 12), "flops": 0}  # half a page on the mean, both
    if op == "compact":
        live = case["seqs"] * case["held"] - (2 * (case["seqs"] - 1) if case["held"] > 2 else 0)
        moved = live * (case["pages"] - live) / case["pages"]  # on the mean
        return {"bytes": int(moved * 4 * size * case["page"]) + 8 * case["seqs"] * case["held"], "flops": 0}
    read = pairs = tokens = 0
    for n, m in zip(*_lengths(case)):
        first = n - m
        pairs += sum(_seen(p, case["window"], case["sinks"]) for p in range(first, n))
        low = max(0, first - case["window"] + 1) if case["window"] else 0
        read += n - low + min(low, case["sinks"])
        tokens += m
    return {"bytes": read * 2 * size + 8 * tokens * case["heads"] * case["dim"],
            "flops": 4 * pairs * case["heads"] * case["dim"]}


def exact(case, seed):
    if case["op"] in ("copy", "compact"):
        return None
    s = prepare(case, seed)
    k_cache, v_cache, page = s["k_cache"].double(), s["v_cache"].double(), case["page"]
    if case["op"] == "rope":
        rot, half = case["rot"], case["rot"] // 2
        # The turns of each position in whole numbers, by Python, then in f64.
        turns = [[(p * f) % 2 ** 64 / 2.0 ** 64 for f in s["steps"].tolist()] for p in s["pos"].tolist()]
        z = torch.polar(torch.full((1,), s["scale"], dtype=torch.float64, device=DEV),
                        torch.tensor(turns, dtype=torch.float64, device=DEV) * (2 * math.pi))[:, None]
        outs = []
        for x in (s["q"].double(), s["k"].double()):
            r = x[..., :rot]
            if case["layout"] == "half":
                w = torch.complex(r[..., :half].contiguous(), r[..., half:].contiguous()) * z
                r = torch.cat([w.real, w.imag], -1)
            else:
                w = torch.view_as_complex(r.reshape(*r.shape[:2], half, 2).contiguous()) * z
                r = torch.view_as_real(w).flatten(2)
            outs.append(torch.cat([r, x[..., rot:]], -1))
        where = s["slots"].long()
        for c, x in ((k_cache, outs[1]), (v_cache, s["v"].double())):
            c[where // page, :, where % page] = x
        return {"q": outs[0], "k_cache": k_cache, "v_cache": v_cache}
    group = case["heads"] // case["kv_heads"]
    starts, out = s["starts"].tolist(), torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lens"].tolist()):
        rows = s["q"][starts[i]:starts[i + 1]].double()
        where = s["table"][i, :-(-n // page)].long()
        key = torch.arange(n, device=DEV)
        mine = torch.arange(n - rows.shape[0], n, device=DEV)[:, None]
        hidden = key > mine
        if case["window"]:
            hidden = hidden | ((mine - key >= case["window"]) & (key >= case["sinks"]))
        for h in range(case["kv_heads"]):
            k, v = (c[where, h].reshape(-1, case["dim"])[:n] for c in (k_cache, v_cache))
            for g in range(h * group, (h + 1) * group):
                score = (rows[:, g] @ k.T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
                out[starts[i]:starts[i + 1], g] = torch.softmax(score, -1) @ v
    return out
