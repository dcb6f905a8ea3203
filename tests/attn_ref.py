"""Plain f64 evaluations of the operators of include/ggml_hip_attn.h, and the
inputs their tests share.  Torch tensors on any device; results f64."""
import math

import torch

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def rope(x, pos, freqs, layout, mscale=1.0):
    """freqs f64 [n_dims / 2], radians per position."""
    x = x.double().clone()
    n = freqs.numel()
    angle = pos.double()[:, None, None] * freqs.to(x.device)
    c, s = torch.cos(angle) * mscale, torch.sin(angle) * mscale
    a, b = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    xa, xb = x[..., a].clone(), x[..., b].clone()
    x[..., a] = xa * c - xb * s
    x[..., b] = xa * s + xb * c
    return x


def rows_of(cache, table_row, n):
    """Tokens 0..n-1 of a sequence, [n, n_kv_heads, head_dim], and which of them lie in the pool."""
    page = cache.shape[2]
    j = torch.arange(n, device=cache.device)
    e = table_row.long()[j // page]
    ok = (e >= 0) & (e < cache.shape[0])
    return cache[e.clamp(0, cache.shape[0] - 1), :, j % page], ok


def seen(m, n, ok, window, sinks):
    """[m, n]: what the queries at positions n - m .. n - 1 see."""
    p = torch.arange(n - m, n, device=ok.device)[:, None]
    j = torch.arange(n, device=ok.device)[None]
    see = (j <= p) & ok
    if window:
        see &= (p - j < window) | (j < sinks)
    return see


def attention(q, k, v, table, lens, starts, scale, window=0, sinks=0):
    """f64 [n_tokens, heads, dim], and the largest |score| among what is seen."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    top = 0.0
    group = q.shape[1] // k.shape[1]
    most = table.shape[1] * k.shape[2]
    for s, n in enumerate(lens.tolist()):
        n = min(max(n, 0), most)
        lo, hi = int(starts[s]), int(starts[s + 1])
        m = hi - lo
        if m == 0 or n == 0:
            continue
        ks, ok = rows_of(k, table[s], n)
        vs, _ = rows_of(v, table[s], n)
        see = seen(m, n, ok, window, sinks)
        for h in range(q.shape[1]):
            kh, vh = ks[:, h // group].double(), vs[:, h // group].double()
            sc = q[lo:hi, h].double() @ torch.where(ok[:, None] & torch.isfinite(kh), kh, 0.0).T * scale
            bad = ~torch.isfinite(kh).all(1)
            sc = sc.masked_fill(~see, -math.inf)
            if (see & bad).any():
                sc = torch.where(see & bad, math.nan, sc)
            mx = sc.amax(1, keepdim=True)
            w = torch.exp(sc - torch.where(mx == -math.inf, 0.0, mx))
            w = torch.where(see, w, 0.0)
            total = w.sum(1, keepdim=True)
            # what is not seen does not matter, whatever it holds
            fin = torch.where(torch.isfinite(vh), vh, 0.0)
            o = w @ fin
            for j in (~torch.isfinite(vh).all(1)).nonzero()[:, 0].tolist():
                add = torch.where(see[:, j:j + 1] & ~torch.isfinite(vh[j]), w[:, j:j + 1] * vh[j], 0.0)
                o = o + add
            out[lo:hi, h] = torch.where(total == 0, torch.zeros_like(o), o / total)
            fs = sc[torch.isfinite(sc)]
            if fs.numel():
                top = max(top, float(fs.abs().max()))
    return out, top


def tolerance(dim, top):
    """Relative 2-norm bound of an f32 evaluation: a score is a sum of dim
    products, each addition rounded to 2^-24 of partial sums of about the
    largest score, with random signs; softmax hands the scores' errors on at most twofold, and
    exp2, the two sums, the parts of q and w and the quotient add a few 2^-24."""
    return math.sqrt(dim) * 2.0 ** -24 * (4 + 2 * top)


def make_cache(gen, dtype, n_pages, kv_heads, page, dim, device="cuda", order="heads"):
    shape = (n_pages, kv_heads, page, dim) if order == "heads" else (n_pages, page, kv_heads, dim)
    c = [torch.randn(shape, generator=gen, device=device).to(dtype) for _ in range(2)]
    return c if order == "heads" else [x.transpose(1, 2) for x in c]


def make_table(gen, lens, page, device="cuda", spare=2, width=None):
    """Scattered pages for each sequence, -1 past its last one; (table, pages in the pool)."""
    need = [-(-max(n, 0) // page) for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=gen, device=device).int()
    width = max(need + [1]) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=device)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = order[at:at + m]
        at += m
    return table, pool


def starts_of(new, device="cuda"):
    out = [0]
    for m in new:
        out.append(out[-1] + m)
    return torch.tensor(out, dtype=torch.int32, device=device)
