"""Plain f64 forms of a mixture-of-experts layer's operators, on the CPU."""
import math

import numpy as np
import torch

U = 2.0 ** -24  # half a step of f32


def route(logits, k, gating="softmax", bias=None, groups=1, keep=1, top=2, renormalize=False, min_sum=2.0 ** -14,
          scale=1.0):
    """(ids, weights f64) from the definition, token by token."""
    logits = np.asarray(logits, np.float64)
    n, e = logits.shape
    b = np.zeros(e) if bias is None else np.asarray(bias, np.float64)
    ids, weights = np.full((n, k), -1, np.int32), np.zeros((n, k))
    size = e // groups
    first = lambda s: (0, 0.0) if math.isnan(s) else (1, -s)  # noqa: E731  NaN first, then descending
    with np.errstate(all="ignore"):
        for t in range(n):
            row = logits[t]
            hidden = (row == -np.inf) | (b == -np.inf)
            p = row.copy()
            if gating == "softmax":
                m = row.max()
                p = np.where(row == -np.inf, 0.0, np.exp(row - m)) if m > -np.inf else np.zeros(e)
                p = p / np.sum(p)
            elif gating == "sigmoid":
                p = 1 / (1 + np.exp(-row))
            score = row if bias is None else p + b
            seen = [x for x in range(e) if not hidden[x]]
            if groups > 1:
                def of_group(g):
                    mine = sorted((x for x in seen if x // size == g), key=lambda x: first(score[x]))[:top]
                    if not mine:
                        return -np.inf
                    if top == 1:
                        return score[mine[0]]
                    return sum(p[x] + b[x] for x in mine)
                s = [of_group(g) for g in range(groups)]
                kept = sorted(range(groups), key=lambda g: (*first(s[g]), g))[:keep]
                seen = [x for x in seen if x // size in kept]
            chosen = sorted(seen, key=lambda x: (*first(score[x]), x))[:k]
            if not chosen:
                continue
            w = p[chosen]
            if gating == "softmax_chosen":
                w = np.exp(row[chosen] - row[chosen].max())
                w = w / w.sum()
            if renormalize:
                w = w / max(w.sum(), float(np.float32(min_sum))) if w.sum() == w.sum() else w * np.nan
            ids[t, :len(chosen)] = chosen
            weights[t, :len(chosen)] = w * float(np.float32(scale))
    return ids, weights


def quantize(x):
    """(q int8, scale f32) of f32 rows, by the f32 product and divisions of the definition."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        most = np.abs(x).max(-1) if x.shape[-1] else np.zeros(x.shape[:-1], np.float32)
        d = (most * (np.float32(1) / np.float32(127))).astype(np.float32)
        fine = np.isfinite(most)
        q = np.where((fine & (d > 0))[..., None], np.clip(np.rint(x / d[..., None]), -127, 127), 0)
    return np.nan_to_num(q).astype(np.int8), np.where(fine, d, np.float32(np.nan)).astype(np.float32)


def product(w, w_scale, q, scale):
    """Exact sums, scaled in f64."""
    acc = torch.as_tensor(q).double() @ torch.as_tensor(w).double().T
    return (acc * torch.as_tensor(scale).double()[:, None] * torch.as_tensor(w_scale).double()).numpy()


def product_id(w, w_scale, q, scale, ids):
    n, k = ids.shape
    out = np.zeros((n, k, w.shape[1]))
    q, scale = np.broadcast_to(q, (n, k, q.shape[2])), np.broadcast_to(scale, (n, k))
    for e in range(w.shape[0]):
        t, s = np.nonzero(ids == e)
        if len(t):
            out[t, s] = product(w[e], w_scale[e], np.ascontiguousarray(q[t, s]), np.ascontiguousarray(scale[t, s]))
    return out


def combine(y, weights, ids=None, add=None):
    """(the sum, the sum of magnitudes)."""
    y, w = np.asarray(y, np.float64), np.asarray(weights, np.float64)[..., None]
    terms = y * w
    if ids is not None:
        terms = np.where((np.asarray(ids) < 0)[..., None], 0.0, terms)
    base = np.zeros(y[:, 0].shape if y.shape[1] else (y.shape[0], y.shape[2])) if add is None else np.asarray(add, np.float64)
    return base + terms.sum(1), np.abs(base) + np.abs(terms).sum(1)
