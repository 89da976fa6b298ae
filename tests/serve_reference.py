"""Plain 64-bit forms of the serving operators, for their tests: written from the definitions, on the CPU."""
import math

import torch


def slot_of(p, sinks, window):
    return p if p < sinks else sinks + (p - sinks) % window


def softmax_attend(q, k, v, seen):
    """(t, hd) x (keys, hd) in 64 bits with ``seen`` (t, keys): output, sum of weight * |value|, and the largest
    sum of |q k| / sqrt(hd) (what a relative error of the products weighs)."""
    q, k, v = q.double(), k.double(), v.double()
    k = torch.where(seen.any(0)[:, None], k, 0.0)
    v = torch.where(seen.any(0)[:, None], v, 0.0)
    s = (q @ k.T / math.sqrt(q.shape[1])).masked_fill(~seen, -math.inf)
    w = torch.softmax(s, 1)
    return w @ v, w @ v.abs(), float((q.abs() @ k.abs().T).max()) / math.sqrt(q.shape[1])


def attend_bound(out, weighted, products, dtype, hd, keys, q_terms=True):
    """How far an output may be: the roundings of the weights (bf16 operands of the second product) and of the output,
    each half a step; the scores' errors (q in one or two bf16 terms, or fp32 products of hd terms); fp32 sums."""
    u = 2.0 ** -24
    if dtype == torch.bfloat16:
        score = ((2.0 ** -17 if q_terms else 2.0 ** -8) + hd * u) * products
        return (2.0 ** -8 + 2 * score + keys * u + 2.0 ** -20) * weighted + 2.0 ** -8 * out.abs() + 1e-30
    score = (hd + 8) * u * products
    return (2 * score + (keys + hd) * u + 2.0 ** -20) * weighted + 1e-30


def rotate(x, cos, sin):
    half = x.shape[-1] // 2
    lo, hi = x[..., :half].double(), x[..., half:].double()
    c, s = cos[..., :half].double(), sin[..., :half].double()
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def tables(n, hd, theta=10000.0):
    f = theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.outer(torch.arange(n, dtype=torch.float64), f)
    return torch.cat([a.cos()] * 2, 1).float(), torch.cat([a.sin()] * 2, 1).float()


def tree_paths(parents):
    paths = []
    for i, up in enumerate(parents):
        paths.append((paths[up] if up >= 0 else []) + [i])
    return paths


def tree_attend(q, k_nodes, v_nodes, k_ring, v_ring, pos, parents, window, sinks):
    """One request: q (t, H, hd) rotated, k_nodes rotated, rings (Hkv, slots, hd), the tree's parents.  Returns out,
    weighted |values| and products as ``softmax_attend`` does, per node and head."""
    t, heads, _ = q.shape
    hkv = k_ring.shape[0]
    rep = heads // hkv
    paths = tree_paths(parents)
    old = [j for j in range(max(0, pos - window) if sinks == 0 else 0, pos) if j < sinks or j >= pos - window]
    slots = [slot_of(j, sinks, window) for j in old]
    seen = torch.zeros((t, len(old) + t), dtype=torch.bool)
    for i in range(t):
        at = pos + len(paths[i]) - 1
        for x, j in enumerate(old):
            seen[i, x] = j < sinks or at - j < window
        for a in paths[i]:
            there = pos + len(paths[a]) - 1
            seen[i, len(old) + a] = there < sinks or at - there < window
    out, weighted = torch.empty(q.shape, dtype=torch.float64), torch.empty(q.shape, dtype=torch.float64)
    products = 0.0
    for h in range(heads):
        g = h // rep
        k = torch.cat([k_ring[g, slots].double(), k_nodes[:, g].double()])
        v = torch.cat([v_ring[g, slots].double(), v_nodes[:, g].double()])
        out[:, h], weighted[:, h], pr = softmax_attend(q[:, h], k, v, seen)
        products = max(products, pr)
    return out, weighted, products


def sample_row(x, u, temperature, top_k=0, top_p=1.0, min_p=0.0, banned=(), limit=None):
    """(token, logprob, distance of u * total from the token's borders in units of the largest weight, kept) of one row."""
    x = x.double().clone()
    if limit is not None and limit < len(x):
        x[limit:] = -math.inf
    for b in banned:
        if b < len(x):
            x[b] = -math.inf
    if torch.isnan(x).any():
        return int(torch.isnan(x).nonzero()[0]), math.nan if temperature > 1e-5 else 0.0, math.inf, None
    best = int(torch.argmax(x))
    best = int((x == x[best]).nonzero()[0])
    if not temperature > 1e-5:
        return best, 0.0, math.inf, None
    if not math.isfinite(float(x[best])):
        return best, math.nan, math.inf, None
    order = sorted(range(len(x)), key=lambda i: (-float(x[i]), i)) if len(x) < 4096 else \
        torch.sort(x, descending=True, stable=True).indices.tolist()
    order = torch.tensor(order)
    w = torch.exp((x[order] - x[best]) / temperature)
    w = torch.where(x[order] == -math.inf, 0.0, w)
    keep = torch.ones(len(x), dtype=torch.bool)
    if top_k > 0:
        keep[top_k:] = False
    if min_p > 0:
        keep &= w >= min(min_p, 1.0)
    mass = torch.where(keep, w, 0.0)
    if top_p < 1:
        ahead = mass.cumsum(0) - mass
        keep &= ahead <= max(top_p, 0.0) * mass.sum()
        mass = torch.where(keep, w, 0.0)
    by_id = torch.zeros_like(w)
    by_id[order] = mass
    below = by_id.cumsum(0)
    total = float(below[-1])
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    token = int((below <= u * total).sum())
    near = min(abs(u * total - float(below[token])), abs(u * total - float(below[token] - by_id[token])))
    return token, math.log(float(by_id[token]) / total), near, by_id > 0
