"""Plain 64-bit restatements of decoding in 4 bits and of beam search's choice, for the tests of the HIP operators."""
import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def fours(x):
    """(codes, scales) of x (.., K), K a multiple of 32: the scale is bf16 of an fp32 product, the quotient fp32."""
    g = x.float().cpu().unflatten(-1, (-1, 32))
    a = g.abs().amax(-1)
    s = (a * torch.tensor(1 / 6, dtype=torch.float32)).bfloat16()
    s = torch.where(s.float() < 2.0 ** -126, torch.zeros_like(s), s)
    s = torch.where(torch.isfinite(a), s, torch.full_like(s, math.nan))
    wide = s.float().unsqueeze(-1)
    t = torch.where(wide > 0, g.abs() / torch.where(wide > 0, wide, torch.ones_like(wide)), torch.zeros_like(g)).double()
    gap = (t.clamp(max=6.0).unsqueeze(-1) - LEVELS).abs()
    near = gap == gap.amin(-1, keepdim=True)
    # of two as near the even one
    code = torch.where(near.sum(-1) > 1, (near * (torch.arange(8) % 2 == 0)).int().argmax(-1), near.int().argmax(-1))
    code = code + 8 * ((g < 0) & (code > 0))
    return code.flatten(-2).to(torch.uint8), s


def values(codes, scales):
    c = codes.long()
    v = torch.where(c >= 8, -1.0, 1.0).double() * LEVELS[c & 7]
    return (v.unflatten(-1, (-1, 32)) * scales.double().unsqueeze(-1)).flatten(-2)


def weight_values(data, n, k):
    """(n, k) fp64 of one packed weight, byte by byte."""
    data = data.cpu()
    tiles, blocks, _ = data.shape
    codes = torch.zeros((16 * tiles, 128 * blocks), dtype=torch.uint8)
    scales = torch.zeros((16 * tiles, 4 * blocks), dtype=torch.bfloat16)
    for r in range(16):
        for h in range(4):
            for g in range(4):
                for j in range(8):
                    byte = data[:, :, (16 * h + r) * 16 + 4 * g + j // 2]
                    codes[r::16, 32 * g + 8 * h + j::128] = (byte >> (4 * (j % 2))) & 15
        for g in range(4):
            at = 1024 + 2 * (4 * r + g)
            scales[r::16, g::4] = data[:, :, at:at + 2].contiguous().view(torch.bfloat16)[..., 0]
    return values(codes, scales)[:n, :k]


def cache_parts(cache, hd):
    """Codes (2, .., blocks, 32, hd) and scales (2, .., blocks, 32, hd / 32) of keys and values of packed blocks (.., bytes)."""
    cache = cache.cpu()
    lead = cache.shape[:-1]
    codes = torch.zeros((2, *lead, 32, hd), dtype=torch.uint8)
    scales = torch.zeros((2, *lead, 32, hd // 32), dtype=torch.bfloat16)
    for slot in range(32):
        t, low, i = slot // 16, slot % 16, slot % 4
        h = low // 4
        for e in range(hd):
            w, lane, j = t * (hd // 32) + e // 32, (e % 32) // 8 * 16 + low, e % 8
            codes[0, ..., slot, e] = cache[..., 1024 * (w // 4) + 16 * lane + 4 * (w % 4) + j // 2] >> (4 * (j % 2)) & 15
            w, lane, j = e // 16, 16 * h + e % 16, 4 * t + i
            at = 16 * hd + 1024 * (w // 4) + 16 * lane + 4 * (w % 4) + j // 2
            codes[1, ..., slot, e] = cache[..., at] >> (4 * (j % 2)) & 15
        for part in range(2):
            for g in range(hd // 32):
                at = 32 * hd + 2 * hd * part + 64 * g + 16 * h + 2 * (4 * t + i)
                scales[part, ..., slot, g] = cache[..., at:at + 2].contiguous().view(torch.bfloat16)[..., 0]
    return codes, scales


def cache_values(cache, hd):
    """Keys and values (.., blocks 32, hd) fp64."""
    k, v = (values(c, s).flatten(-3, -2) for c, s in zip(*cache_parts(cache, hd)))
    return k, v


def place(p, window, sinks):
    """The slot of position p, over all blocks."""
    return p if p < sinks else -(-sinks // 32) * 32 + (p - sinks) % window


def rotate(x, cos, sin):
    lo, hi = x.chunk(2, -1)
    return x * cos + torch.cat([-hi, lo], -1) * sin


def paths(parents, count):
    """Each node's path from the context, itself last; None where a parent is none."""
    line = []
    for i in range(count):
        up = int(parents[i])
        if not -1 <= up < i:
            return None
        line.append((line[up] if up >= 0 else []) + [i])
    return line


def tree(q, k_nodes, v_nodes, keys, vals, pos, window, sinks, parents, count):
    """One request: (out (T, H, hd), magnitudes (T, H, hd), widest score error factor (T, H)) in 64 bits; q rotated already,
    keys / vals (Hkv, slots, hd) the cache's, k_nodes / v_nodes (T, Hkv, hd)."""
    t, heads, hd = q.shape
    hkv = keys.shape[0]
    line = paths(parents, count)
    out, size, score_size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(t, heads, dtype=torch.float64)
    for i in range(count):
        at = pos + len(line[i]) - 1
        old = [j for j in range(max(0, pos - window - sinks), pos) if at - j < window] + list(range(min(sinks, pos)))
        old = sorted(set(old))
        slots = [place(j, window, sinks) for j in old]
        mine = [j for x, j in enumerate(line[i]) if at - (pos + x) < window or pos + x < sinks]
        for h in range(heads):
            g = h * hkv // heads
            kk = torch.cat([keys[g, slots], k_nodes[mine, g]])
            vv = torch.cat([vals[g, slots], v_nodes[mine, g]])
            s = kk @ q[i, h] / math.sqrt(hd)
            w = torch.softmax(s, 0)
            out[i, h], size[i, h] = w @ vv, w @ vv.abs()
            score_size[i, h] = (kk.abs() @ q[i, h].abs()).max() / math.sqrt(hd)
    return out, size, score_size


def beams(logits, scores, n, ended, banned, limit, eos, pad):
    """(tokens, sources, scores, ended) of every group in 64 bits."""
    rows, vocab = logits.shape
    tokens, sources, best, over = [], [], [], []
    for r in range(0, rows, n):
        found = []
        for b in range(r, r + n):
            score = float(scores[b])
            if not math.isfinite(score):
                continue
            if ended is not None and int(ended[b]):
                found.append((-score, b, pad, True))
                continue
            x = logits[b].double().clone()
            if limit is not None:
                x[limit:] = -math.inf
            for i in banned:
                if i < vocab:
                    x[i] = -math.inf
            if torch.isnan(x).any() or not math.isfinite(float(x.max())):
                continue
            top = float(x.max())
            norm = math.log(float(torch.exp(x - top).sum()))
            order = torch.sort(x, descending=True, stable=True).indices[:n].tolist()
            found += [(-(score + ((float(x[i]) - top) - norm)), b, i, False) for i in order if float(x[i]) > -math.inf]
        found.sort(key=lambda c: c[:3])
        for k in range(n):
            if k < len(found):
                value, b, token, was = found[k]
                tokens.append(token), sources.append(b), best.append(-value), over.append(int(was or token == eos))
            else:
                tokens.append(pad), sources.append(r + k), best.append(-math.inf), over.append(1)
    return torch.tensor(tokens), torch.tensor(sources), torch.tensor(best, dtype=torch.float64), torch.tensor(over)
