"""Decoding in 4 bits and beam search, in plain form and as the framework's calls, for timing and comparing.

* ``linear``   products of a step's rows with weights in 4 bits (slow projections, LM head), optionally the input's RMSNorm
               and a residual;
* ``readout``  the fast-weight readout of every request through its own weights in 4 bits;
* ``attend``   attention of new tokens (one, or a tree of drafted ones) over ring caches in 4 bits with sink slots;
* ``commit``   accepted tokens' keys and values into such caches, all layers at once;
* ``beam``     the best continuations of every group of beams, for ``kv_fork`` to reorder the caches by.

With ``own`` false ``run`` computes them with elementary torch operations; with ``own`` true it calls the framework.

Four bits: 32 neighbours along the contracted axis (a head's elements in caches) share the scale
s = bf16(largest magnitude * fp32(1 / 6)), 0 where that is below 2^-126; a value is the level of ``LEVELS`` next to x / s (the
quotient in fp32, ties to the even code), its sign in bit 3.  Layouts:

* weights (n, k), padded with zeros to whole blocks of 16 rows and 128 columns: per block 64 x 16 bytes of codes and 16 x 4
  scales.  Piece 16 h + r of the codes holds, for the groups g = 0..3, eight codes (the first in the lowest bits) of row r,
  columns 32 g + 8 h ..; the scales lie row by row.
* caches: per request, head and 32 slots (the sinks' blocks first, then the window's) keys, values and both
  scales.  With word (t, g) of lane 16 h + r for keys: slot 16 t + r, elements 32 g + 8 h ..; word t of lane 16 h + r for
  values: element 16 t + r of the slots 4 h .. 4 h + 3, 16 + 4 h .. 16 + 4 h + 3; words w, w + 1, .. of four lie beside each
  other, 1024 bytes apart from the next four; scales per group in the slots' order of the values.
"""
from __future__ import annotations

import math

import torch

own = False

BANNED = (0, 1, 3)  # padding, begin of text, unknown
EOS, PAD = 2, 0
THETA = 10000.0
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one user's packed query / key / value projection in the small model: latency
        dict(name="linear_1x1280x768", kind="linear", rows=1, n=1280, k=768, norm=True, residual=False, dtype="bf16"),
        # the LM head of a full batch in the large model
        dict(name="linear_32x32000x2048", kind="linear", rows=32, n=32000, k=2048, norm=True, residual=False, dtype="bf16"),
        # sizes that fill no tile, an output projection onto its residual in research precision
        dict(name="linear_61x1999x5501_fp32", kind="linear", rows=61, n=1999, k=5501, norm=False, residual=True,
             dtype="fp32"),
        # one user's readout in the small model: latency
        dict(name="readout_1x768x2048", kind="readout", rows=1, tokens=1, d=768, ff=2048, norm=True, dtype="bf16"),
        # a full batch, every request with fast weights of its own: what a decode step is bound by
        dict(name="readout_32x768x2048", kind="readout", rows=32, tokens=1, d=768, ff=2048, norm=True, dtype="bf16"),
        # one user, one token: latency
        dict(name="attend_1x512", kind="attend", rows=1, nodes=1, heads=12, kv_heads=4, hd=64, window=512, sinks=4,
             longest=3000, dtype="bf16"),
        # batched serving over long windows, ragged contexts from short to wrapped
        dict(name="attend_32x4096", kind="attend", rows=32, nodes=1, heads=16, kv_heads=4, hd=128, window=4096, sinks=4,
             longest=12000, dtype="bf16"),
        # trees of drafted tokens over an odd window, research precision
        dict(name="attend_7x24_fp32", kind="attend", rows=7, nodes=24, heads=12, kv_heads=4, hd=64, window=1001, sinks=33,
             longest=2500, dtype="fp32"),
        # one user's step: a token into twelve layers' caches
        dict(name="commit_1x1", kind="commit", layers=12, rows=1, nodes=1, kv_heads=4, hd=64, window=512, sinks=4,
             longest=3000, dtype="bf16"),
        # prompts as long as the window into fresh caches
        dict(name="commit_4x1024", kind="commit", layers=6, rows=4, nodes=1024, kv_heads=4, hd=128, window=1024, sinks=4,
             longest=2000, dtype="bf16"),
        # four beams of one user
        dict(name="beam_1x4x32000", kind="beam", groups=1, beams=4, vocab=32000, limit=21478, ended=False, dtype="bf16"),
        # many users' beams over a large vocabulary, some of them ended
        dict(name="beam_16x16x131072", kind="beam", groups=16, beams=16, vocab=131072, limit=131072, ended=True,
             dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges."""
    kind = rng.choice(["linear", "linear", "readout", "attend", "attend", "commit", "beam"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "linear":
        rows, k, n = _log(rng, 1, 100), _log(rng, 64, 6000), _log(rng, 64, 32000)
        n = min(n, 2048 * 32000 // k)
        if rng.random() < 0.5:
            n, k = -(-n // 32) * 32, -(-k // 64) * 64
        return dict(kind=kind, rows=rows, n=n, k=k, norm=rng.random() < 0.5, residual=rng.random() < 0.5, dtype=dtype)
    if kind == "readout":
        d, ff = rng.choice([256, 512, 768, 1024, 2048]), 64 * _log(rng, 4, 86)
        rows = min(_log(rng, 1, 32), max(1, 32 * 768 * 2048 // (d * ff)))
        return dict(kind=kind, rows=rows, tokens=rng.choice([1, 1, rng.randint(2, 16)]), d=d, ff=ff,
                    norm=rng.random() < 0.5, dtype=dtype)
    if kind == "beam":
        beams = rng.choice([1, 2, 4, 4, 8, 16, rng.randint(1, 32)])
        vocab = _log(rng, 256, 131072)
        return dict(kind=kind, groups=min(_log(rng, 1, 16), 256 // beams), beams=beams, vocab=vocab,
                    limit=rng.choice([vocab, vocab - rng.randint(1, vocab // 3)]), ended=rng.random() < 0.5, dtype=dtype)
    hd = rng.choice([64, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 4])
    sinks = rng.choice([0, 1, 4, rng.randint(2, 64)])
    window = rng.choice([512, 1024, _log(rng, 64, 4096)])
    longest = _log(rng, 16, 3 * window)
    if kind == "attend":
        return dict(kind=kind, rows=_log(rng, 1, 32), nodes=rng.choice([1, 1, rng.randint(2, 16), rng.randint(17, 64)]),
                    heads=min(16, kv_heads * rng.choice([1, 2, 3, 4, 8])), kv_heads=kv_heads, hd=hd, window=window,
                    sinks=sinks, longest=longest, dtype=dtype)
    window = min(window, 1024)
    rows, nodes = _log(rng, 1, 8), rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 1024)])
    return dict(kind=kind, layers=max(1, min(rng.choice([1, 6, 12]), 24 // rows)), rows=rows, nodes=nodes,
                kv_heads=kv_heads, hd=hd, window=window, sinks=sinks, longest=min(longest, 3000), dtype=dtype)


# ------------------------------------------------------------------------------------------------
# what a program has in hand
# ------------------------------------------------------------------------------------------------

def _dtype(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.bfloat16


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _quantise(x):
    """Codes (.., K) uint8 and scales (.., K / 32) bf16 of fp32 x (.., K)."""
    groups = x.float().unflatten(-1, (-1, 32))
    largest = groups.abs().amax(-1)
    scale = (largest * torch.tensor(1.0 / 6.0, dtype=torch.float32, device=x.device)).bfloat16()
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    wide = scale.float()[..., None]
    t = torch.where(wide > 0, groups.abs() / torch.where(wide > 0, wide, 1.0), 0.0)
    code = (t > 0.25).to(torch.uint8)
    code += t >= 0.75
    code += t > 1.25
    code += t >= 1.75
    code += t > 2.5
    code += t >= 3.5
    code += t > 5.0
    code += ((groups < 0) & (code > 0)).to(torch.uint8) * 8
    return code.flatten(-2), scale


def _nibbles(codes):
    """(.., 8) codes as (.., 4) bytes."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _pack_weight(w):
    """(.., n, k) as bytes (.., n / 16, k / 128, 1152)."""
    n, k = w.shape[-2:]
    w = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 16))
    codes, scales = _quantise(w)
    lead = w.dim() - 2
    at = lambda *d: [*range(lead), *(lead + i for i in d)]  # noqa: E731
    codes = codes.unflatten(-1, (-1, 4, 4, 8)).unflatten(lead, (-1, 16))  # tile, r, block, g, h, j
    codes = _nibbles(codes.permute(at(0, 2, 4, 1, 3, 5))).flatten(-4)
    scales = scales.unflatten(-1, (-1, 4)).unflatten(lead, (-1, 16)).permute(at(0, 2, 1, 3)).flatten(-2)
    return torch.cat([codes, scales.contiguous().view(torch.uint8)], dim=-1)


def _pack_cache(k_codes, k_scales, v_codes, v_scales):
    """(.., blocks, 32, hd) codes and (.., blocks, 32, hd / 32) scales as bytes (.., blocks, 36 hd)."""
    lead = k_codes.dim() - 2
    at = lambda *d: [*range(lead), *(lead + i for i in d)]  # noqa: E731
    words = k_codes.shape[-1] // 16

    def lanes(c):  # (.., words, h, r, j) to bytes, four words of a lane together
        return _nibbles(c.unflatten(lead, (words // 4, 4)).permute(at(0, 2, 3, 1, 4))).flatten(lead)

    k = k_codes.unflatten(-1, (-1, 4, 8)).unflatten(lead, (2, 16))  # t, r, g, h, j
    k = lanes(k.permute(at(0, 2, 3, 1, 4)).flatten(lead, lead + 1))
    v = v_codes.unflatten(-1, (-1, 16)).unflatten(lead, (2, 4, 4))  # t, h, i, word, r
    v = lanes(v.permute(at(3, 1, 4, 0, 2)).flatten(-2))
    scales = [s.unflatten(lead, (2, 4, 4)).permute(at(3, 1, 0, 2)).flatten(lead).contiguous().view(torch.uint8)
              for s in (k_scales, v_scales)]
    return torch.cat([k, v, *scales], dim=-1)


def _blocks(case):
    return -(-case["sinks"] // 32) + -(-case["window"] // 32)


def _cache(g, case, *lead):
    """A cache that earlier tokens filled, packed."""
    hd, parts = case["hd"], []
    for _ in range(2):
        parts += _quantise(_normal(g, torch.bfloat16, *lead, case["kv_heads"], _blocks(case), 32, hd).float())
    return _pack_cache(*parts)


def _positions(g, case, at_least=1):
    """Ragged contexts: lengths spread over [at_least, longest], the longest among them."""
    n = torch.randint(at_least, case["longest"] + 1, (case["rows"],), generator=g, device="cuda", dtype=torch.int64)
    n[0] = case["longest"]
    return n


def _tables(positions, hd):
    """RoPE tables of a program: fp32 cos and sin for every position, both halves of the head alike."""
    freq = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device="cuda"), freq)
    return torch.cat([angle.cos()] * 2, dim=1).float(), torch.cat([angle.sin()] * 2, dim=1).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    dt, f32 = _dtype(case), torch.float32
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        s["x"] = _normal(g, dt, m, k)
        s["w"] = _pack_weight(_normal(g, f32, n, k) / k ** 0.5)
        s["r"] = _normal(g, dt, m, n) if case["residual"] else None
        return s
    if case["kind"] == "readout":
        b, d, ff = case["rows"], case["d"], case["ff"]
        s["x"] = _normal(g, dt, b, case["tokens"], d)
        s["gain"] = (1.0 + 0.1 * _normal(g, f32, d)).to(dt) if case["norm"] else None
        # rows of the products: (B, ff, d) up and gate, (B, d, ff) down
        s["up"], s["gate"] = (_pack_weight(_normal(g, f32, b, ff, d) / d ** 0.5) for _ in range(2))
        s["down"] = _pack_weight(_normal(g, f32, b, d, ff) / ff ** 0.5)
        s["ln_w"], s["ln_b"] = 1.0 + 0.1 * _normal(g, f32, d), 0.1 * _normal(g, f32, d)
        return s
    if case["kind"] == "beam":
        rows = case["groups"] * case["beams"]
        s["logits"] = (3.0 * _normal(g, f32, rows, case["vocab"])).to(dt)
        s["scores"] = -20.0 + 2.0 * _normal(g, f32, rows)
        s["ended"] = None
        if case["ended"]:
            s["ended"] = (torch.rand(rows, generator=g, device="cuda") < 0.2).to(torch.int32)
        return s
    hkv, hd = case["kv_heads"], case["hd"]
    s["positions"] = _positions(g, case)
    if case["kind"] == "attend":
        rows, t = case["rows"], case["nodes"]
        s["cos"], s["sin"] = _tables(case["longest"] + t + 1, hd)
        s["cache"] = _cache(g, case, rows)
        # one packed projection, as a model's step has it
        qkv = _normal(g, dt, rows, t, case["heads"] + 2 * hkv, hd)
        s["q"], s["k_new"], s["v_new"] = qkv.split([case["heads"], hkv, hkv], dim=2)
        s["parents"] = None
        if t > 1:  # drafts branch now and then: a node follows the one before it, or any earlier one (-1: the context)
            i = torch.arange(t, device="cuda").expand(rows, t)
            any_earlier = (torch.rand((rows, t), generator=g, device="cuda") * (i + 1)).floor().long().clamp(max=i) - 1
            follow = torch.rand((rows, t), generator=g, device="cuda") < 0.6
            s["parents"] = torch.where(follow, i - 1, any_earlier).to(torch.int32)
        return s
    layers, rows, t = case["layers"], case["rows"], case["nodes"]
    s["cache"] = _cache(g, case, layers, rows)
    s["k_nodes"], s["v_nodes"] = _normal(g, dt, layers, rows, t, hkv, hd), _normal(g, dt, layers, rows, t, hkv, hd)
    # the accepted path: nodes in any order, from none to all of them (a step's one token and a prompt's: all)
    s["nodes"] = torch.rand((rows, t), generator=g, device="cuda").argsort(dim=1).to(torch.int32)
    s["counts"] = torch.randint(0, t + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    s["counts"][0] = t
    return s


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------

def _values(codes):
    """Bytes (.., b) as the levels (.., 2 b) that their codes stand for."""
    table = torch.tensor(LEVELS + tuple(-x for x in LEVELS), dtype=torch.float32, device=codes.device)
    return table[torch.stack([codes & 15, codes >> 4], dim=-1).long()].flatten(-2)


def _plain_weight(data, n, k):
    """(.., n, k) in fp32 of packed bytes."""
    lead = data.dim() - 3
    at = lambda *d: [*range(lead), *(lead + i for i in d)]  # noqa: E731
    w = _values(data[..., :1024]).unflatten(-1, (4, 16, 4, 8)).permute(at(0, 3, 1, 4, 2, 5))  # tile, r, block, g, h, j
    scale = data[..., 1024:].contiguous().view(torch.bfloat16).float().unflatten(-1, (16, 4)).permute(at(0, 2, 1, 3))
    w = w * scale[..., None, None]
    return w.flatten(lead + 2).flatten(lead, lead + 1)[..., :n, :k]


def _plain_linear(s):
    x = s["x"].float()
    if s["norm"]:
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6)
    y = x @ _plain_weight(s["w"], s["n"], s["k"]).T
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(s["x"].dtype)


def _plain_readout(s):
    x, d, ff = s["x"].float(), s["d"], s["ff"]
    if s["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * s["gain"].float()
    u = x @ _plain_weight(s["up"], ff, d).transpose(1, 2)
    g = x @ _plain_weight(s["gate"], ff, d).transpose(1, 2)
    z = (g / (1.0 + torch.exp(-g)) * u) @ _plain_weight(s["down"], d, ff).transpose(1, 2)
    z = z - z.mean(-1, keepdim=True)
    z = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-5)
    return (x + z * s["ln_w"] + s["ln_b"]).to(s["x"].dtype)


def _plain_cache(cache, hd):
    """Keys and values (.., blocks 32, hd) in fp32 of a packed cache (.., blocks, bytes)."""
    lead = cache.dim() - 1
    at = lambda *d: [*range(lead), *(lead + i for i in d)]  # noqa: E731
    words = hd // 16
    codes = _values(cache[..., :32 * hd]).unflatten(-1, (2, words // 4, 64, 4, 8))
    codes = codes.permute(at(0, 1, 3, 2, 4)).flatten(lead + 1, lead + 2)  # keys / values, word, lane, j
    scales = cache[..., 32 * hd:].contiguous().view(torch.bfloat16).float().unflatten(-1, (2, hd // 32, 4, 2, 4))
    scales = scales.permute(at(0, 3, 2, 4, 1)).flatten(lead + 1, lead + 3)  # keys / values, slot, g
    k = codes.select(lead, 0).unflatten(lead, (2, -1)).unflatten(lead + 2, (4, 16))  # t, g, h, r, j
    k = k.permute(at(0, 3, 1, 2, 4)).flatten(lead + 2).flatten(lead, lead + 1)
    v = codes.select(lead, 1).unflatten(lead + 1, (4, 16)).unflatten(-1, (2, 4))  # word, h, r, t, i
    v = v.permute(at(3, 1, 4, 0, 2)).flatten(lead + 3).flatten(lead, lead + 2)
    spread = scales.repeat_interleave(32, dim=-1)
    k, v = k * spread.select(lead, 0), v * spread.select(lead, 1)
    return k.flatten(lead - 1, lead), v.flatten(lead - 1, lead)


def _rotate(x, cos, sin):
    lo, hi = x.chunk(2, dim=-1)
    return x * cos + torch.cat([-hi, lo], dim=-1) * sin


def _attend(q, k, v, seen):
    """(n, heads, t, hd) over (n, kv heads, keys, hd); ``seen`` (n, t, keys)."""
    n, h, t, hd = q.shape
    hkv = k.shape[1]
    q = q.reshape(n, hkv, h // hkv * t, hd)
    score = (q @ k.transpose(2, 3).contiguous()) / math.sqrt(hd)
    score = score.view(n, h, t, -1).masked_fill(~seen[:, None], -math.inf)
    weight = (score - score.amax(3, keepdim=True)).exp()
    weight = weight / weight.sum(3, keepdim=True)
    return (weight.view(n, hkv, h // hkv * t, -1) @ v).view(n, h, t, hd)


def _reach(parents):
    """(n, t, t): whether node j is node i or one of its ancestors."""
    t = parents.shape[1]
    step = (parents[:, :, None] == torch.arange(t, device=parents.device)).float() + torch.eye(t, device=parents.device)
    for _ in range(6):  # paths of up to 64 steps, by doubling
        step = ((step @ step) > 0).float()
    return step > 0


def _held(s, p):
    """(n, slots of all blocks): the newest position below p that each slot can hold, negative where there is none."""
    win, sinks = s["window"], s["sinks"]
    front = -(-sinks // 32) * 32
    i = torch.arange(_blocks(s) * 32, device=p.device)
    ring = i - front
    newest = p[:, None] - 1 - (p[:, None] - 1 - sinks - ring) % win
    newest = torch.where((newest >= sinks) & (ring < win), newest, -1)
    return torch.where(i < front, torch.where((i < sinks) & (i < p[:, None]), i, -1), newest)


def _plain_attend(s):
    p, dt = s["positions"], s["q"].dtype
    n, t = s["q"].shape[:2]
    win, sinks = s["window"], s["sinks"]
    parents = s["parents"]
    if parents is None:
        parents = torch.arange(-1, t - 1, device=p.device).expand(n, t)
    reach = _reach(parents)
    where = p[:, None] + reach.sum(2) - 1  # (n, t)
    cos, sin = s["cos"][where][:, :, None], s["sin"][where][:, :, None]
    q, k = _rotate(s["q"].float(), cos, sin), _rotate(s["k_new"].float(), cos, sin).to(dt)
    held = _held(s, p)
    seen_ring = (held >= 0)[:, None] & ((held < sinks)[:, None] | (where[:, :, None] - held[:, None] < win))
    seen_tree = reach & ((where[:, None] < sinks) | (where[:, :, None] - where[:, None] < win))
    keys, values = _plain_cache(s["cache"], s["hd"])
    keys = torch.cat([keys, k.float().transpose(1, 2)], dim=2)
    values = torch.cat([values, s["v_new"].float().transpose(1, 2)], dim=2)
    out = _attend(q.transpose(1, 2), keys, values, torch.cat([seen_ring, seen_tree], dim=2))
    return out.transpose(1, 2).to(dt), k, s["v_new"].clone()


def _plain_commit(s):
    t, hd, win, sinks = s["nodes"].shape[1], s["hd"], s["window"], s["sinks"]
    front = -(-sinks // 32) * 32
    step = torch.arange(t, device=s["nodes"].device)
    at = s["positions"][:, None] + step
    slot = torch.where(at < sinks, at, front + (at - sinks) % win)
    last = (step < s["counts"][:, None]) & ((at < sinks) | (step + win >= s["counts"][:, None]))
    done = []
    for old, new in zip(_plain_cache(s["cache"], hd), (s["k_nodes"], s["v_nodes"])):
        layers, n, hkv, slots, _ = old.shape
        codes, scales = _quantise(new)
        table = torch.tensor(LEVELS + tuple(-x for x in LEVELS), dtype=torch.float32, device=old.device)
        new = (table[codes.long()].unflatten(-1, (-1, 32)) * scales.float()[..., None]).flatten(-2)
        order = s["nodes"].long()[None, :, None, :, None].expand(layers, n, hkv, t, hd)
        new = new.transpose(2, 3).gather(3, order)
        room = torch.cat([old, torch.zeros_like(old[..., :1, :])], dim=3)  # steps without a slot go behind the last
        index = torch.where(last, slot, slots)[None, :, None, :, None].expand(layers, n, hkv, t, hd)
        room.scatter_(3, index, new)
        done.append(torch.cat([room[..., :sinks, :], room[..., front:front + win, :]], dim=3).to(s["k_nodes"].dtype))
    return done


def _plain_beam(s):
    # in 64 bits: candidates of different beams are ordered by their sums
    x = s["logits"].double()
    rows, vocab = x.shape
    beams = s["beams"]
    ids = torch.arange(vocab, device=x.device)
    out_of_use = ids >= s["limit"]
    out_of_use[list(BANNED)] = True
    x = x.masked_fill(out_of_use, -math.inf)
    top = x.amax(1, keepdim=True)
    value = s["scores"].double()[:, None] + (x - top) - torch.log(torch.exp(x - top).sum(1, keepdim=True))
    if s["ended"] is not None:  # an ended beam goes on as it is
        stay = torch.where(ids == PAD, s["scores"].double()[:, None], -math.inf)
        value = torch.where(s["ended"][:, None] != 0, stay, value)
    value = value.view(-1, beams * vocab)
    best, order = torch.sort(value, dim=1, descending=True, stable=True)  # ties: the lowest beam, then the lowest id
    best, order = best[:, :beams], order[:, :beams]
    first = torch.arange(0, rows, beams, device=x.device)[:, None]
    token, source = (order % vocab).reshape(rows), (first + order // vocab).reshape(rows)
    ended = token == EOS
    if s["ended"] is not None:
        ended = ended | (s["ended"][source] != 0)
    return token, source.to(torch.int32), best.reshape(rows).float(), ended.to(torch.int32)


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------

def _own(s):
    from utttcompanion_amd import kernels as K
    kind = s["kind"]
    if kind == "linear":
        return K.linear4(s["x"], K.Weight4(s["w"], s["n"], s["k"]), residual=s["r"], x_eps=1e-6 if s["norm"] else 0.0)
    if kind == "readout":
        d, ff = s["d"], s["ff"]
        return K.readout4(s["x"], K.Weight4(s["up"], ff, d), K.Weight4(s["gate"], ff, d), K.Weight4(s["down"], d, ff),
                          s["ln_w"], s["ln_b"], 1e-5, x_norm=(s["gain"], 1e-6) if s["norm"] else None)
    if kind == "attend":
        return K.swa_tree4(s["q"], s["k_new"], s["v_new"], s["cache"], s["positions"], s["window"], s["parents"], s["cos"],
                           s["sin"], sinks=s["sinks"])
    if kind == "commit":
        K.kv_commit4(s["k_nodes"], s["v_nodes"], s["nodes"], s["counts"], s["cache"], s["positions"], s["window"],
                     sinks=s["sinks"])
        return K.kv_values4(s["cache"], s["window"], sinks=s["sinks"], dtype=s["k_nodes"].dtype)
    return K.beam_select(s["logits"], s["scores"], s["beams"], ended=s["ended"], banned=BANNED, active_limit=s["limit"],
                         eos=EOS, pad=PAD)


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "readout": _plain_readout, "attend": _plain_attend, "commit": _plain_commit,
            "beam": _plain_beam}[state["kind"]](state)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------

def _cached(case):
    """Cached tokens per request of a ragged batch, on average."""
    slots, longest = case["sinks"] + case["window"], case["longest"]
    spread = longest / 2 if longest <= slots else slots * (1 - slots / (2 * longest))
    return ((case["rows"] - 1) * spread + min(longest, slots)) / case["rows"]


def work(case):
    size = _size(case)
    four = 9 / 16  # bytes of a value with its share of the scale
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k * four + size * m * (k + n * (2 if case["residual"] else 1)), "flops": 2 * m * n * k}
    if case["kind"] == "readout":
        b, t, d, ff = case["rows"], case["tokens"], case["d"], case["ff"]
        return {"bytes": 3 * b * d * ff * four + 2 * size * b * t * d, "flops": 6 * b * t * d * ff}
    if case["kind"] == "beam":
        # every logit once; its exponential, its share of the sum and the comparisons
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * size + 24), "flops": 8 * rows * case["limit"]}
    rows, t, hkv, hd = case["rows"], case["nodes"], case["kv_heads"], case["hd"]
    if case["kind"] == "attend":
        mean = _cached(case)
        n = rows * hd * size * (2 * t * case["heads"] + 4 * t * hkv)
        return {"bytes": n + rows * mean * 2 * hkv * hd * four,
                "flops": 4 * rows * case["heads"] * t * (mean + (t + 1) / 2) * hd}
    # the new tokens read and written in 4 bits, the whole caches read and their values written
    taken = (1 + (rows - 1) / 2) * min(t, case["sinks"] + case["window"])
    held = rows * (case["sinks"] + case["window"])
    return {"bytes": case["layers"] * 2 * hkv * hd * (taken * (size + four) + held * (four + size)), "flops": 0}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------

def _level(code):
    """The number a code stands for: sign, two bits of exponent, one of mantissa."""
    sign, e, m = 1.0 - 2.0 * (code >> 3).double(), (code >> 1) & 3, (code & 1).double()
    return sign * torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * torch.exp2((e - 1).clamp(min=0).double()))


def _at(data, byte, high=None):
    """The code at a byte index per element (its high half where ``high``), of flat bytes."""
    b = data.reshape(-1)[byte].long()
    return b & 15 if high is None else torch.where(high, b >> 4, b & 15)


def _bf16_at(data, byte):
    b = data.reshape(-1)
    bits = (b[byte].int() | (b[byte + 1].int() << 8)) << 16
    return bits.view(torch.float32).double()


def _exact_weight(data, n, k):
    """(n, k) in 64 bits of one packed matrix, element by element from its address."""
    i, j = torch.arange(n, device=data.device)[:, None], torch.arange(k, device=data.device)[None]
    block = ((i // 16) * data.shape[-2] + j // 128) * 1152
    c = j % 128
    word = block + (((c % 32) // 8) * 16 + i % 16) * 16 + (c // 32) * 4
    byte = word + (c % 8) // 2
    value = _level(_at(data, byte, (c % 2 == 1).expand_as(byte)))
    return value * _bf16_at(data, block + 1024 + ((i % 16) * 4 + c // 32) * 2)


def _exact_cache(cache, hd, slots):
    """Keys and values (slots, hd) in 64 bits of one head's packed blocks (blocks, bytes), of the slots given."""
    e = torch.arange(hd, device=cache.device)[None]
    slot, base = (slots % 32)[:, None], (slots // 32)[:, None] * cache.shape[-1]
    got = []
    for part in range(2):
        if part == 0:
            word = (slot // 16) * (hd // 32) + e // 32
            lane, j = ((e % 32) // 8) * 16 + slot % 16, (e % 8).expand(len(slots), hd)
        else:
            word = (e // 16).expand(len(slots), hd)
            lane, j = ((slot % 16) // 4) * 16 + e % 16, (slot // 16 * 4 + slot % 4).expand(len(slots), hd)
        byte = base + part * 16 * hd + (word // 4) * 1024 + lane * 16 + (word % 4) * 4 + j // 2
        scale = base + 32 * hd + part * 2 * hd + (e // 32) * 64 + ((slot % 16) // 4) * 16 + (slot // 16 * 4 + slot % 4) * 2
        got.append(_level(_at(cache, byte, j % 2 == 1)) * _bf16_at(cache, scale))
    return got


def _exact_fours(x):
    """x (.., K) as 4 bits hold it: the scale's and the quotient's roundings are the definition's."""
    y = x.float().reshape(-1, 32)
    s = (y.abs().max(1, keepdim=True).values * torch.tensor(1 / 6, dtype=torch.float32, device=x.device)).bfloat16().float()
    s = s * (s >= 2.0 ** -126)
    t = (y / torch.where(s > 0, s, 1.0)).double()
    grid = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    gap = (t.abs().clamp(max=6.0)[..., None] - grid).abs()
    # the nearest level; of two as near the one with an even code
    gap = gap + torch.arange(8, device=x.device) % 2 * 1e-12
    return (grid[gap.argmin(-1)] * t.sign() * s.double()).reshape(x.shape)


def _softmax_rows(q, k, v, seen):
    """One head: (t, hd) over (keys, hd) with ``seen`` (t, keys), in 64 bits."""
    e = torch.where(seen, q @ k.T / q.shape[1] ** 0.5, -math.inf)
    e = torch.exp(e - e.max(1, keepdim=True).values)
    return e @ torch.where(seen.any(0)[:, None], v, 0.0) / e.sum(1, keepdim=True)


def _turn(x, c, s):
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half], x[..., half:], c[..., :half], s[..., :half]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _exact_attend(s, case):
    hd, win, sinks, rep = case["hd"], case["window"], case["sinks"], case["heads"] // case["kv_heads"]
    front = -(-sinks // 32) * 32
    q, kn, vn = s["q"].double(), s["k_new"].double(), s["v_new"].double()
    t, dev = q.shape[1], q.device
    p, cos, sin = s["positions"].tolist(), s["cos"].double(), s["sin"].double()
    parents = [list(range(-1, t - 1))] * len(p) if s["parents"] is None else s["parents"].tolist()
    out, turned = torch.empty_like(q), torch.empty_like(kn)
    for n in range(len(p)):
        line = []  # each node's path from the context, itself last
        for i, up in enumerate(parents[n]):
            line.append((line[up] if up >= 0 else []) + [i])
        at = p[n] + torch.tensor([len(x) - 1 for x in line], device=dev)
        qn, turned[n] = _turn(q[n], cos[at][:, None], sin[at][:, None]), _turn(kn[n], cos[at][:, None], sin[at][:, None])
        stored = turned[n].to(s["q"].dtype).double()
        # the positions that the cache still holds, and their slots
        old = torch.tensor([j for j in range(p[n]) if j < sinks or j >= p[n] - win], dtype=torch.int64, device=dev)
        slot = torch.where(old < sinks, old, front + (old - sinks) % win)
        on_path = torch.zeros((t, t), dtype=torch.bool)
        for i in range(t):
            on_path[i, line[i]] = True
        key_at = torch.cat([old, at])
        near = (at[:, None] - key_at[None] < win) | (key_at < sinks)[None]
        seen = torch.cat([torch.ones((t, len(old)), dtype=torch.bool, device=dev), on_path.to(dev)], dim=1) & near
        for g in range(case["kv_heads"]):
            keys, values = _exact_cache(s["cache"][n, g], hd, slot)
            keys, values = torch.cat([keys, stored[:, g]]), torch.cat([values, vn[n, :, g]])
            for h in range(g * rep, (g + 1) * rep):
                out[n, :, h] = _softmax_rows(qn[:, h], keys, values, seen)
    return out, turned, vn


def _exact_commit(s, case):
    hd, win, sinks = case["hd"], case["window"], case["sinks"]
    front = -(-sinks // 32) * 32
    slots = torch.cat([torch.arange(sinks), torch.arange(front, front + win)]).to(s["cache"].device)
    layers, rows, hkv = s["cache"].shape[:3]
    k, v = (torch.empty((layers, rows, hkv, sinks + win, hd), dtype=torch.float64, device=slots.device) for _ in range(2))
    for i in range(layers):
        for n in range(rows):
            for h in range(hkv):
                k[i, n, h], v[i, n, h] = _exact_cache(s["cache"][i, n, h], hd, slots)
    p, nodes, counts = s["positions"].tolist(), s["nodes"].tolist(), s["counts"].tolist()
    k_new, v_new = _exact_fours(s["k_nodes"]), _exact_fours(s["v_nodes"])
    for n in range(rows):
        newest = {}
        for a in range(counts[n]):
            j = p[n] + a
            newest[j if j < sinks else sinks + (j - sinks) % win] = nodes[n][a]
        if newest:
            to, of = list(newest), list(newest.values())
            k[:, n, :, to], v[:, n, :, to] = k_new[:, n, of].transpose(1, 2), v_new[:, n, of].transpose(1, 2)
    return k, v


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        x = s["x"].double()
        if case["norm"]:
            x = x / (x.pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
        y = torch.cat([x @ _exact_weight(s["w"][i // 16:i // 16 + 256], min(4096, case["n"] - i), case["k"]).T
                       for i in range(0, case["n"], 4096)], dim=1)
        return y if s["r"] is None else y + s["r"].double()
    if case["kind"] == "readout":
        out = []
        for b in range(case["rows"]):
            x = s["x"][b].double()
            if case["norm"]:
                x = x / (x.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * s["gain"].double()
            h = x @ _exact_weight(s["gate"][b], case["ff"], case["d"]).T
            h = h * torch.sigmoid(h) * (x @ _exact_weight(s["up"][b], case["ff"], case["d"]).T)
            z = h @ _exact_weight(s["down"][b], case["d"], case["ff"]).T
            z = (z - z.mean(1, keepdim=True)) / (z.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
            out.append(x + z * s["ln_w"].double() + s["ln_b"].double())
        return torch.stack(out)
    if case["kind"] == "attend":
        return _exact_attend(s, case)
    if case["kind"] == "commit":
        return _exact_commit(s, case)
    beams, best = case["beams"], []
    for r in range(0, case["groups"] * beams, beams):
        found = []
        for b in range(r, r + beams):
            if s["ended"] is not None and int(s["ended"][b]):
                found.append(s["scores"][b:b + 1].double())
                continue
            row = s["logits"][b, :case["limit"]].double()
            row[list(BANNED)] = -math.inf
            found.append(float(s["scores"][b]) + torch.log_softmax(row, 0).topk(beams).values)
        best.append(torch.cat(found).topk(beams).values)
    return None, None, torch.cat(best), None
