"""The serving operators around batched decoding, in plain form and as the framework's calls, for timing and comparing.

* ``sample``   next tokens from logits by temperature, top-k, min-p and top-p, each request with its own settings, from
               given uniform numbers (beside the greedy choice of a decode step);
* ``prefill``  sliding-window attention of a prompt whose first keys (sinks) stay visible;
* ``decode``   the same for one token per request, over ring caches with sink slots in front;
* ``tree``     attention of a tree of drafted tokens per request over such caches;
* ``commit``   the accepted nodes' keys and values into the caches of all layers;
* ``fork``     requests' caches copied over others' (forks of one prompt, beams, gaps closed after requests end).

With ``own`` false ``run`` computes them with elementary torch operations; with ``own`` true it calls the framework.
Widths come from the benchmark's model configurations and ``uTTTConfig``'s defaults.
"""
from __future__ import annotations

import math

import torch

own = False

BANNED = (0, 1, 3)  # padding, begin of text, unknown
THETA = 10000.0


def listed():
    return [
        # one user's next token, the default temperature and top-p, half of the vocabulary in use
        dict(name="sample_1x32000", kind="sample", rows=1, vocab=32000, limit=21478, settings="default", dtype="bf16"),
        # a full batch over a large vocabulary, every request with settings of its own, greedy ones among them
        dict(name="sample_256x131072", kind="sample", rows=256, vocab=131072, limit=131072, settings="mixed",
             dtype="fp32"),
        # a follow-up turn on top of a full cache, odd length, research precision
        dict(name="prefill_3x777_fp32", kind="prefill", rows=3, tokens=777, heads=12, kv_heads=4, hd=64, window=512,
             sinks=4, history=515, dtype="fp32"),
        # long prompts
        dict(name="prefill_4x4096", kind="prefill", rows=4, tokens=4096, heads=16, kv_heads=4, hd=128, window=1024,
             sinks=64, history=0, dtype="bf16"),
        # one user, one token: latency
        dict(name="decode_1x512", kind="decode", rows=1, heads=16, kv_heads=4, hd=64, window=512, sinks=4, longest=3000,
             dtype="bf16"),
        # batched serving over long windows, ragged contexts from short to wrapped
        dict(name="decode_32x4096", kind="decode", rows=32, heads=16, kv_heads=4, hd=128, window=4096, sinks=4,
             longest=12000, dtype="bf16"),
        # one user's few drafted tokens: latency
        dict(name="tree_1x8", kind="tree", rows=1, nodes=8, heads=12, kv_heads=4, hd=64, window=512, sinks=4,
             longest=2000, dtype="bf16"),
        # the largest trees for several users over long windows
        dict(name="tree_16x64", kind="tree", rows=16, nodes=64, heads=16, kv_heads=4, hd=128, window=4096, sinks=4,
             longest=12000, dtype="bf16"),
        # the accepted part of one user's draft into twelve layers' rings
        dict(name="commit_1x8", kind="commit", layers=12, rows=1, nodes=8, kv_heads=4, hd=64, window=512, sinks=4,
             longest=2000, dtype="bf16"),
        # the same for a batch of large drafts through the 24 layers of the large model
        dict(name="commit_32x64", kind="commit", layers=24, rows=32, nodes=64, kv_heads=4, hd=128, window=1024,
             sinks=4, longest=4000, dtype="bf16"),
        # one prompt continued by four samplers
        dict(name="fork_4", kind="fork", layers=12, rows=4, kv_heads=4, hd=64, window=512, sinks=4, longest=2000,
             moves="first", dtype="bf16"),
        # beams of a batch reordered: any request may take any other's cache
        dict(name="fork_16_reorder", kind="fork", layers=24, rows=16, kv_heads=4, hd=128, window=1024, sinks=4,
             longest=4000, moves="any", dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges."""
    kind = rng.choice(["sample", "sample", "prefill", "decode", "tree", "tree", "commit", "fork"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "sample":
        rows, vocab = _log(rng, 1, 256), _log(rng, 256, 131072)
        return dict(kind=kind, rows=rows, vocab=vocab, limit=rng.choice([vocab, vocab - rng.randint(1, vocab // 3)]),
                    settings=rng.choice(["default", "mixed", "plain"]), dtype=dtype)
    hd = rng.choice([64, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 4])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 8])
    sinks = rng.choice([0, 1, 4, rng.randint(2, 64)])
    if kind == "prefill":
        window = rng.choice([512, 1024, _log(rng, 16, 1024)])
        tokens = _log(rng, 1, 4096 if dtype == "bf16" else 1024)
        return dict(kind=kind, rows=_log(rng, 1, 4), tokens=tokens, heads=min(heads, 16), kv_heads=kv_heads, hd=hd,
                    window=window, sinks=max(sinks, 1), history=rng.choice([0, rng.randint(0, sinks + window - 1)]),
                    dtype=dtype)
    window = rng.choice([512, 1024, _log(rng, 64, 4096)])
    longest = _log(rng, 16, 3 * window)
    if kind == "decode":
        return dict(kind=kind, rows=_log(rng, 1, 32), heads=heads, kv_heads=kv_heads, hd=hd, window=window,
                    sinks=max(sinks, 1), longest=longest, dtype=dtype)
    if kind == "tree":
        return dict(kind=kind, rows=_log(rng, 1, 16), nodes=rng.choice([1, rng.randint(2, 16), rng.randint(17, 64)]),
                    heads=min(heads, 16), kv_heads=kv_heads, hd=hd, window=window, sinks=sinks, longest=longest,
                    dtype=dtype)
    layers = rng.choice([1, 6, 12, 24])
    if kind == "commit":
        return dict(kind=kind, layers=layers, rows=_log(rng, 1, 32), nodes=_log(rng, 1, 64), kv_heads=kv_heads, hd=hd,
                    window=min(window, 1024), sinks=sinks, longest=longest, dtype=dtype)
    return dict(kind=kind, layers=min(layers, 12) if dtype == "fp32" else layers, rows=_log(rng, 2, 16),
                kv_heads=kv_heads, hd=hd, window=min(window, 1024), sinks=sinks, longest=longest,
                moves=rng.choice(["first", "any"]), dtype=dtype)


# ------------------------------------------------------------------------------------------------
# what a program has in hand
# ------------------------------------------------------------------------------------------------

def _dtype(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.bfloat16


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


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
    dt, rows = _dtype(case), case["rows"]
    if case["kind"] == "sample":
        s["logits"] = (3.0 * torch.randn((rows, case["vocab"]), generator=g, device="cuda")).to(dt)
        s["uniforms"] = torch.rand(rows, generator=g, device="cuda")
        ones = torch.ones(rows, device="cuda")
        pick = torch.rand((4, rows), generator=g, device="cuda")
        if case["settings"] == "default":
            s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.7 * ones, None, 0.9 * ones, None
        elif case["settings"] == "plain":
            s["temperature"], s["top_k"], s["top_p"], s["min_p"] = ones, None, None, None
        else:  # every request its own: some greedy, some without a top-k, top-p or min-p
            s["temperature"] = torch.where(pick[0] < 0.1, 0.0 * ones, 0.3 + 1.2 * pick[0])
            s["top_k"] = torch.where(pick[1] < 0.4, 0.0 * ones, 1 + 200 * pick[1]).to(torch.int32)
            s["top_p"] = torch.where(pick[2] < 0.4, ones, 0.3 + 0.69 * pick[2])
            s["min_p"] = torch.where(pick[3] < 0.5, 0.0 * ones, 0.1 * pick[3])
        return s
    hkv, hd, win, sinks = case["kv_heads"], case["hd"], case["window"], case["sinks"]
    if case["kind"] == "prefill":
        t, kv = case["tokens"], case["history"] + case["tokens"]
        s["q"] = _normal(g, dt, rows, t, case["heads"], hd).transpose(1, 2)
        s["k"], s["v"] = _normal(g, dt, rows, hkv, kv, hd), _normal(g, dt, rows, hkv, kv, hd)
        return s
    slots = sinks + win
    if case["kind"] in ("decode", "tree"):
        s["positions"] = _positions(g, case)
        t = case.get("nodes", 1)
        s["cos"], s["sin"] = _tables(case["longest"] + t + 1, hd)
        s["k_ring"], s["v_ring"] = _normal(g, dt, rows, hkv, slots, hd), _normal(g, dt, rows, hkv, slots, hd)
        # one packed projection, as a model's step has it
        qkv = _normal(g, dt, rows, t, case["heads"] + 2 * hkv, hd)
        q, k, v = qkv.split([case["heads"], hkv, hkv], dim=2)
        s["q"], s["k_new"], s["v_new"] = q, k, v
        if case["kind"] == "decode":
            s["q"], s["k_new"], s["v_new"] = q[:, 0], k[:, 0], v[:, 0]
        else:  # drafts branch now and then: a node follows the one before it, or any earlier one (-1: the context)
            i = torch.arange(t, device="cuda").expand(rows, t)
            any_earlier = (torch.rand((rows, t), generator=g, device="cuda") * (i + 1)).floor().long().clamp(max=i) - 1
            follow = torch.rand((rows, t), generator=g, device="cuda") < 0.6
            s["parents"] = torch.where(follow, i - 1, any_earlier).to(torch.int32)
        return s
    layers = case["layers"]
    s["positions"] = _positions(g, case)
    s["k_ring"] = _normal(g, dt, layers, rows, hkv, slots, hd)
    s["v_ring"] = _normal(g, dt, layers, rows, hkv, slots, hd)
    if case["kind"] == "commit":
        t = case["nodes"]
        s["k_nodes"], s["v_nodes"] = _normal(g, dt, layers, rows, t, hkv, hd), _normal(g, dt, layers, rows, t, hkv, hd)
        # the accepted path: nodes in rising order, from none to all of them
        s["nodes"] = torch.rand((rows, t), generator=g, device="cuda").argsort(dim=1).to(torch.int32)
        s["counts"] = torch.randint(0, t + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["counts"][0] = (t + 1) // 2
        return s
    if case["moves"] == "first":
        s["sources"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    else:
        s["sources"] = torch.randint(0, rows, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return s


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------

def _plain_sample(s):
    x = s["logits"].float()
    vocab = x.shape[1]
    ids = torch.arange(vocab, device=x.device)
    out_of_use = ids >= s["limit"]
    out_of_use[list(BANNED)] = True
    x = x.masked_fill(out_of_use, -math.inf)
    greedy = s["temperature"] <= 1e-5
    heat = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    ranked, order = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest id first
    # in 64 bits: the sums decide between neighbours
    weight = torch.exp((ranked.double() - ranked[:, :1].double()) / heat)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] <= 0, vocab, s["top_k"])[:, None]
        weight = weight * (ids < k)
    if s["min_p"] is not None:
        weight = weight * (weight >= s["min_p"].double()[:, None])
    if s["top_p"] is not None:
        ahead = weight.cumsum(1) - weight
        weight = weight * (ahead <= s["top_p"].double()[:, None] * weight.sum(1, keepdim=True))
    by_id = torch.zeros_like(weight).scatter_(1, order, weight)
    below = by_id.cumsum(1)
    total = below[:, -1]
    drawn = (below <= (s["uniforms"].double() * total)[:, None]).sum(1)
    token = torch.where(greedy, order[:, 0], drawn)
    chosen = by_id.gather(1, token[:, None])[:, 0]
    logprob = torch.where(greedy, 0.0, torch.log(chosen / total))
    return token, logprob.float()


def _plain_prefill(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    rep = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    i = torch.arange(q.shape[2], device=q.device)[:, None] + s["history"]
    j = torch.arange(k.shape[2], device=q.device)
    seen = (j <= i) & ((i - j < s["window"]) | (j < s["sinks"]))
    score = (q @ k.transpose(2, 3)) / math.sqrt(q.shape[3])
    score.masked_fill_(~seen, -math.inf)
    score -= score.amax(3, keepdim=True)
    weight = score.exp_()
    return ((weight @ v) / weight.sum(3, keepdim=True)).to(s["q"].dtype)


def _rotate(x, cos, sin):
    lo, hi = x.chunk(2, dim=-1)
    return x * cos + torch.cat([-hi, lo], dim=-1) * sin


def _slots(positions, s):
    """The cache slots of absolute positions."""
    return torch.where(positions < s["sinks"], positions, s["sinks"] + (positions - s["sinks"]) % s["window"])


def _attend(q, k, v, seen):
    """(n, heads, t, hd) over (n, kv heads, keys, hd); ``seen`` (n, t, keys)."""
    n, h, t, hd = q.shape
    hkv = k.shape[1]
    q = q.reshape(n, hkv, h // hkv * t, hd)
    score = (q @ k.transpose(2, 3)) / math.sqrt(hd)
    score = score.view(n, h, t, -1).masked_fill(~seen[:, None], -math.inf)
    weight = (score - score.amax(3, keepdim=True)).exp()
    weight = weight / weight.sum(3, keepdim=True)
    return (weight.view(n, hkv, h // hkv * t, -1) @ v).view(n, h, t, hd)


def _plain_decode(s):
    p, dt = s["positions"], s["q"].dtype
    n, slots = p.shape[0], s["k_ring"].shape[2]
    cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]
    q, k = _rotate(s["q"].float(), cos, sin), _rotate(s["k_new"].float(), cos, sin)
    at = _slots(p, s)
    rows = torch.arange(n, device=p.device)
    s["k_ring"][rows, :, at] = k.to(dt)
    s["v_ring"][rows, :, at] = s["v_new"]
    seen = torch.arange(slots, device=p.device) < (p + 1).clamp(max=slots)[:, None]
    out = _attend(q[:, :, None], s["k_ring"].float(), s["v_ring"].float(), seen[:, None])
    return out[:, :, 0].to(dt), s["k_ring"], s["v_ring"]


def _reach(parents):
    """(n, t, t): whether node j is node i or one of its ancestors."""
    t = parents.shape[1]
    step = (parents[:, :, None] == torch.arange(t, device=parents.device)).float() + torch.eye(t, device=parents.device)
    for _ in range(6):  # paths of up to 64 steps, by doubling
        step = ((step @ step) > 0).float()
    return step > 0


def _plain_tree(s):
    p, dt = s["positions"], s["q"].dtype
    win, sinks, slots = s["window"], s["sinks"], s["k_ring"].shape[2]
    reach = _reach(s["parents"])
    depth = reach.sum(2) - 1
    where = p[:, None] + depth  # (n, t)
    cos, sin = s["cos"][where][:, :, None], s["sin"][where][:, :, None]
    q, k = _rotate(s["q"].float(), cos, sin), _rotate(s["k_new"].float(), cos, sin)
    # the newest position before p that each slot can hold
    slot = torch.arange(slots, device=p.device)
    held = p[:, None] - 1 - (p[:, None] - 1 - slot) % win
    held = torch.where(slot < sinks, slot, held)
    there = (held < p[:, None]) & (held >= torch.where(slot < sinks, 0, sinks))
    seen_ring = there[:, None] & ((slot < sinks) | (where[:, :, None] - held[:, None] < win))
    seen_tree = reach & ((where[:, None] < sinks) | (where[:, :, None] - where[:, None] < win))
    keys = torch.cat([s["k_ring"].float(), k.transpose(1, 2)], dim=2)
    values = torch.cat([s["v_ring"].float(), s["v_new"].float().transpose(1, 2)], dim=2)
    # unwritten slots may hold anything
    used = torch.cat([there, torch.ones_like(where, dtype=torch.bool)], dim=1)[:, None, :, None]
    values = values.masked_fill(~used, 0.0)
    out = _attend(q.transpose(1, 2), keys, values, torch.cat([seen_ring, seen_tree], dim=2))
    return out.transpose(1, 2).to(dt), k.to(dt), s["v_new"].clone()


def _plain_commit(s):
    t = s["nodes"].shape[1]
    step = torch.arange(t, device=s["nodes"].device)
    valid = (step < s["counts"][:, None])[None, :, None, :, None]
    at = _slots(s["positions"][:, None] + step, s)
    for ring, nodes in ((s["k_ring"], s["k_nodes"]), (s["v_ring"], s["v_nodes"])):
        layers, n, hkv, _, hd = ring.shape
        index = at[None, :, None, :, None].expand(layers, n, hkv, t, hd)
        order = s["nodes"].long()[None, :, None, :, None].expand(layers, n, hkv, t, hd)
        new = nodes.transpose(2, 3).gather(3, order)
        ring.scatter_(3, index, torch.where(valid, new, ring.gather(3, index)))
    return s["k_ring"], s["v_ring"]


def _plain_fork(s):
    src, p = s["sources"].long(), s["positions"]
    slots = s["k_ring"].shape[3]
    moved = (src != torch.arange(len(src), device=src.device))[:, None]
    take = (moved & (torch.arange(slots, device=src.device) < p[src][:, None]))[None, :, None, :, None]
    for ring in (s["k_ring"], s["v_ring"]):
        ring.copy_(torch.where(take, ring[:, src], ring))
    p.copy_(p[src])
    return s["k_ring"], s["v_ring"], p


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------

def _own(s):
    from utttcompanion_amd import kernels as K
    kind = s["kind"]
    if kind == "sample":
        return K.sample_select(s["logits"], s["uniforms"], s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                               min_p=s["min_p"], banned=BANNED, active_limit=s["limit"])
    if kind == "prefill":
        return K.swa_prefill(s["q"], s["k"], s["v"], s["window"], s["history"], sinks=s["sinks"])
    if kind == "decode":
        out = K.swa_decode(s["q"], s["k_new"], s["v_new"], s["k_ring"], s["v_ring"], s["positions"], s["cos"],
                           s["sin"], sinks=s["sinks"])
        return out, s["k_ring"], s["v_ring"]
    if kind == "tree":
        return K.swa_tree(s["q"], s["k_new"], s["v_new"], s["k_ring"], s["v_ring"], s["positions"], s["parents"],
                          s["cos"], s["sin"], sinks=s["sinks"])
    if kind == "commit":
        K.kv_commit(s["k_nodes"], s["v_nodes"], s["nodes"], s["counts"], s["k_ring"], s["v_ring"], s["positions"],
                    sinks=s["sinks"])
        return s["k_ring"], s["v_ring"]
    K.kv_fork(s["k_ring"], s["v_ring"], s["sources"], s["positions"])
    return s["k_ring"], s["v_ring"], s["positions"]


def run(state):
    if own:
        return _own(state)
    return {"sample": _plain_sample, "prefill": _plain_prefill, "decode": _plain_decode, "tree": _plain_tree,
            "commit": _plain_commit, "fork": _plain_fork}[state["kind"]](state)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------

def _cached(case):
    """Cached tokens per request of a ragged batch, on average."""
    slots, longest = case["sinks"] + case["window"], case["longest"]
    spread = longest / 2 if longest <= slots else slots * (1 - slots / (2 * longest))
    return ((case["rows"] - 1) * spread + min(longest, slots)) / case["rows"]


def work(case):
    size, rows = _size(case), case["rows"]
    if case["kind"] == "sample":
        # every logit once; its exponential, its share of the sums and the comparisons
        return {"bytes": rows * (case["vocab"] * size + 32), "flops": 8 * rows * case["limit"]}
    hkv, hd, win, sinks = case["kv_heads"], case["hd"], case["window"], case["sinks"]
    pairs = 0
    mean = _cached(case) if "longest" in case else 0
    if case["kind"] == "prefill":
        t, hist = case["tokens"], case["history"]
        for i in range(hist, hist + t):
            recent = min(i + 1, win)
            pairs += recent + min(sinks, i + 1 - recent)
        n = rows * hd * ((2 * t * case["heads"]) + 2 * hkv * (hist + t))
        return {"bytes": n * size, "flops": 4 * rows * case["heads"] * pairs * hd}
    if case["kind"] in ("decode", "tree"):
        t = case.get("nodes", 1)
        n = rows * hd * (2 * hkv * mean + 2 * t * case["heads"] + 4 * t * hkv)
        return {"bytes": n * size, "flops": 4 * rows * case["heads"] * t * (mean + (t + 1) / 2) * hd}
    if case["kind"] == "commit":
        moved = rows * case["nodes"]  # half of the nodes, read and written
    else:  # each source once, every request that takes another's cache
        moved = mean * (rows - 1 + (1 if case["moves"] == "first" else 0.63 * rows))
    return {"bytes": moved * case["layers"] * 2 * hkv * hd * size, "flops": 0}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------

def _softmax_rows(q, k, v, seen):
    """One head: (t, hd) over (keys, hd) with ``seen`` (t, keys), in 64 bits."""
    e = torch.where(seen, q @ k.T / q.shape[1] ** 0.5, -math.inf)
    e = torch.exp(e - e.max(1, keepdim=True).values)
    return e @ torch.where(seen.any(0)[:, None], v, 0.0) / e.sum(1, keepdim=True)


def _turn(x, c, s):
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half], x[..., half:], c[..., :half], s[..., :half]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _exact_sample(s):
    """The logarithm of the chosen token's share, from log-sum-exp over the tokens that stay."""
    token = _plain_sample(s)[0]
    x = s["logits"].double()
    got = torch.zeros(len(token), dtype=torch.float64, device=x.device)
    for r in range(x.shape[0]):
        heat = float(s["temperature"][r])
        if heat <= 1e-5:
            continue
        row = x[r, :s["limit"]].clone()
        row[list(BANNED)] = -math.inf
        z = row / heat
        top, ids = z.sort(descending=True, stable=True)
        p = torch.softmax(top, 0)
        n = len(top)
        k = int(s["top_k"][r]) if s["top_k"] is not None else 0
        if k > 0:
            n = min(n, k)
        if s["min_p"] is not None and float(s["min_p"][r]) > 0:
            n = min(n, int((p >= float(s["min_p"][r]) * p[0]).sum()))
        if s["top_p"] is not None:
            before = torch.cat([p.new_zeros(1), p[:n].cumsum(0)[:-1]])
            n = int((before <= float(s["top_p"][r]) * p[:n].sum()).sum())
        got[r] = z[token[r]] - torch.logsumexp(top[:n], 0)
    return None, got


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] in ("commit", "fork"):
        # copies: the definition, request by request
        k, v = s["k_ring"].double(), s["v_ring"].double()
        p = s["positions"].tolist()
        slots = k.shape[3]
        place = lambda j: j if j < s["sinks"] else s["sinks"] + (j - s["sinks"]) % s["window"]  # noqa: E731
        if case["kind"] == "commit":
            nodes, counts = s["nodes"].tolist(), s["counts"].tolist()
            for n in range(case["rows"]):
                for a in range(counts[n]):
                    k[:, n, :, place(p[n] + a)] = s["k_nodes"][:, n, nodes[n][a]].double()
                    v[:, n, :, place(p[n] + a)] = s["v_nodes"][:, n, nodes[n][a]].double()
            return k, v
        src = s["sources"].tolist()
        for n in range(case["rows"]):
            if src[n] != n:
                m = min(p[src[n]], slots)
                k[:, n, :, :m] = s["k_ring"][:, src[n], :, :m].double()
                v[:, n, :, :m] = s["v_ring"][:, src[n], :, :m].double()
        return k, v, None
    rep = case["heads"] // case["kv_heads"]
    win, sinks = case["window"], case["sinks"]
    dev = s["q"].device
    if case["kind"] == "prefill":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        at = case["history"] + torch.arange(case["tokens"], device=dev)
        key = torch.arange(k.shape[2], device=dev)
        gap = at[:, None] - key[None]
        seen = (gap >= 0) & ((gap < win) | (key < sinks)[None])
        out = torch.empty_like(q)
        for b in range(q.shape[0]):
            for h in range(q.shape[1]):
                out[b, h] = _softmax_rows(q[b, h], k[b, h // rep], v[b, h // rep], seen)
        return out
    p = s["positions"].tolist()
    cos, sin = s["cos"].double(), s["sin"].double()
    if case["kind"] == "decode":
        q, kn, vn = (s[x].double()[:, None] for x in ("q", "k_new", "v_new"))
        parents = [[-1]] * case["rows"]
    else:
        q, kn, vn = s["q"].double(), s["k_new"].double(), s["v_new"].double()
        parents = s["parents"].tolist()
    k_ring, v_ring = s["k_ring"].double(), s["v_ring"].double()
    out, turned = torch.empty_like(q), torch.empty_like(kn)
    t = q.shape[1]
    for n in range(case["rows"]):
        line, depth = [], []  # each node's path from the context, itself last
        for i, up in enumerate(parents[n]):
            line.append((line[up] if up >= 0 else []) + [i])
            depth.append(len(line[i]) - 1)
        at = p[n] + torch.tensor(depth, device=dev)
        qn, turned[n] = _turn(q[n], cos[at][:, None], sin[at][:, None]), _turn(kn[n], cos[at][:, None], sin[at][:, None])
        # the positions that the cache still holds, and their slots
        old = torch.tensor([j for j in range(p[n]) if j < sinks or j >= p[n] - win], dtype=torch.int64, device=dev)
        slot = torch.where(old < sinks, old, sinks + (old - sinks) % win)
        on_path = torch.zeros((t, t), dtype=torch.bool)
        for i in range(t):
            on_path[i, line[i]] = True
        key_at = torch.cat([old, at])
        near = (at[:, None] - key_at[None] < win) | (key_at < sinks)[None]
        seen = torch.cat([torch.ones((t, len(old)), dtype=torch.bool, device=dev), on_path.to(dev)], dim=1) & near
        for h in range(q.shape[2]):
            g = h // rep
            keys = torch.cat([k_ring[n, g, slot], turned[n, :, g]])
            values = torch.cat([v_ring[n, g, slot], vn[n, :, g]])
            out[n, :, h] = _softmax_rows(qn[:, h], keys, values, seen)
        if case["kind"] == "decode":
            here = p[n] if p[n] < sinks else sinks + (p[n] - sinks) % win
            k_ring[n, :, here], v_ring[n, :, here] = turned[n, 0], vn[n, 0]
    if case["kind"] == "decode":
        return out[:, 0], k_ring, v_ring
    return out, turned, vn
