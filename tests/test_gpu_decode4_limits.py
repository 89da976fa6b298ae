"""Attention over caches in 4 bits where numbers are not finite: a key of score -inf has no weight, one of +inf or NaN makes the rows
that see it NaN."""
import math

import pytest
import torch

import decode_reference as R
from test_gpu_decode4 import DEV, STEP, U, cache_of, gen, normal, within
from utttcompanion_amd import kernels as K

pytestmark = pytest.mark.gpu


def attention_bound(score, size, want, hd, keys, dt):
    """What test_gpu_decode4 allows an output, from the largest sum of magnitudes behind a score and the sum behind the output."""
    carried, weight = (2.0 ** -16, 2.0 ** -8) if dt is torch.bfloat16 else (2.0 ** -23, 2.0 ** -23)
    ds = score * (carried + (34 + hd / 32 + 8) * U) + 4 * U * 40
    rel = (2 * ds * (1 + ds)).unsqueeze(-1) + weight + 2 * (34 + keys / 32 + 80) * U + 8 * U
    return rel * size + STEP[dt] * want.abs() * (1 + 2 ** -7)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t", [1, 6, 40])
def test_infinite_new_keys(t, hd, dt):
    """Single infinite elements of a few nodes' keys, seen by heads whose q has either sign, or 0, there."""
    g = gen(t + hd)
    window, sinks, heads, hkv = 50, 3, 4, 2
    positions = torch.tensor([0, 30, 200])
    n = len(positions)
    c = cache_of(g, 1, n, hkv, window, sinks, hd)[0]
    q, k, v = (normal(g, n, t, h, hd) for h in (heads, hkv, hkv))
    q[1, 0, 1, 5] = 0.0
    q, k, v = (x.to(dt) for x in (q, k, v))
    parents = None
    if t > 1:
        parents = torch.tensor([[i // 2 - 1 if i % 2 else i - 1 for i in range(t)]] * n, dtype=torch.int32)
        parents[:, 0] = -1
    strange = [(0, 0), (1, 0), (2, min(3, t - 1))] + ([(0, 4), (1, 33), (2, 35)] if t > 33 else [])
    for i, (row, node) in enumerate(strange):
        k[row, node, 0, (5, 61)[i % 2]] = -math.inf if i % 3 == 2 else math.inf
    out = K.swa_tree4(q.to(DEV), k.to(DEV), v.to(DEV), c.to(DEV), positions.to(DEV), window,
                      None if parents is None else parents.to(DEV), sinks=sinks)[0].cpu()
    keys, vals = R.cache_values(c, hd)
    calm = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
    none = some = 0
    for i in range(n):
        up = [-1] if parents is None else parents[i].tolist()
        args = v[i].double(), keys[i], vals[i], int(positions[i]), window, sinks, up, t
        want, size, seen = R.tree(q[i].double(), k[i].double(), *args)
        score = R.tree(q[i].double(), calm[i].double(), *args)[2]  # of the keys that have a weight, and more
        bad = torch.isnan(want).any(-1)
        assert torch.isnan(out[i][bad]).all()
        within(out[i][~bad], want[~bad], attention_bound(score, size, want, hd, window + sinks + t, dt)[~bad])
        none, some = none + int(bad.sum()), some + int((~bad & ~torch.isfinite(seen)).sum())
    assert none and some


def whole_in_two_parts(g, n, hd):
    """n fp32 numbers, of either sign, that times the scale of head_dim ``hd`` are two bf16 parts and nothing more: what is left of
    the product behind the first has its own leading 8 bits alone.  Products are kept whole between the parts, or rounded."""
    scale = torch.tensor(hd ** -0.5, dtype=torch.float32) * torch.tensor(1.44269504088896340736, dtype=torch.float32)
    x = 0.5 + torch.rand(1 << 23, generator=g)
    rounded = x * scale
    first = (rounded.view(torch.int32) & -65536).view(torch.float32)
    rest = (x.double() * scale.double() - first.double()).float()
    fused, apart = x[rest.view(torch.int32) & 65535 == 0], x[(rounded - first).view(torch.int32) & 65535 == 0]
    half = n // 2
    assert len(fused) >= half and len(apart) >= n - half
    x = torch.cat([fused[:half], apart[:n - half]])[torch.randperm(n, generator=g)]
    return x * torch.where(torch.rand(n, generator=g) < 0.5, -1.0, 1.0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t", [2, 36])
def test_infinite_new_keys_where_a_part_of_q_is_zero(t, hd):
    """fp32 rows whose third part is 0 at the infinite element of node 0's key, which every node sees; full windows behind it."""
    g = gen(t + hd)
    window, heads, hkv = 50, 4, 2
    c = cache_of(g, 1, 1, hkv, window, 0, hd)[0]
    q, k, v = (normal(g, 1, t, h, hd) for h in (heads, hkv, hkv))
    q[..., 9] = whole_in_two_parts(g, t * heads, hd).view(1, t, heads)
    k[0, 0, :, 9] = math.inf
    out = K.swa_tree4(q.to(DEV), k.to(DEV), v.to(DEV), c.to(DEV), torch.tensor([80], device=DEV), window)[0].cpu()
    negative = q[0, ..., 9] < 0  # scores of -inf
    assert torch.isfinite(out[0][negative]).all() and torch.isnan(out[0][~negative]).all() and negative.any() and not negative.all()
    keys, vals = R.cache_values(c, hd)
    args = v[0].double(), keys[0], vals[0], 80, window, 0, list(range(-1, t - 1)), t
    want, size, _ = R.tree(q[0].double(), k[0].double(), *args)
    score = R.tree(q[0].double(), torch.where(torch.isfinite(k[0]), k[0], torch.zeros_like(k[0])).double(), *args)[2]
    within(out[0][negative], want[negative], attention_bound(score, size, want, hd, window + t, torch.float32)[negative])


@pytest.mark.parametrize("layers_inside", [False, True])
def test_caches_between_others(layers_inside):
    """Every other request of an odd number, every other layer: taken in and forked in place, what lies between left alone."""
    g = gen(6)
    window, sinks, hd, hkv, t = 40, 2, 64, 2, 9
    whole = cache_of(g, 5, 5, hkv, window, sinks, hd).to(DEV)
    if layers_inside:
        whole = whole.transpose(0, 1)
    k, v = (normal(g, 3, 3, t, hkv, hd).to(DEV) for _ in range(2))
    positions = torch.tensor([0, 5, 77], device=DEV)
    for pick in ((slice(None, None, 2), slice(None, None, 2)), (slice(0, 3), slice(None, None, 2)), (slice(None, None, 2), slice(2, 5))):
        got, at = whole.clone(memory_format=torch.preserve_format), positions.clone()
        view = got[pick]
        alone, alone_at = view.clone(memory_format=torch.contiguous_format), positions.clone()
        for c, p in ((view, at), (alone, alone_at)):
            K.kv_commit4(k, v, None, None, c, p, window, sinks, advance=True)
            K.kv_fork4(c, torch.tensor([2, 0, 1], dtype=torch.int32, device=DEV), p, window, sinks)
        assert torch.equal(view, alone) and torch.equal(at, alone_at)
        want = whole.clone()
        want[pick] = alone
        assert torch.equal(got, want)
        for a, b in zip(K.kv_values4(view, window, sinks), K.kv_values4(alone, window, sinks)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
