"""Products, readouts, caches and attention in 4 bits on the GPU against plain 64-bit restatements.

Tolerances count roundings: u = 2^-24 per fp32 operation of a sum's longest chain times the sum of magnitudes, a part that bf16
carries of an operand (2^-16 for two parts, nothing for three of fp32), 2^-8 for a weight of the softmax in bf16, and half a step of the result's type."""
import math

import pytest
import torch

import decode_reference as R
from utttcompanion_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative to the value


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype)


def within(got, want, bound):
    got, want = got.detach().double().cpu(), want.double()
    over = (got - want).abs() - bound
    assert not torch.isnan(got).any() and float(over.max()) <= 0, float(over.max())


# ---------------------------------------------------------------------------- weights and products
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (37, 150), (100, 31)])
def test_packed_weights(n, k):
    w = normal(gen(n), n, k)
    w[0, 0] = 0.0
    p = K.pack_weight4(w.to(DEV))
    padded = torch.zeros(n, -(-k // 32) * 32)
    padded[:, :k] = w
    assert torch.equal(R.weight_values(p.data, n, k), R.values(*R.fours(padded))[:, :k])
    assert torch.equal(K.pack_weight4(w).data, p.data.cpu())


def test_packed_weights_of_odd_values():
    w = torch.zeros(4, 64)
    w[0, 3], w[0, 40] = math.inf, 1.0
    w[1, 5] = math.nan
    w[2, :4] = torch.tensor([1e-41, -1e-41, 0.0, -0.0])
    w[3, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, -1.75, 2.5, -3.5, 5.0])  # every tie
    got = R.weight_values(K.pack_weight4(w.to(DEV)).data, 4, 64)
    assert torch.isnan(got[0, :32]).all() and torch.isnan(got[1, :32]).all()
    assert got[0, 40] == 6 * torch.tensor(1 / 6).bfloat16().double() and (got[2] == 0).all()
    assert got[3, :8].tolist() == [6.0, 0.0, 1.0, 1.0, -2.0, 2.0, -4.0, 4.0]


def linear_bound(x, w, k, dt, norm, want, residual):
    size = x.abs() @ w.abs().T
    rows = (x.pow(2).mean(1, keepdim=True) + norm).rsqrt() if norm else 1.0
    chain = 34 + k / 32 + 16 + (k / 32 + 40 if norm else 0)
    bound = chain * U * size * rows + STEP[dt] * want.abs() * (1 + 2 ** -7)
    return bound + (U * 2 * (want.abs() + residual.abs()) if residual is not None else 0)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 1280, 768), (3, 33, 100), (16, 16, 128), (17, 100, 1), (33, 5, 300), (64, 64, 64),
                                   (65, 48, 1000), (130, 31, 2049), (5, 4100, 96)])
@pytest.mark.parametrize("norm,res", [(0.0, False), (1e-6, True)])
def test_linear(m, n, k, dt, norm, res):
    g = gen(m + n + k)
    x, r = normal(g, m, k, dtype=dt), normal(g, m, n, dtype=dt)
    p = K.pack_weight4(normal(g, n, k).to(DEV))
    w, xd = R.weight_values(p.data, n, k), x.double()
    want = (xd * (xd.pow(2).mean(1, keepdim=True) + norm).rsqrt() if norm else xd) @ w.T
    if res:
        want = want + r.double()
    got = K.linear4(x.to(DEV), p, residual=r.to(DEV) if res else None, x_eps=norm)
    within(got, want, linear_bound(xd, w, k, dt, norm, want, r.double() if res else None))


@pytest.mark.parametrize("m,n,k", [(5, 100, 11000), (16, 64, 2048), (61, 199, 5501), (2, 1, 1921)])
def test_linear_whose_columns_are_divided(m, n, k):
    """Workgroups that share rows and columns of the result: eager, and replayed from a graph between other calls."""
    g = gen(m + n + k)
    x, r = normal(g, m, k), normal(g, m, n)
    p = K.pack_weight4(normal(g, n, k).to(DEV))
    w, xd = R.weight_values(p.data, n, k), x.double()
    want = (xd * (xd.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt()) @ w.T + r.double()
    xg, rg = x.to(DEV), r.to(DEV)
    eager = K.linear4(xg, p, residual=rg, x_eps=1e-6)
    within(eager, want, linear_bound(xd, w, k, torch.float32, 1e-6, want, r.double()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = K.linear4(xg, p, residual=rg, x_eps=1e-6)
        twice = K.linear4(xg, p, residual=held, x_eps=1e-6)
    then = K.linear4(xg, p, residual=eager, x_eps=1e-6)
    for _ in range(3):
        held.zero_(), twice.zero_()
        graph.replay()
        assert torch.equal(K.linear4(xg, p, residual=rg, x_eps=1e-6), eager)
        assert torch.equal(held, eager) and torch.equal(twice, then)


@pytest.mark.parametrize("n", [40, 3100, 24600])
@pytest.mark.parametrize("k", [1, 7, 8, 9, 20, 63, 65, 190, 532, 1029])
def test_linear_whose_last_columns_are_few(n, k):
    """Rows in bf16 whose last pieces are short, at few, many and very many outputs, between numbers that are not finite."""
    g = gen(n + k)
    m = 18
    wide = torch.full((m, k + 16), math.nan, dtype=torch.bfloat16)
    wide[:, 8:8 + k] = normal(g, m, k, dtype=torch.bfloat16)
    wide[3:5, 8 + k:] = math.inf
    x = wide.to(DEV)[:, 8:8 + k]
    p = K.pack_weight4(normal(g, n, k).to(DEV))
    w, xd = R.weight_values(p.data, n, k), x.double().cpu()
    want = xd @ w.T
    within(K.linear4(x, p), want, linear_bound(xd, w, k, torch.bfloat16, 0.0, want, None))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_linear_takes_any_rows(dt):
    """Views at odd offsets with wide rows, expanded rows, results into views, and onto the residual itself."""
    g = gen(5)
    m, n, k = 21, 50, 133
    base = normal(g, m, k + 40, dtype=dt).to(DEV)
    p = K.pack_weight4(normal(g, n, k).to(DEV))
    w = R.weight_values(p.data, n, k)
    for x in (base[:, 3:3 + k], base[:, 8:8 + k], base[:1, 1:1 + k].expand(m, k), base[:, :k].t().contiguous().t()):
        want = x.double().cpu() @ w.T
        wide = torch.full((m, n + 11), 7.0, dtype=dt, device=DEV)
        out = wide[:, 5:5 + n]
        assert K.linear4(x, p, out=out).data_ptr() == out.data_ptr()
        within(out, want, linear_bound(x.double().cpu(), w, k, dt, 0.0, want, None))
        assert (wide[:, :5] == 7).all() and (wide[:, 5 + n:] == 7).all()
        first = normal(g, m, n, dtype=dt)
        h = first.to(DEV)
        K.linear4(x, p, out=h, residual=h)
        within(h, want + first.double(), linear_bound(x.double().cpu(), w, k, dt, 0.0, want + first.double(), first.double()))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_linear_keeps_rows_apart(dt):
    """What is not finite stays in its row, and behind k nothing is read into the sums."""
    g = gen(6)
    m, n, k = 20, 40, 100
    wide = torch.full((m, 128), math.nan, dtype=dt)
    wide[:, :k] = normal(g, m, k, dtype=dt)
    p = K.pack_weight4(normal(g, n, k).to(DEV))
    x = wide.to(DEV)[:, :k]
    fine = K.linear4(x, p)
    assert torch.isfinite(fine).all()
    x[3, 7], x[17, 99] = math.nan, math.inf
    got = K.linear4(x, p)
    rest = [i for i in range(m) if i not in (3, 17)]
    assert torch.equal(got[rest], fine[rest]) and torch.isnan(got[3]).all() and not torch.isfinite(got[17]).all()
    assert K.linear4(x[:0], p).shape == (0, n)


def readout_reference(x, up, gate, down, ln_w, ln_b, gain, dt):
    """(out, bound) of one row's tokens in 64 bits; the bound follows the roundings through the products."""
    d, ff = x.shape[1], up.shape[0]
    carried = 2.0 ** -16 if dt is torch.bfloat16 else 2.0 ** -24
    e1 = (34 + d / 32 + 16 + 40) * U + (carried if gain is not None else 0)
    e2 = (34 + ff / 32 + 16) * U + carried
    if gain is not None:
        x = x * (x.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * gain
    u, g = x @ up.T, x @ gate.T
    du, dg = e1 * (x.abs() @ up.abs().T), e1 * (x.abs() @ gate.abs().T)
    act = g * torch.sigmoid(g)
    h = act * u
    dh = 1.1 * dg * u.abs() + act.abs() * du + 1.1 * dg * du + 8 * U * h.abs()
    z = h @ down.T
    dz = dh @ down.abs().T + e2 * (h.abs() @ down.abs().T)
    rs = (z.var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    y = (z - z.mean(1, keepdim=True)) * rs
    # an error of z moves its own element, the mean and the deviation
    rms = dz.pow(2).mean(1, keepdim=True).sqrt()
    dy = (dz + dz.mean(1, keepdim=True)) * rs + y.abs() * rms * rs + 32 * U * (1 + y.abs())
    out = x + y * ln_w + ln_b
    return out, dy * ln_w.abs() + 16 * U * (x.abs() + y.abs() + ln_b.abs()) + STEP[dt] * out.abs() * (1 + 2 ** -7)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,t,d,ff", [(1, 1, 64, 64), (3, 1, 768, 2048), (2, 5, 192, 320), (1, 17, 128, 256), (2, 70, 64, 128),
                                      (1, 1, 4096, 64)])
@pytest.mark.parametrize("norm,shared", [(True, False), (False, True)])
def test_readout(b, t, d, ff, norm, shared, dt):
    g = gen(b + t + d)
    x = normal(g, b, t, d, dtype=dt)
    nb = 1 if shared else b
    mats = [normal(g, nb, *s) / s[1] ** 0.5 for s in ((ff, d), (ff, d), (d, ff))]
    packed = [K.pack_weight4(w.to(DEV)) for w in mats]
    ln_w, ln_b = 1 + 0.1 * normal(g, d), 0.1 * normal(g, d)
    gain = (1 + 0.1 * normal(g, d)).to(dt)
    got = K.readout4(x.to(DEV), *packed, ln_w.to(DEV), ln_b.to(DEV), 1e-5, x_norm=(gain.to(DEV), 1e-6) if norm else None)
    for i in range(b):
        w = [R.weight_values(p.data[0 if shared else i], p.n, p.k) for p in packed]
        want, bound = readout_reference(x[i].double(), *w, ln_w.double(), ln_b.double(), gain.double() if norm else None, dt)
        within(got[i], want, bound)


def test_readout_views_and_workspace():
    g = gen(8)
    b, t, d, ff = 3, 2, 128, 192
    packed = [K.pack_weight4((normal(g, b, *s) / 12).to(DEV)) for s in ((ff, d), (ff, d), (d, ff))]
    ln = torch.ones(d, device=DEV), torch.zeros(d, device=DEV)
    wide = normal(g, b, t, 2 * d, dtype=torch.bfloat16).to(DEV)
    x = wide[..., d:]
    want = K.readout4(x.contiguous(), *packed, *ln)
    big = torch.full((b, t + 1, d + 3), 5.0, dtype=torch.bfloat16, device=DEV)
    ws = K.readout4_workspace(b, t, d, ff, x.device)
    got = K.readout4(x, *packed, *ln, out=big[:, 1:, 3:], workspace=ws)
    assert torch.equal(got, want) and (big[:, 0] == 5).all() and (big[..., :3] == 5).all()
    assert torch.equal(K.readout4(x, *packed, ln[0].bfloat16(), ln[1].bfloat16()), want)
    assert torch.equal(K.readout4(wide[:, :, 1:1 + d], *packed, *ln), K.readout4(wide[:, :, 1:1 + d].contiguous(), *packed, *ln))
    # a batch's matrices apart in memory
    far = [K.Weight4(torch.cat([p.data, p.data], 1)[:, :p.data.shape[1]], p.n, p.k) for p in packed]
    assert torch.equal(K.readout4(x, *far, *ln), want)
    assert K.readout4(x[:, :0], *packed, *ln).shape == (b, 0, d)


# ---------------------------------------------------------------------------- caches
def cache_of(g, layers, n, hkv, window, sinks, hd):
    """A cache with codes of all kinds, and its parts."""
    c = K.kv_cache4(layers, n, hkv, window=window, sinks=sinks, head_dim=hd, device=torch.device("cpu"))
    c.random_(0, 256, generator=g)
    scales = (0.1 + torch.rand(c.shape[:-1] + (2 * hd,), generator=g)).bfloat16()
    c[..., 32 * hd:] = scales.view(torch.uint8).view(*c.shape[:-1], 4 * hd)
    return c


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,sinks,hd", [(1, 0, 64), (33, 1, 64), (64, 32, 128), (100, 33, 128)])
def test_values(window, sinks, hd, dt):
    c = cache_of(gen(1), 2, 3, 2, window, sinks, hd)
    k, v = K.kv_values4(c.to(DEV), window, sinks, dt)
    front = -(-sinks // 32) * 32
    rows = list(range(sinks)) + list(range(front, front + window))
    for got, want in zip((k, v), R.cache_values(c, hd)):
        assert got.shape == (2, 3, 2, sinks + window, hd)
        assert torch.equal(got.cpu(), want[..., rows, :].to(dt))  # exact products, rounded once
    one = K.kv_values4(c[1].to(DEV), window, sinks, dt)
    assert torch.equal(one[0], k[1]) and torch.equal(one[1], v[1])


def commit_reference(c, k, v, nodes, counts, positions, window, sinks, hd):
    """(codes, scales) after the call."""
    codes, scales = R.cache_parts(c, hd)
    codes, scales = codes.flatten(-3, -2).clone(), scales.flatten(-3, -2).clone()
    for part, x in enumerate((k, v)):
        new_c, new_s = R.fours(x)
        for n in range(x.shape[1]):
            p = int(positions[n])
            path = list(range(x.shape[2])) if nodes is None else nodes[n].tolist()
            count = len(path) if counts is None else min(max(int(counts[n]), 0), len(path))
            last = {R.place(p + a, window, sinks): path[a] for a in range(count)} if p >= 0 else {}
            for slot, node in last.items():
                if 0 <= node < x.shape[2]:
                    codes[part, :, n, :, slot] = new_c[:, n, node]
                    scales[part, :, n, :, slot] = new_s[:, n, node]
    return codes, scales


def same_cache(got, codes, scales, hd):
    gc, gs = R.cache_parts(got, hd)
    assert torch.equal(gc.flatten(-3, -2), codes)
    assert torch.equal(gs.flatten(-3, -2).view(torch.int16), scales.view(torch.int16))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,sinks,hd,t", [(1, 0, 64, 3), (31, 1, 64, 40), (33, 32, 128, 5), (64, 33, 64, 1), (100, 40, 128, 250),
                                               (40, 0, 64, 39)])
def test_commit(window, sinks, hd, t, dt):
    """Paths of any order and length, wrapped, longer than the window, over the sinks' border; ids, counts and positions out of
    range; slots that no token takes keep every bit."""
    g = gen(window + t)
    layers, n, hkv = 2, 6, 2
    c = cache_of(g, layers, n, hkv, window, sinks, hd)
    k, v = normal(g, layers, n, t, hkv, hd, dtype=dt), normal(g, layers, n, t, hkv, hd, dtype=dt)
    k[0, 0, 0, 0, 3], v[0, 0, 0, 1, 40] = math.inf, math.nan
    k[1, 1], v[1, 1, :, :, :32] = 0.0, 1e-41
    nodes = torch.rand((n, t), generator=g).argsort(1).to(torch.int32)
    nodes[2, 0], nodes[3, -1] = -1, t
    counts = torch.tensor([t, t, t // 2, t, 0, t + 5], dtype=torch.int32)
    positions = torch.tensor([0, sinks, max(sinks - 3, 0), 5 * window + 17, 9, -1 if window > 60 else window - 1])
    got = c.to(DEV)
    pos = positions.to(DEV)
    K.kv_commit4(k.to(DEV), v.to(DEV), nodes.to(DEV), counts.to(DEV), got, pos, window, sinks)
    same_cache(got, *commit_reference(c, k, v, nodes, counts, positions, window, sinks, hd), hd)
    assert torch.equal(pos.cpu(), positions)
    # all nodes in order, a layer, positions advanced; rows of a wider projection
    got = c[0].to(DEV)
    wide = torch.cat([k[0], v[0]], dim=2).to(DEV)
    K.kv_commit4(wide[:, :, :hkv], wide[:, :, hkv:], None, None, got, pos, window, sinks, advance=True)
    same_cache(got[None], *commit_reference(c[:1], k[:1], v[:1], None, None, positions, window, sinks, hd), hd)
    assert torch.equal(pos.cpu(), torch.where(positions >= 0, positions + t, positions))


def test_commit_at_far_positions():
    g = gen(2)
    c = cache_of(g, 1, 2, 1, 50, 4, 64)
    k, v = normal(g, 1, 2, 7, 1, 64), normal(g, 1, 2, 7, 1, 64)
    positions = torch.tensor([2 ** 33 + 11, 2 ** 31 - 3])
    got = c.to(DEV)
    K.kv_commit4(k.to(DEV), v.to(DEV), None, None, got, positions.to(DEV), 50, 4)
    same_cache(got, *commit_reference(c, k, v, None, None, positions, 50, 4, 64), 64)


@pytest.mark.parametrize("n", [1, 5, 20, 40, 128])
def test_fork(n):
    g = gen(n)
    window, sinks, hd = 70, 33, 64
    c = cache_of(g, 2, n, 1, window, sinks, hd)
    positions = torch.randint(0, 200, (n,), generator=g)
    positions[0] = 0
    sources = torch.randint(-1, n + 1, (n,), generator=g).to(torch.int32)
    got, pos = c.to(DEV), positions.to(DEV)
    K.kv_fork4(got, sources.to(DEV), pos, window, sinks)
    before, after = R.cache_parts(c, hd), R.cache_parts(got, hd)
    for i in range(n):
        s = int(sources[i])
        s = s if 0 <= s < n else i
        assert int(pos[i]) == int(positions[s])
        slots = sorted({R.place(p, window, sinks) for p in range(int(positions[s]))})
        for a, b in zip(after, before):
            a, b = a.flatten(-3, -2), b.flatten(-3, -2)
            assert torch.equal(a[:, :, i][..., slots, :].to(torch.float32), b[:, :, s][..., slots, :].to(torch.float32))
    whole = c.to(DEV)
    K.kv_fork4(whole, sources.to(DEV), None, window, sinks)
    src = [int(s) if 0 <= int(s) < n else i for i, s in enumerate(sources)]
    assert torch.equal(whole.cpu(), c[:, src])


# ---------------------------------------------------------------------------- attention
def tables(length, hd):
    angle = torch.outer(torch.arange(length, dtype=torch.float64), 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd))
    return torch.cat([angle.cos()] * 2, 1).float(), torch.cat([angle.sin()] * 2, 1).float()


def check_tree(q, k_new, v_new, c, positions, window, sinks, hd, parents, counts, tab, got, dt):
    """Every request's output, keys and values against the definition; the keys that the outputs are held to are the returned ones."""
    out, kn, vn = (t.cpu() for t in got)
    n, t = q.shape[:2]
    keys, vals = R.cache_values(c, hd)
    for i in range(n):
        count = t if counts is None else min(max(int(counts[i]), 0), t)
        up = list(range(-1, t - 1)) if parents is None else parents[i].tolist()
        line = R.paths(up, count)
        pos = int(positions[i])
        bad = pos < 0 or line is None or (tab is not None and count and pos + max(len(p) for p in line) > tab[0].shape[0])
        assert (out[i, count:] == 0).all() and (kn[i, count:] == 0).all()
        if bad:
            assert torch.isnan(out[i, :count]).all()
            continue
        if not count:
            continue
        at = torch.tensor([pos + len(p) - 1 for p in line])
        qd, kd = q[i, :count].double(), k_new[i, :count].double()
        if tab is not None:
            cs, sn = tab[0][at].double()[:, None], tab[1][at].double()[:, None]
            lo, hi = kd.chunk(2, -1)
            turned = R.rotate(kd, cs, sn)
            mag = torch.cat([lo.abs() + hi.abs()] * 2, -1)
            within(kn[i, :count], turned, 3 * U * mag + STEP[dt] * (turned.abs() + 3 * U * mag))
            qd = R.rotate(qd, cs, sn)
        else:
            assert torch.equal(kn[i, :count], k_new[i, :count])
        assert torch.equal(vn[i, :count], v_new[i, :count])
        want, size, score = R.tree(qd, kn[i].double(), vn[i].double(), keys[i], vals[i], pos, window, sinks, up, count)
        carried = 2.0 ** -16 if dt is torch.bfloat16 else 2.0 ** -23
        ds = score * (carried + (34 + hd / 32 + 8) * U) + 4 * U * 40  # the exponent's own rounding at up to 2^5 below the top
        weight = 2.0 ** -8 if dt is torch.bfloat16 else 2.0 ** -23
        keys_seen = window + sinks + t
        chain = (34 + keys_seen / 32 + 80) * U
        rel = (2 * ds * (1 + ds)).unsqueeze(-1) + weight + 2 * chain + 8 * U
        within(out[i, :count], want[:count], rel[:count] * size[:count] + STEP[dt] * (want[:count].abs() * (1 + 2 ** -7)))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,heads,hkv", [(64, 3, 1), (64, 8, 2), (128, 16, 1), (128, 4, 4)])
@pytest.mark.parametrize("t,window,sinks", [(1, 40, 0), (1, 100, 33), (1, 1, 1), (5, 3, 2), (33, 64, 4), (64, 30, 40)])
def test_tree(t, window, sinks, hd, heads, hkv, dt):
    g = gen(t + window + heads)
    positions = torch.tensor([0, 1, sinks + 1, sinks + window, 3 * window + sinks + 5, 32])
    n = len(positions)
    c = cache_of(g, 1, n, hkv, window, sinks, hd)[0]
    qkv = normal(g, n, t, heads + 2 * hkv, hd, dtype=dt).to(DEV)
    q, k_new, v_new = qkv.split([heads, hkv, hkv], dim=2)
    tab = tables(int(positions.max()) + t, hd)
    parents = None
    if t > 1:
        parents = torch.tensor([[int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(t)] for _ in range(n)],
                               dtype=torch.int32)
    counts = torch.tensor([t, t, max(t // 2, 1), t, t, 0], dtype=torch.int32)
    args = (None if parents is None else parents.to(DEV), tab[0].to(DEV), tab[1].to(DEV), sinks)
    got = K.swa_tree4(q, k_new, v_new, c.to(DEV), positions.to(DEV), window, *args, counts.to(DEV))
    check_tree(q.cpu(), k_new.cpu(), v_new.cpu(), c, positions, window, sinks, hd, parents, counts, tab, got, dt)
    whole = K.swa_tree4(q, k_new, v_new, c.to(DEV), positions.to(DEV), window, *args)
    check_tree(q.cpu(), k_new.cpu(), v_new.cpu(), c, positions, window, sinks, hd, parents, None, tab, whole, dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_caches_are_split(hd, dt):
    """One request over many blocks: several workgroups a head, joined; a shared cache (stride 0); positions past 32 bits."""
    g = gen(hd)
    window, sinks, heads, hkv = 1500, 3, 4, 2
    c = cache_of(g, 1, 1, hkv, window, sinks, hd)[0]
    positions = torch.tensor([1400, 2 ** 33 + 5])
    q, k_new, v_new = (normal(g, 2, 3, h, hd, dtype=dt) for h in (heads, hkv, hkv))
    got = K.swa_tree4(q.to(DEV), k_new.to(DEV), v_new.to(DEV), c.to(DEV).expand(2, -1, -1, -1), positions.to(DEV), window, sinks=sinks)
    check_tree(q, k_new, v_new, c.expand(2, -1, -1, -1), positions, window, sinks, hd, None, None, None, got, dt)


@pytest.mark.parametrize("t", [1, 40])
def test_requests_out_of_range_are_nan(t):
    g = gen(t)
    window, sinks, hd = 50, 2, 64
    positions = torch.tensor([-1, 10, 10, 100 - t + 1, 100 - t])
    n = len(positions)
    c = cache_of(g, 1, n, 1, window, sinks, hd)[0]
    q, k_new, v_new = (normal(g, n, t, h, hd) for h in (2, 1, 1))
    parents = torch.arange(-1, t - 1, dtype=torch.int32).repeat(n, 1)
    parents[1, t - 1], parents[2, 0] = t - 1, -2
    tab = tables(100, hd)
    marks = [torch.full((n, t, 1, hd), 3.0, device=DEV) for _ in range(2)]
    got = K.swa_tree4(q.to(DEV), k_new.to(DEV), v_new.to(DEV), c.to(DEV), positions.to(DEV), window, parents.to(DEV),
                      tab[0].to(DEV), tab[1].to(DEV), sinks, node_outputs=marks)
    check_tree(q, k_new, v_new, c, positions, window, sinks, hd, parents, None, tab, got, torch.float32)
    assert all((m[:4] == 3).all() and (m[4] != 3).any() for m in marks)


@pytest.mark.parametrize("t", [1, 3])
def test_the_largest_positions(t):
    """Positions next to 2^63: past the tables where there are any; without them one like any other behind a full window."""
    g = gen(t)
    window, sinks, hd = 50, 2, 64
    c = cache_of(g, 1, 2, 1, window, sinks, hd)[0].to(DEV)
    q, k_new, v_new = (normal(g, 2, t, h, hd).to(DEV) for h in (2, 1, 1))
    far = torch.tensor([2 ** 63 - 1, 2 ** 63 - 2])
    cos, sin = (x.to(DEV) for x in tables(100, hd))
    assert torch.isnan(K.swa_tree4(q, k_new, v_new, c, far.to(DEV), window, None, cos, sin, sinks)[0]).all()
    alike = sinks + window * 4 + (far - sinks) % window  # the same slots, the same window
    got, want = (K.swa_tree4(q, k_new, v_new, c, p.to(DEV), window, sinks=sinks)[0] for p in (far, alike))
    assert torch.equal(got, want) and not torch.isnan(got).any()


def test_outputs_apart_from_inputs():
    g = gen(9)
    x = normal(g, 3, 64).to(DEV)
    p = K.pack_weight4(normal(g, 64, 64).to(DEV))
    with pytest.raises(ValueError, match="apart from x"):
        K.linear4(x, p, out=x)
    c = cache_of(g, 1, 1, 1, 32, 0, 64)[0].to(DEV)
    q, k, v = (normal(g, 1, 20, 1, 64).to(DEV) for _ in range(3))
    for nodes in ((k, v), (torch.empty_like(k), k), (v, torch.empty_like(k))):
        with pytest.raises(ValueError, match="apart from the new"):
            K.swa_tree4(q, k, v, c, torch.tensor([5], device=DEV), 32, node_outputs=nodes)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_what_a_query_does_not_see_may_be_anything(dt):
    """Scales that are NaN or infinite in slots without a visible token, infinities and NaN in nodes on other branches, rows
    behind the counts: nothing of it reaches a row that does not see it; one that does is not finite."""
    g = gen(4)
    window, sinks, hd, t = 70, 5, 64, 6
    positions = torch.tensor([30, 200])
    c = cache_of(g, 1, 2, 1, window, sinks, hd)[0]
    q, k_new, v_new = (normal(g, 2, t, h, hd, dtype=dt) for h in (3, 1, 1))
    parents = torch.tensor([[-1, 0, 0, 1, 2, 2]] * 2, dtype=torch.int32)
    counts = torch.tensor([6, 5], dtype=torch.int32)

    def run(c, k, v):
        return K.swa_tree4(q.to(DEV), k.to(DEV), v.to(DEV), c.to(DEV), positions.to(DEV), window, parents.to(DEV), sinks=sinks,
                           counts=counts.to(DEV))[0]

    fine = run(c, k_new, v_new)
    dirty, k2, v2 = c.clone(), k_new.clone(), v_new.clone()
    blocks = dirty[..., 32 * hd:].view(2, 1, -1, 2, 2, 4, 8, 2).view(torch.bfloat16)[..., 0]  # part, group, h, place
    nan = torch.tensor(math.nan, dtype=torch.bfloat16)
    for i, p in enumerate(positions.tolist()):
        held = {R.place(x, window, sinks) for x in range(p) if x < sinks or x >= p - window + 1}
        for slot in range(dirty.shape[2] * 32):
            if slot not in held:
                blocks[i, 0, slot // 32, :, :, slot % 16 // 4, slot % 32 // 16 * 4 + slot % 4] = nan if slot % 2 else math.inf
    k2[:, 3], v2[:, 3] = math.inf, math.nan  # a leaf: nodes 0, 1 lead to it, none follows
    v2[1, 5], k2[1, 5] = math.inf, math.nan  # behind the second request's nodes
    got = run(dirty, k2, v2)
    rest = [0, 1, 2, 4, 5]
    assert torch.equal(got[:, rest], fine[:, rest]) and torch.isnan(got[:, 3]).all()
    k3 = k_new.clone()
    k3[0, 0, 0, 0] = math.nan
    assert torch.isnan(run(c, k3, v_new)[0]).all() and torch.isfinite(run(c, k3, v_new)[1]).all()


def test_a_run_of_steps_sees_what_it_committed():
    """Attention, its token into the cache, the next step: as the definition on the values that the cache then holds."""
    g = gen(9)
    window, sinks, hd, heads, hkv, n = 40, 2, 64, 4, 2, 3
    c = K.kv_cache4(n, hkv, window=window, sinks=sinks, head_dim=hd, device=torch.device(DEV))
    tab = tables(120, hd)
    gtab = tab[0].to(DEV), tab[1].to(DEV)
    pos = torch.tensor([0, 37, 60], device=DEV)
    prompt_k, prompt_v = (normal(g, n, 60, hkv, hd, dtype=torch.bfloat16) for _ in range(2))
    start = torch.zeros(n, dtype=torch.int64, device=DEV)
    K.kv_commit4(prompt_k.to(DEV), prompt_v.to(DEV), None, pos.to(torch.int32), c, start, window, sinks, advance=True)
    assert torch.equal(start, pos)
    for _ in range(4):
        q, k_new, v_new = (normal(g, n, 1, h, hd, dtype=torch.bfloat16) for h in (heads, hkv, hkv))
        held, at = c.cpu(), pos.cpu()
        got = K.swa_tree4(q.to(DEV), k_new.to(DEV), v_new.to(DEV), c, pos, window, None, *gtab, sinks)
        check_tree(q, k_new, v_new, held, at, window, sinks, hd, None, None, tab, got, torch.bfloat16)
        K.kv_commit4(got[1], got[2], None, None, c, pos, window, sinks, advance=True)
        same_cache(c[None], *commit_reference(held[None], got[1].cpu()[None], got[2].cpu()[None], None, None, at, window, sinks, hd), hd)
        assert torch.equal(pos.cpu(), at + 1)


def test_captured_on_another_stream():
    """All calls of a step in one graph, replayed with other inputs between eager calls."""
    g = gen(10)
    window, sinks, hd, heads, hkv, n, d, ff = 64, 4, 64, 4, 2, 2, 256, 192
    c0 = cache_of(g, 1, n, hkv, window, sinks, hd).to(DEV)
    w = K.pack_weight4(normal(g, (heads + 2 * hkv) * hd, d).to(DEV) / 16)
    fast = [K.pack_weight4((normal(g, n, *s) / 14).to(DEV)) for s in ((ff, d), (ff, d), (d, ff))]
    ln = torch.ones(d, device=DEV), torch.zeros(d, device=DEV)
    x, c, pos = torch.zeros(n, d, dtype=torch.bfloat16, device=DEV), c0.clone(), torch.tensor([70, 9], device=DEV)

    def step():
        qkv = K.linear4(x, w, x_eps=1e-6).view(n, 1, -1, hd)
        q, k, v = qkv.split([heads, hkv, hkv], dim=2)
        out, kn, vn = K.swa_tree4(q, k, v, c[0], pos, window, sinks=sinks)
        K.kv_commit4(kn[None], vn[None], None, None, c, pos, window, sinks, advance=True)
        return out, K.readout4(x.view(n, 1, d), *fast, *ln)

    step()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = step()
    for i in range(4):
        x.copy_(normal(g, n, d))
        c.copy_(c0)
        pos.copy_(torch.tensor([70 + i, 9]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in (*held, c, pos)]
        c.copy_(c0)
        pos.copy_(torch.tensor([70 + i, 9]))
        again = step()
        for a, b in zip(kept, (*again, c, pos)):
            assert torch.equal(a, b)
