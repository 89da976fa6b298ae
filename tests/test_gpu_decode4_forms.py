"""Every form that the calls in 4 bits choose by size: products of many rows by many outputs, readouts of several tokens in every
division of their columns, attention with four waves to a workgroup and with many splits.  Bounds as in test_gpu_decode4."""
import functools

import pytest
import torch

import decode_reference as R
from test_gpu_decode4 import DEV, cache_of, check_tree, gen, linear_bound, normal, readout_reference, tables, within
from utttcompanion_amd import kernels as K

pytestmark = pytest.mark.gpu


@functools.lru_cache(maxsize=2)
def weight(n, k):
    p = K.pack_weight4(normal(gen(n + k), n, k))
    return p, R.weight_values(p.data, n, k)


def product(m, n, k, dt, norm, res):
    g = gen(m + n + k)
    x, r = normal(g, m, k, dtype=dt), normal(g, m, n, dtype=dt)
    p, w = weight(n, k)
    xd = x.double()
    want = (xd * (xd.pow(2).mean(1, keepdim=True) + norm).rsqrt() if norm else xd) @ w.T
    want = want + r.double() if res else want
    got = K.linear4(x.to(DEV), K.Weight4(p.data.to(DEV), n, k), residual=r.to(DEV) if res else None, x_eps=norm)
    within(got, want, linear_bound(xd, w, k, dt, norm, want, r.double() if res else None))


@pytest.mark.parametrize("norm,res", [(0.0, False), (1e-6, True)])
@pytest.mark.parametrize("n,k", [(3100, 190), (3100, 1029), (24600, 190), (24600, 1029)])
@pytest.mark.parametrize("m", [5, 18, 33, 64, 70])
def test_rows_that_share_x(m, n, k, norm, res):
    """Teams of two and of four waves, 16, 32 and 64 rows to a workgroup, more than one block of rows."""
    product(m, n, k, torch.bfloat16, norm, res)


@pytest.mark.parametrize("m,n,k", [(300, 3100, 190), (1000, 100, 77), (520, 40, 130)])
def test_hundreds_of_rows(m, n, k):
    """As a verified batch of trees brings them."""
    for dt in (torch.bfloat16, torch.float32):
        product(m, n, k, dt, 1e-6, True)


@pytest.mark.parametrize("m,n,k", [(20, 12300, 300), (70, 6200, 300), (8200, 20, 2048), (40, 8300, 2100)])
def test_rows_in_parts(m, n, k):
    """fp32: many outputs of few columns, more rows than columns are divided for, and columns divided among many outputs."""
    product(m, n, k, torch.float32, 1e-6, True)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,t,d,ff", [(32, 3, 768, 192), (32, 20, 768, 64), (2, 5, 64, 2048), (1, 40, 128, 2112), (2, 1, 128, 8192),
                                      (3, 6, 192, 8256)])
@pytest.mark.parametrize("norm,shared", [(True, True), (False, False)])
def test_readouts_of_every_division(b, t, d, ff, norm, shared, dt):
    """Many blocks of outputs, many columns, and single tokens whose hidden values do not fit beside each other."""
    g = gen(b + t + d + ff)
    x = normal(g, b, t, d, dtype=dt)
    nb = 1 if shared else b
    mats = [normal(g, nb, *s) / s[1] ** 0.5 for s in ((ff, d), (ff, d), (d, ff))]
    packed = [K.pack_weight4(w.to(DEV)) for w in mats]
    ln_w, ln_b = 1 + 0.1 * normal(g, d), 0.1 * normal(g, d)
    gain = (1 + 0.1 * normal(g, d)).to(dt)
    got = K.readout4(x.to(DEV), *packed, ln_w.to(DEV), ln_b.to(DEV), 1e-5, x_norm=(gain.to(DEV), 1e-6) if norm else None)
    values = [R.weight_values(p.data[0], p.n, p.k) for p in packed]
    for i in range(b) if shared else sorted({0, b // 2, b - 1}):
        if not shared and i:
            values = [R.weight_values(p.data[i], p.n, p.k) for p in packed]
        want, bound = readout_reference(x[i].double(), *values, ln_w.double(), ln_b.double(), gain.double() if norm else None, dt)
        within(got[i], want, bound)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,t,heads,hkv", [(70, 1, 8, 4), (66, 3, 4, 4), (30, 40, 4, 2)])
def test_many_requests(n, t, heads, hkv, hd, dt):
    """More than 256 workgroups, which have four waves each."""
    g = gen(n + t + hd)
    window, sinks = 70, 3
    positions = torch.randint(0, 300, (n,), generator=g)
    positions[:4] = torch.tensor([0, 1, sinks, sinks + window])
    c = cache_of(g, 1, n, hkv, window, sinks, hd)[0]
    q, k_new, v_new = (normal(g, n, t, h, hd, dtype=dt) for h in (heads, hkv, hkv))
    tab = tables(int(positions.max()) + t, hd)
    got = K.swa_tree4(q.to(DEV), k_new.to(DEV), v_new.to(DEV), c.to(DEV), positions.to(DEV), window, None, tab[0].to(DEV),
                      tab[1].to(DEV), sinks)
    check_tree(q, k_new, v_new, c, positions, window, sinks, hd, None, None, tab, got, dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t,window", [(1, 3300), (1, 4500), (6, 4500)])
def test_many_splits(t, window, hd, dt):
    """Five and seven splits, joined in two rounds: full caches, ones that leave splits empty, and a request out of range."""
    g = gen(t + window + hd)
    sinks, heads, hkv = 5, 4, 2
    positions = torch.tensor([window + 900, 10, -1, window // 2, 2 ** 33 + 7, 700])
    n = len(positions)
    assert K._tree4_workspace(n, heads, hkv, t, hd, window, sinks) == 4 * (window // 32 // 20) * n * heads * t * (hd + 2)
    c = cache_of(g, 1, n, hkv, window, sinks, hd)[0]
    q, k_new, v_new = (normal(g, n, t, h, hd, dtype=dt) for h in (heads, hkv, hkv))
    counts = torch.tensor([t, t, t, t, max(t - 2, 1), 0], dtype=torch.int32)
    for have in (None, counts):
        got = K.swa_tree4(q.to(DEV), k_new.to(DEV), v_new.to(DEV), c.to(DEV), positions.to(DEV), window, sinks=sinks,
                          counts=None if have is None else have.to(DEV))
        check_tree(q, k_new, v_new, c, positions, window, sinks, hd, None, have, None, got, dt)
