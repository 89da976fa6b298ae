"""``kernels.swa_tree`` where many rows share each tile of a workgroup (``k_swa_tree_wide``): rows that fill a group in part,
several groups, one split and more, ragged node counts, infinities and NaN, against the 64-bit definition."""
import os

import pytest
import torch

from serve_reference import tree_paths
from test_gpu_tree import check, make

DEV = "cuda"
# requests, nodes, query and kv heads, window, sinks, splits
CASES = [
    (19, 49, 8, 2, 300, 4, 1),    # 196 rows: seven of eight waves, the last one with 4 rows
    (15, 64, 10, 1, 300, 0, 1),   # 640 rows: three groups, the last of them half
    (16, 57, 10, 2, 2000, 3, 4),  # 285 rows: a second group of 29
    (32, 64, 4, 1, 500, 60, 2),   # 256 rows, all of one group; odd numbers of tiles
    (27, 33, 8, 2, 1100, 4, 4),   # 132 rows: three waves have none
]


@pytest.mark.parametrize("n,t,heads,hkv,window,sinks,splits", CASES)
def test_these_sizes_share_tiles(n, t, heads, hkv, window, sinks, splits):
    """The workspace tells the splits, and with a cache of any length these tell the workgroups: one per 256 rows of a
    request's kv head where tiles are shared, one per 32 (so that they fill the card by themselves) where not."""
    from utttcompanion_amd import _native as N
    from utttcompanion_amd import build
    if not os.path.exists(build.LIB_PATH):
        build.build()

    def splits_of(slots):
        nbytes = N.load_library().uttt_swa_tree_workspace(n, heads, hkv, t, 128, slots, N.DTYPE_BF16)
        return 1 if nbytes == 16 else nbytes // (4 * n * heads * t * 130)

    rows = heads // hkv * t
    assert n * hkv * -(-rows // 32) >= 256
    assert splits_of(1 << 20) == min(64, 256 // (n * hkv * -(-rows // 256))) > 1
    assert splits_of(window + sinks) == splits


def case(n, t, heads, hkv, window, sinks, seed):
    g = torch.Generator().manual_seed(seed)
    positions = torch.randint(0, 3 * window, (n,), generator=g).tolist()
    positions[:4] = [0, 1, window + sinks - 1, 2 * window + 77]
    return positions, *make(n, t, heads, hkv, 128, window, sinks, positions, torch.bfloat16, seed)


def args_of(pos, parents, cos, sin):
    return pos.to(DEV), parents.to(DEV), cos.to(DEV), sin.to(DEV)


def pick(some, *tensors):
    return [x[some] for x in tensors]


@pytest.mark.gpu
@pytest.mark.parametrize("n,t,heads,hkv,window,sinks,splits", CASES)
def test_all_and_some_nodes(n, t, heads, hkv, window, sinks, splits):
    from utttcompanion_amd import kernels as K
    positions, qkv, rings, pos, parents, (cos, sin) = case(n, t, heads, hkv, window, sinks, t)
    q, k, v = qkv.to(DEV).split([heads, hkv, hkv], dim=2)
    kr, vr = (r.to(DEV) for r in rings)
    some = list(range(5))  # the definition is slow: the edges, and a request of the others
    the = [positions[i] for i in some]
    full = K.swa_tree(q, k, v, kr, vr, *args_of(pos, parents, cos, sin), sinks=sinks)
    check(*pick(some, *full), qkv[some], pick(some, *rings), the, parents[some], cos, sin, heads, hkv, window, sinks)
    # a chain, without tables
    out = K.swa_tree(q, k, v, kr, vr, pos.to(DEV), sinks=sinks)
    check(*pick(some, *out), qkv[some], pick(some, *rings), the, None, cos, sin, heads, hkv, window, sinks, rotated=False)
    # ragged counts: rows behind them are neither read nor written
    g = torch.Generator().manual_seed(1)
    counts = torch.randint(0, t + 1, (n,), generator=g).tolist()
    counts[:5] = [1, t, 0, t - 1, t // 2]
    ragged, up = qkv.clone(), parents.clone()
    for i, c in enumerate(counts):
        ragged[i, c:] = float("nan")
        up[i, c:] = 99
    out = torch.full((n, t, heads, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    nodes = tuple(torch.full((n, t, hkv, 128), 4.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    K.swa_tree(*ragged.to(DEV).split([heads, hkv, hkv], dim=2), kr, vr, *args_of(pos, up, cos, sin), sinks=sinks, out=out,
               counts=torch.tensor(counts, dtype=torch.int32, device=DEV), node_outputs=nodes)
    check(*pick(some, out, *nodes), ragged[some], pick(some, *rings), the, up[some], cos, sin, heads, hkv, window, sinks,
          counts[:5])
    for i, c in enumerate(counts):
        assert bool((out[i, c:] == 3).all()) and bool((nodes[0][i, c:] == 4).all()) and bool((nodes[1][i, c:] == 4).all())
        assert not bool(out[i, :c].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("n,t,heads,hkv,window,sinks,splits", CASES)
def test_infinities_and_nan_stay_with_the_rows_that_see_them(n, t, heads, hkv, window, sinks, splits):
    """A branch of NaN among one request's nodes, values of infinity at the edge of another's window, and a request that
    cannot be computed: the rows that see none of it keep the definition's values, other requests their bits."""
    from utttcompanion_amd import kernels as K
    positions, qkv, rings, pos, parents, (cos, sin) = case(n, t, heads, hkv, window, sinks, t + 1)
    kr, vr = (r.to(DEV) for r in rings)
    parents[1] = torch.arange(t) - 1
    parents[1, 2] = 0  # node 1 is a leaf beside the chain 2, 3, ..
    run = lambda x, at, values: K.swa_tree(*x.to(DEV).split([heads, hkv, hkv], dim=2), kr, values,  # noqa: E731
                                           *args_of(at, parents, cos, sin), sinks=sinks)
    want = run(qkv, pos, vr)[0]
    assert not bool(want.isnan().any())
    odd = qkv.clone()
    odd[1, 1] = float("nan")
    got, kn, vn = run(odd, pos, vr)
    keep = [i for i in range(n) if i != 1]
    assert torch.equal(got[keep], want[keep]) and bool(got[1, 1].isnan().all())
    others = [i for i in range(t) if i != 1]
    finite = qkv[1:2, others]  # the tree without the leaf: the same keys, the leaf's rows left out
    up = torch.cat((torch.tensor([-1, 0]), torch.arange(1, t - 2)))[None].to(torch.int32)
    check(got[1:2, others], kn[1:2, others], vn[1:2, others], finite, pick([1], *rings), [positions[1]], up, cos, sin, heads, hkv,
          window, sinks)
    # the oldest token in the window of depth 0, seen by the roots alone
    p, held = positions[3], vr.clone()
    held[3, :, sinks + (p - window + 1 - sinks) % window] = float("inf")
    got, kn, vn = run(qkv, pos, held)
    keep = [i for i in range(n) if i != 3]
    assert torch.equal(got[keep], want[keep])
    deep = torch.tensor([len(x) - 1 for x in tree_paths(parents[3].tolist())]) > 0
    assert bool(got[3].float()[~deep].isinf().all()) and bool(got[3].float()[deep].isfinite().all())
    out = torch.where(deep[:, None, None].to(DEV), got[3], want[3])
    check(out[None], kn[3:4], vn[3:4], qkv[3:4], pick([3], *rings), [p], parents[3:4], cos, sin, heads, hkv, window, sinks)
    # requests out of range
    bad = pos.clone()
    bad[2], bad[0] = -1, len(cos)
    got = run(qkv, bad, vr)[0]
    keep = [i for i in range(n) if i not in (0, 2)]
    assert torch.equal(got[keep], want[keep]) and bool(got[0].isnan().all()) and bool(got[2].isnan().all())
