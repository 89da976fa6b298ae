"""``kernels.swa_tree`` against the 64-bit definition: trees and chains over ring caches, ragged node counts, windows shorter
than a path, strides, infinities and NaN where a node may not look."""
import pytest
import torch

from serve_reference import attend_bound, rotate, tables, tree_attend, tree_paths

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = [torch.bfloat16, torch.float32]


def trees(n, t, g, follow=0.6):
    i = torch.arange(t)
    anyone = (torch.rand((n, t), generator=g) * (i + 1)).floor().long().clamp(max=i) - 1
    return torch.where(torch.rand((n, t), generator=g) < follow, (i - 1).expand(n, t), anyone).to(torch.int32)


def make(n, t, heads, hkv, hd, window, sinks, positions, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    slots = window + sinks
    qkv = torch.randn((n, t, heads + 2 * hkv, hd), generator=g).to(dtype)
    rings = [torch.randn((n, hkv, slots, hd), generator=g).to(dtype) for _ in range(2)]
    for i, p in enumerate(positions):
        for r in rings:
            r[i, :, min(p, slots):] = float("nan")
    return qkv, rings, torch.tensor(positions, dtype=torch.int64), trees(n, t, g), tables(max(positions) + t + 1, hd)


def check(out, kn, vn, qkv, rings, positions, parents, cos, sin, heads, hkv, window, sinks, counts=None, rotated=True):
    dtype, hd = qkv.dtype, qkv.shape[-1]
    out, kn, vn = out.cpu(), kn.cpu(), vn.cpu()
    for i, p in enumerate(positions):
        t = qkv.shape[1] if counts is None else counts[i]
        if t == 0:
            continue
        q, k, v = qkv[i, :t].split([heads, hkv, hkv], dim=1)
        up = parents[i, :t].tolist() if parents is not None else list(range(-1, t - 1))
        at = p + torch.tensor([len(x) - 1 for x in tree_paths(up)])
        if rotated:
            turned_q = rotate(q, cos[at][:, None], sin[at][:, None])
            turned = rotate(k, cos[at][:, None], sin[at][:, None])
            # rotated in fp32 (two products and a sum), rounded once
            room = (2.0 ** -8 if dtype == torch.bfloat16 else 0) * turned.abs() + 6 * 2.0 ** -24 * k.double().abs().max()
            assert bool(((kn[i, :t].double() - turned).abs() <= room).all())
        else:
            turned_q = q
            assert torch.equal(kn[i, :t], k)
        assert torch.equal(vn[i, :t], v)
        want, weighted, pr = tree_attend(turned_q, kn[i, :t], v, rings[0][i], rings[1][i], p, up, window, sinks)
        err = (out[i, :t].double() - want).abs()
        bound = attend_bound(want, weighted, pr, dtype, hd, window + sinks + t)
        assert bool((err <= bound).all()), (i, p, float((err / bound).max()))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,t,heads,hkv,hd,window,sinks,positions", [
    (1, 1, 2, 1, 64, 16, 0, [0]),                      # one node, nothing cached
    (3, 5, 4, 2, 64, 24, 4, [0, 2, 30]),               # drafts that reach into and past the sinks
    (2, 8, 12, 4, 64, 512, 4, [515, 700]),
    (4, 7, 8, 1, 128, 50, 0, [0, 44, 50, 333]),
    (2, 64, 4, 1, 64, 30, 3, [10, 100]),               # paths longer than the window
    (2, 64, 16, 2, 128, 100, 0, [99, 1000]),
    (1, 33, 6, 2, 64, 1, 2, [50]),                     # a window of the node alone
    (1, 64, 8, 8, 128, 63, 64, [127]),
    (2, 16, 8, 2, 64, 4096, 4, [77, 12000]),           # long: splits
    (1, 13, 16, 4, 128, 3000, 1, [2999]),
])
def test_tree_matches_the_definition(n, t, heads, hkv, hd, window, sinks, positions, dtype):
    from utttcompanion_amd import kernels as K
    qkv, rings, pos, parents, (cos, sin) = make(n, t, heads, hkv, hd, window, sinks, positions, dtype, t + window)
    q, k, v = qkv.to(DEV).split([heads, hkv, hkv], dim=2)
    kr, vr = (r.to(DEV) for r in rings)
    before = kr.clone(), vr.clone()
    out, kn, vn = K.swa_tree(q, k, v, kr, vr, pos.to(DEV), parents.to(DEV), cos.to(DEV), sin.to(DEV), sinks=sinks)
    check(out, kn, vn, qkv, rings, positions, parents, cos, sin, heads, hkv, window, sinks)
    for a, b in zip((kr, vr), before):
        assert torch.equal(a.nan_to_num(nan=-7.0), b.nan_to_num(nan=-7.0))
    # without tables; a chain without parents
    out, kn, vn = K.swa_tree(q, k, v, kr, vr, pos.to(DEV), parents.to(DEV), sinks=sinks)
    check(out, kn, vn, qkv, rings, positions, parents, cos, sin, heads, hkv, window, sinks, rotated=False)
    out, kn, vn = K.swa_tree(q, k, v, kr, vr, pos.to(DEV), None, cos.to(DEV), sin.to(DEV), sinks=sinks)
    check(out, kn, vn, qkv, rings, positions, None, cos, sin, heads, hkv, window, sinks)


def wide_case(n, t, hd, seed):
    """Enough rows per key head and requests that the rows share a workgroup's tiles."""
    heads, hkv, window, sinks = 8, 2, 300, 4
    g = torch.Generator().manual_seed(seed)
    positions = torch.randint(0, 1000, (n,), generator=g).tolist()
    return (heads, hkv, window, sinks, positions, *make(n, t, heads, hkv, hd, window, sinks, positions, torch.bfloat16, seed))


@pytest.mark.parametrize("n,t,hd", [(43, 25, 64), (17, 64, 64), (40, 31, 128), (17, 49, 128)])
def test_many_rows_share_tiles(n, t, hd):
    from utttcompanion_amd import kernels as K
    heads, hkv, window, sinks, positions, qkv, rings, pos, parents, (cos, sin) = wide_case(n, t, hd, t)
    g = torch.Generator().manual_seed(1)
    counts = torch.randint(0, t + 1, (n,), generator=g).tolist()
    counts[0], counts[1] = t, 1
    q, k, v = qkv.to(DEV).split([heads, hkv, hkv], dim=2)
    kr, vr = (r.to(DEV) for r in rings)
    out, kn, vn = K.swa_tree(q, k, v, kr, vr, pos.to(DEV), parents.to(DEV), cos.to(DEV), sin.to(DEV), sinks=sinks,
                             counts=torch.tensor(counts, dtype=torch.int32, device=DEV))
    check(out, kn, vn, qkv, rings, positions, parents, cos, sin, heads, hkv, window, sinks, counts)
    # infinities and NaN in one branch of a request, and at the edge of another's window
    odd = qkv.clone()
    parents = parents.clone()
    parents[0] = torch.arange(t) - 1
    parents[0, 2] = 0  # node 1 is a leaf beside the chain 2, 3, ..
    odd[0, 1] = float("nan")
    args = (pos.to(DEV), parents.to(DEV), cos.to(DEV), sin.to(DEV))
    want = K.swa_tree(q, k, v, kr, vr, *args, sinks=sinks)[0]
    got = K.swa_tree(*odd.to(DEV).split([heads, hkv, hkv], dim=2), kr, vr, *args, sinks=sinks)[0]
    tol = 2.0 ** -6  # the same sums in another order, values up to about 4
    others = [i for i in range(t) if i != 1]
    assert float((got[0, others].float() - want[0, others].float()).abs().max()) <= tol
    assert bool(got[0, 1].isnan().all()) and torch.equal(got[1:], want[1:])
    full = next(i for i, p in enumerate(positions) if p > window + sinks)
    p = positions[full]
    vr[full, :, sinks + (p - window + 1 - sinks) % window] = float("inf")  # the oldest in the window of depth 0
    got = K.swa_tree(q, k, v, kr, vr, *args, sinks=sinks)[0]
    depth = torch.tensor([len(x) - 1 for x in tree_paths(parents[full].tolist())])
    deep = depth > 0
    assert float((got[full].float() - want[full].float())[deep].abs().max()) <= tol
    assert bool(got[full].float()[~deep].isinf().all())


def test_many_rows_split_over_slots():
    """The same with the slots of a request split over workgroups, and requests that cannot be computed."""
    from utttcompanion_amd import kernels as K
    n, t, heads, hkv, hd, window, sinks = 16, 64, 16, 4, 128, 2500, 4
    positions = [0, 5000, 100, 2503, 2504, 900] + [3000 + i for i in range(10)]
    qkv, rings, pos, parents, (cos, sin) = make(n, t, heads, hkv, hd, window, sinks, positions, torch.bfloat16, 7)
    q, k, v = qkv.to(DEV).split([heads, hkv, hkv], dim=2)
    kr, vr = (r.to(DEV) for r in rings)
    out, kn, vn = K.swa_tree(q, k, v, kr, vr, pos.to(DEV), parents.to(DEV), cos.to(DEV), sin.to(DEV), sinks=sinks)
    some = [0, 1, 3, 4]
    check(out[some], kn[some], vn[some], qkv[some], [r[some] for r in rings], [positions[i] for i in some], parents[some], cos,
          sin, heads, hkv, window, sinks)
    bad = pos.clone()
    bad[2], bad[7] = -1, len(cos)
    got = K.swa_tree(q, k, v, kr, vr, bad.to(DEV), parents.to(DEV), cos.to(DEV), sin.to(DEV), sinks=sinks)[0]
    assert bool(got[2].isnan().all()) and bool(got[7].isnan().all())
    keep = [i for i in range(n) if i not in (2, 7)]
    assert torch.equal(got[keep], out[keep])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hd,window", [(64, 40), (128, 40), (64, 3000)])
def test_ragged_node_counts_leave_the_rows_behind_alone(hd, window, dtype):
    from utttcompanion_amd import kernels as K
    n, t, heads, hkv, sinks = 5, 17, 8, 2, 3
    counts, positions = [17, 0, 1, 9, 30], [100, 7, 0, 45, 3]
    qkv, rings, pos, parents, (cos, sin) = make(n, t, heads, hkv, hd, window, sinks, positions, dtype, 3)
    for i, c in enumerate(counts):
        qkv[i, c:] = float("nan")
        parents[i, c:] = 99
    q, k, v = qkv.to(DEV).split([heads, hkv, hkv], dim=2)
    kr, vr = (r.to(DEV) for r in rings)
    out = torch.full((n, t, heads, hd), 3.0, dtype=dtype, device=DEV)
    nodes = tuple(torch.full((n, t, hkv, hd), 4.0, dtype=dtype, device=DEV) for _ in range(2))
    got = K.swa_tree(q, k, v, kr, vr, pos.to(DEV), parents.to(DEV), cos.to(DEV), sin.to(DEV), sinks=sinks,
                     counts=torch.tensor(counts, dtype=torch.int32, device=DEV), out=out, node_outputs=nodes)
    assert got[0] is out and got[1] is nodes[0] and got[2] is nodes[1]
    check(out, *nodes, qkv, rings, positions, parents, cos, sin, heads, hkv, window, sinks, [min(c, t) for c in counts])
    for i, c in enumerate(counts):
        assert bool((out[i, c:] == 3).all()) and bool((nodes[0][i, c:] == 4).all()) and bool((nodes[1][i, c:] == 4).all())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hd", [64, 128])
def test_infinities_and_nan_where_a_node_may_not_look(hd, dtype):
    """A branch that holds NaN, and cached values at the window's edge that only the shallow nodes see, change no
    other node's output."""
    from utttcompanion_amd import kernels as K
    n, t, heads, hkv, window, sinks = 1, 6, 4, 2, 70, 2
    for p in (60, 72, 200):
        qkv, rings, pos, _, (cos, sin) = make(n, t, heads, hkv, hd, window, sinks, [p], dtype, p)
        parents = torch.tensor([[-1, 0, 0, 2, 3, -1]], dtype=torch.int32)  # 1 and 5 are leaves beside 2, 3, 4
        args = [pos.to(DEV), parents.to(DEV), cos.to(DEV), sin.to(DEV)]
        run = lambda x, r: K.swa_tree(*x.to(DEV).split([heads, hkv, hkv], dim=2), *(y.to(DEV) for y in r), *args,  # noqa: E731
                                      sinks=sinks)[0]
        want = run(qkv, rings)
        assert not bool(want.isnan().any())
        odd = qkv.clone()
        odd[0, 1] = float("nan")
        odd[0, 5, heads:] = float("inf")
        got = run(odd, rings)
        tol = 2.0 ** -6 if dtype == torch.bfloat16 else 1e-5  # the same sums in another order, values up to about 4
        for i in (0, 2, 3, 4):
            assert float((got[0, i].float() - want[0, i].float()).abs().max()) <= tol, (p, i)
        assert bool(got[0, 1].isnan().all()) and bool(got[0, 5].isnan().any())
        if p >= 72:  # the oldest cached token in the window: seen at depth 0 (nodes 0 and 5) only
            rings2 = [r.clone() for r in rings]
            oldest = p - window + 1
            for r in rings2:
                r[0, :, sinks + (oldest - sinks) % window] = float("nan")
            got = run(qkv, rings2)
            for i in (1, 2, 3, 4):
                assert float((got[0, i].float() - want[0, i].float()).abs().max()) <= tol, (p, i)
            assert bool(got[0, 0].isnan().all()) and bool(got[0, 5].isnan().all())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("window", [48, 2048])
def test_requests_that_cannot_be_computed_are_loud(window, dtype):
    from utttcompanion_amd import kernels as K
    n, t, heads, hkv, hd, sinks = 6, 4, 4, 2, 64, 4
    qkv, rings, _, _, (cos, sin) = make(n, t, heads, hkv, hd, window, sinks, [30] * n, dtype, 5)
    end = len(cos)
    pos = torch.tensor([30, -1, end, end - 3, 30, 30], device=DEV)
    parents = torch.tensor([[-1, 0, 1, 2]] * n, dtype=torch.int32)
    parents[4, 2] = 2
    parents[5, 1] = -2
    q, k, v = qkv.to(DEV).split([heads, hkv, hkv], dim=2)
    nodes = tuple(torch.full((n, t, hkv, hd), 4.0, dtype=dtype, device=DEV) for _ in range(2))
    out, _, _ = K.swa_tree(q, k, v, *(r.to(DEV) for r in rings), pos, parents.to(DEV), cos.to(DEV), sin.to(DEV), sinks=sinks,
                           node_outputs=nodes)
    assert not bool(out[0].isnan().any())
    assert bool(out[1:].isnan().all())  # request 3: its deepest node lies past the tables
    assert bool((nodes[0][1:] == 4).all()) and bool((nodes[1][1:] == 4).all()) and not bool((nodes[0][0] == 4).any())


def test_one_node_equals_a_decode_step():
    from utttcompanion_amd import kernels as K
    for dtype in BOTH:
        qkv, rings, pos, _, (cos, sin) = make(4, 1, 8, 2, 64, 100, 4, [0, 50, 104, 1000], dtype, 6)
        q, k, v = qkv.to(DEV).split([8, 2, 2], dim=2)
        kr, vr = (r.to(DEV) for r in rings)
        tree, kn, vn = K.swa_tree(q, k, v, kr, vr, pos.to(DEV), None, cos.to(DEV), sin.to(DEV), sinks=4)
        step = K.swa_decode(q[:, 0], k[:, 0], v[:, 0], kr, vr, pos.to(DEV), cos.to(DEV), sin.to(DEV), sinks=4)
        assert torch.equal(tree[:, 0], step)
        for i, p in enumerate(pos.tolist()):
            at = p if p < 4 else 4 + (p - 4) % 100
            assert torch.equal(kr[i, :, at], kn[i, 0]) and torch.equal(vr[i, :, at], vn[i, 0])


def test_strides_streams_capture_and_repeatability():
    from utttcompanion_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(31)
    n, t, heads, hkv, hd, window, sinks = 3, 12, 8, 2, 128, 2000, 4
    big = torch.randn((n, 2 * t, heads + 3 * hkv, hd), generator=g, device=DEV).bfloat16()
    q, k, v = big[:, ::2, :heads], big[:, 1::2, heads:heads + hkv], big[:, ::2, heads + 2 * hkv:]
    rings = torch.randn((2, 2 * n, hkv, window + sinks, hd), generator=g, device=DEV).bfloat16()
    kr, vr = rings[0, ::2], rings[1, ::2]  # every other request of a larger cache
    pos = torch.tensor([3, 1500, 7000], device=DEV)
    parents = trees(n, t, torch.Generator().manual_seed(1)).to(DEV)
    cos, sin = (x.to(DEV) for x in tables(7100, hd))
    want = K.swa_tree(*(x.contiguous() for x in (q, k, v)), kr.contiguous(), vr.contiguous(), pos, parents, cos, sin, sinks=sinks)
    out = torch.empty((n, heads, t, hd), dtype=torch.bfloat16, device=DEV).transpose(1, 2)
    nodes = torch.empty_like(want[1]), torch.empty_like(want[2])
    ws = torch.empty(1 << 26, dtype=torch.uint8, device=DEV)
    call = lambda: K.swa_tree(q, k, v, kr, vr, pos, parents, cos, sin, sinks=sinks, out=out, node_outputs=nodes,  # noqa: E731
                              workspace=ws)
    call()
    assert all(torch.equal(a, b) for a, b in zip((out, *nodes), want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        big.copy_(torch.randn(big.shape, generator=g, device=DEV).bfloat16())
        pos += 7
        want = K.swa_tree(q, k, v, kr, vr, pos, parents, cos, sin, sinks=sinks)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, *nodes), want)), i
