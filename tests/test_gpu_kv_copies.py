"""``kernels.kv_commit`` and ``kernels.kv_fork`` against loops over requests: copies, so equal to the bit."""
import pytest
import torch

from serve_reference import slot_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = [torch.bfloat16, torch.float32]


def commit_reference(ring, nodes, path, counts, positions, window, sinks):
    want = ring.clone()
    for n, p in enumerate(positions):
        for a in range(max(0, min(counts[n], path.shape[1]))):
            x = int(path[n, a])
            if p >= 0 and 0 <= x < nodes.shape[2]:
                want[:, n, :, slot_of(p + a, sinks, window)] = nodes[:, n, x]
    return want


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("layers,n,t,path,hkv,hd,window,sinks,positions,counts", [
    (1, 1, 1, 1, 1, 64, 16, 0, [0], [1]),
    (2, 4, 5, 5, 2, 64, 24, 4, [0, 2, 25, 1000], [5, 3, 4, 0]),     # into the sinks, over the ring's end
    (3, 3, 8, 3, 1, 128, 7, 2, [0, 5, 100], [3, 2, 3]),
    (1, 3, 40, 40, 2, 64, 9, 3, [0, 1, 50], [40, 33, 12]),          # paths longer than the window: the last ones stay
    (12, 32, 16, 16, 4, 64, 512, 4, list(range(500, 532)), [i % 17 for i in range(32)]),
    (2, 3, 6, 4, 2, 8, 10, 1, [-3, 4, 5], [2, -1, 99]),             # counts out of range, a request that does not run
])
def test_commit(layers, n, t, path, hkv, hd, window, sinks, positions, counts, dtype):
    from utttcompanion_amd import kernels as K
    g = torch.Generator().manual_seed(t)
    slots = window + sinks
    rings = [torch.randn((layers, n, hkv, slots, hd), generator=g).to(dtype) for _ in range(2)]
    nodes = [torch.randn((layers, n, t, hkv, hd), generator=g).to(dtype) for _ in range(2)]
    order = torch.stack([torch.randperm(t, generator=g)[:path] for _ in range(n)]).to(torch.int32)
    want = [commit_reference(r, x, order, counts, positions, window, sinks) for r, x in zip(rings, nodes)]
    d = [r.to(DEV) for r in rings]
    pos = torch.tensor(positions, dtype=torch.int64, device=DEV)
    cnt = torch.tensor(counts, dtype=torch.int32, device=DEV)
    K.kv_commit(nodes[0].to(DEV), nodes[1].to(DEV), order.to(DEV), cnt, *d, pos, sinks=sinks)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(d, want)) and pos.tolist() == positions
    d = [r.to(DEV) for r in rings]
    K.kv_commit(nodes[0].to(DEV), nodes[1].to(DEV), order.to(DEV), cnt, *d, pos, sinks=sinks, advance=True)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(d, want))
    assert pos.tolist() == [p + max(0, min(c, path)) if p >= 0 else p for p, c in zip(positions, counts)]
    one = [r[0].to(DEV) for r in rings]  # one layer
    K.kv_commit(nodes[0][0].to(DEV), nodes[1][0].to(DEV), order.to(DEV), cnt, *one,
                torch.tensor(positions, dtype=torch.int64, device=DEV), sinks=sinks)
    assert all(torch.equal(a.cpu(), b[0]) for a, b in zip(one, want))


def test_commit_node_ids_out_of_range_and_strided_operands():
    from utttcompanion_amd import kernels as K
    g = torch.Generator().manual_seed(2)
    layers, n, t, hkv, hd, window, sinks = 2, 3, 4, 2, 64, 12, 2
    wide = [torch.randn((layers, 2 * n, hkv, window + sinks, hd), generator=g).bfloat16() for _ in range(2)]
    nodes = [torch.randn((layers, n, 2 * t, hkv, hd), generator=g).bfloat16()[:, :, :t] for _ in range(2)]
    order = torch.tensor([[0, -1, 3, 9], [4, 2, 1, 0], [3, 3, 3, 3]], dtype=torch.int32)
    counts, positions = [4, 4, 4], [1, 13, 40]
    d = [w.to(DEV) for w in wide]
    views = [x[:, ::2] for x in d]
    K.kv_commit(*(x.to(DEV) for x in nodes), order.to(DEV), torch.tensor(counts, dtype=torch.int32, device=DEV), *views,
                torch.tensor(positions, device=DEV), sinks=sinks)
    for got, had, x in zip(d, wide, nodes):
        want = had.clone()
        want[:, ::2] = commit_reference(had[:, ::2], x, order, counts, positions, window, sinks)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("layers,n,hkv,hd,slots", [(1, 1, 1, 64, 5), (2, 3, 2, 64, 20), (3, 5, 1, 128, 33), (2, 16, 4, 64, 68),
                                                   (1, 17, 2, 8, 9), (2, 32, 1, 64, 12), (1, 33, 2, 64, 9), (2, 64, 1, 64, 12), (1, 65, 2, 64, 11), (1, 128, 1, 64, 7)])
def test_fork_any_map(layers, n, hkv, hd, slots, dtype):
    from utttcompanion_amd import kernels as K
    g = torch.Generator().manual_seed(n)
    for kind in range(5):
        rings = [torch.randn((layers, n, hkv, slots, hd), generator=g).to(dtype) for _ in range(2)]
        pos = torch.randint(0, 3 * slots, (n,), generator=g)
        src = [torch.arange(n), torch.zeros(n), torch.arange(n).roll(1), torch.randint(0, n, (n,), generator=g),
               torch.randint(-2, n + 2, (n,), generator=g)][kind].to(torch.int32)
        want, wpos = [r.clone() for r in rings], pos.clone()
        for i, s in enumerate(src.tolist()):
            if s != i and 0 <= s < n:
                m = min(int(pos[s]), slots)
                for w, r in zip(want, rings):
                    w[:, i, :, :m] = r[:, s, :, :m]
                wpos[i] = pos[s]
        d, p = [r.to(DEV) for r in rings], pos.to(DEV)
        K.kv_fork(*d, src.to(DEV), p)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(d, want)) and torch.equal(p.cpu(), wpos), kind
        if layers == 1:
            d, p = [r[0].to(DEV) for r in rings], pos.to(DEV)
            K.kv_fork(*d, src.to(DEV), p)
            assert all(torch.equal(a.cpu(), b[0]) for a, b in zip(d, want)), kind


def test_fork_of_strided_requests_and_captured():
    from utttcompanion_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(5)
    wide = torch.randn((2, 3, 8, 2, 30, 64), generator=g, device=DEV)
    k, v = wide[0, :, ::2], wide[1, :, ::2]
    pos = torch.tensor([3, 30, 77, 0], device=DEV)
    src = torch.tensor([1, 2, 0, 1], dtype=torch.int32, device=DEV)
    K.kv_fork(k.clone(), v.clone(), src, pos.clone())  # loads the kernels
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.kv_fork(k, v, src, pos)
    for _ in range(3):
        before, p0 = wide.clone(), pos.clone()
        a, b, p = k.contiguous(), v.contiguous(), pos.clone()
        K.kv_fork(a, b, src, p)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, a) and torch.equal(v, b) and torch.equal(pos, p)
        assert torch.equal(wide[:, :, 1::2], before[:, :, 1::2])
        src.copy_(torch.randint(0, 4, (4,), generator=g, device=DEV))
