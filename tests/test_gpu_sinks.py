"""Sliding-window attention with sinks against the 64-bit definition: prompts (``swa_prefill(sinks=)``) and single tokens
over ring caches with sink slots (``swa_decode(sinks=)``)."""
import pytest
import torch

from serve_reference import attend_bound, rotate, slot_of, softmax_attend, tables, tree_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("b,heads,hkv,tq,hist,hd,window,sinks", [
    (1, 2, 1, 1, 0, 64, 16, 4),         # one token
    (1, 4, 4, 1, 33, 128, 16, 1),       # one token behind a history, one sink
    (2, 6, 2, 77, 0, 64, 24, 5),        # heads in threes
    (1, 8, 1, 130, 20, 64, 16, 64),     # more sinks than window; a sink tile that is full
    (1, 4, 2, 200, 7, 128, 50, 65),     # a second sink tile of one key
    (2, 4, 2, 300, 0, 64, 300, 9),      # a window as long as the prompt
    (1, 4, 1, 257, 63, 128, 64, 200),   # sinks in several tiles
    (3, 12, 4, 777, 515, 64, 512, 4),   # a follow-up turn on a full cache
    (1, 2, 1, 40, 0, 64, 8, 1000),      # all keys are sinks: plain causal attention
    (1, 4, 2, 96, 0, 64, 1, 2),         # a window of the token alone
    (4, 16, 4, 64, 1023, 128, 1024, 16),  # a chunk of a long prompt, few rows: splits
])
def test_prefill_with_sinks(b, heads, hkv, tq, hist, hd, window, sinks, dtype):
    from utttcompanion_amd import kernels as K
    g = torch.Generator().manual_seed(tq + hist)
    kv = hist + tq
    q = torch.randn((b, tq, heads, hd), generator=g).to(dtype).transpose(1, 2)
    k, v = (torch.randn((b, hkv, kv, hd), generator=g).to(dtype) for _ in range(2))
    out = K.swa_prefill(q.to(DEV), k.to(DEV), v.to(DEV), window, hist, sinks=sinks).cpu().double()
    i, j = hist + torch.arange(tq)[:, None], torch.arange(kv)[None]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    for n in range(b):
        for h in range(heads):
            want, weighted, pr = softmax_attend(q[n, h], k[n, h // (heads // hkv)], v[n, h // (heads // hkv)], seen)
            err = (out[n, h] - want).abs()
            bound = attend_bound(want, weighted, pr, dtype, hd, kv)
            assert bool((err <= bound).all()), (n, h, float((err / bound).max()))


@pytest.mark.parametrize("dtype", BOTH)
def test_prefill_sinks_zero_is_the_plain_call_and_strided_operands(dtype):
    from utttcompanion_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(3)
    kv = torch.randn((2, 150, 2, 3, 64), generator=g, device=DEV).to(dtype)  # keys and values of one buffer
    q = torch.randn((2, 4, 100, 64), generator=g, device=DEV).to(dtype)
    k, v = kv[:, :, :, 0].transpose(1, 2), kv[:, :, :, 2].transpose(1, 2)
    assert torch.equal(K.swa_prefill(q, k, v, 20, 50), K.swa_prefill(q, k, v, 20, 50, sinks=0))
    assert torch.equal(K.swa_prefill(q, k, v, 20, 50, sinks=7),
                       K.swa_prefill(q, k.contiguous(), v.contiguous(), 20, 50, sinks=7))
    # all keys sinks: the window does not matter
    assert torch.equal(K.swa_prefill(q, k, v, 200, 50), K.swa_prefill(q, k, v, 200, 50, sinks=3))


@pytest.mark.parametrize("dtype", BOTH)
def test_prefill_keys_between_sinks_and_window_do_not_matter(dtype):
    """NaN keys and values that no query may see, in tiles that hold nothing else visible."""
    from utttcompanion_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(4)
    q = torch.randn((1, 4, 64, 64), generator=g, device=DEV).to(dtype)
    k, v = (torch.randn((1, 2, 640, 64), generator=g, device=DEV).to(dtype) for _ in range(2))
    want = K.swa_prefill(q, k, v, 64, 576, sinks=64)
    for t in (k, v):
        t[:, :, 64:449] = float("nan")
    assert torch.equal(K.swa_prefill(q, k, v, 64, 576, sinks=64), want)


def decode_case(n, heads, hkv, hd, window, sinks, positions, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    slots = window + sinks
    qkv = torch.randn((n, heads + 2 * hkv, hd), generator=g).to(dtype)
    rings = [torch.randn((n, hkv, slots, hd), generator=g).to(dtype) for _ in range(2)]
    for i, p in enumerate(positions):  # unwritten slots hold anything
        for r in rings:
            r[i, :, min(p, slots):] = float("nan")
    return qkv, rings, torch.tensor(positions, dtype=torch.int64), tables(max(positions) + 2, hd)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,heads,hkv,hd,window,sinks,positions", [
    (1, 2, 1, 64, 16, 4, [0]),
    (6, 4, 2, 64, 24, 4, [0, 3, 4, 5, 27, 28]),          # around the sinks' end and the ring's
    (5, 8, 1, 128, 50, 1, [49, 50, 51, 52, 1000]),
    (3, 4, 4, 64, 512, 4, [515, 516, 2000]),
    (2, 16, 2, 128, 1, 2, [1, 77]),                      # a window of the token alone
    (4, 16, 4, 128, 1000, 60, [3, 999, 1060, 5000]),
    (2, 12, 4, 64, 4096, 4, [100, 9000]),                # long: splits
    (1, 8, 8, 64, 63, 64, [200]),
])
def test_decode_with_sinks(n, heads, hkv, hd, window, sinks, positions, dtype):
    from utttcompanion_amd import kernels as K
    qkv, (kr, vr), pos, (cos, sin) = decode_case(n, heads, hkv, hd, window, sinks, positions, dtype, n + window)
    q, k, v = qkv.split([heads, hkv, hkv], dim=1)
    dqkv, dk, dv = qkv.to(DEV), kr.to(DEV), vr.to(DEV)
    dq, dkn, dvn = dqkv.split([heads, hkv, hkv], dim=1)
    out = K.swa_decode(dq, dkn, dvn, dk, dv, pos.to(DEV), cos.to(DEV), sin.to(DEV), sinks=sinks).cpu()
    got_k, got_v = dk.cpu(), dv.cpu()
    for i, p in enumerate(positions):
        at = slot_of(p, sinks, window)
        turned = rotate(k[i], cos[p], sin[p])
        # the new key: rotated in fp32 (two products and a sum), rounded once
        room = (2.0 ** -8 if dtype == torch.bfloat16 else 0) * turned.abs() + 3 * 2.0 ** -24 * k[i].double().abs().amax() * 2
        assert bool(((got_k[i, :, at].double() - turned).abs() <= room).all())
        assert torch.equal(got_v[i, :, at], v[i])
        rest = torch.ones(window + sinks, dtype=torch.bool)
        rest[at] = False
        for got, had in ((got_k, kr), (got_v, vr)):
            assert torch.equal(got[i][:, rest].nan_to_num(nan=-7.0), had[i][:, rest].nan_to_num(nan=-7.0))
        want, weighted, pr = tree_attend(rotate(q[i], cos[p], sin[p])[None], got_k[i, None, :, at], v[i][None], kr[i], vr[i], p,
                                         [-1], window, sinks)
        err = (out[i].double() - want[0]).abs()
        bound = attend_bound(want[0], weighted[0], pr, dtype, hd, window + sinks)
        assert bool((err <= bound).all()), (i, p, float((err / bound).max()))


@pytest.mark.parametrize("dtype", BOTH)
def test_decode_steps_follow_the_prompt(dtype):
    """A prompt's attention with sinks equals its tokens one by one through the ring."""
    from utttcompanion_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(8)
    t, heads, hkv, hd, window, sinks = 90, 4, 2, 64, 20, 5
    q, k, v = (torch.randn((1, h, t, hd), generator=g, device=DEV).to(dtype) for h in (heads, hkv, hkv))
    want = K.swa_prefill(q, k, v, window, 0, sinks=sinks)
    kr, vr = (torch.full((1, hkv, window + sinks, hd), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    for i in range(t):
        out = K.swa_decode(q[:, :, i].contiguous(), k[:, :, i].contiguous(), v[:, :, i].contiguous(), kr, vr,
                           torch.tensor([i], device=DEV), sinks=sinks)
        err = (out.float() - want[:, :, i].float()).abs().max()
        # two computations of one output, each within half a step of weights and output of values up to about 4
        assert float(err) <= (4 * 4 * 2.0 ** -8 if dtype == torch.bfloat16 else 2e-5), i


def test_decode_positions_out_of_range_are_loud_and_write_nothing():
    from utttcompanion_amd import kernels as K
    dtype = torch.bfloat16
    qkv, (kr, vr), _, (cos, sin) = decode_case(3, 4, 2, 64, 16, 4, [30, 30, 30], dtype, 5)
    q, k, v = (t.to(DEV) for t in qkv.split([4, 2, 2], dim=1))
    for d, n in ((torch.bfloat16, 16), (torch.float32, 16), (torch.bfloat16, 4096)):
        kr2, vr2 = (torch.randn((3, 2, n + 4, 64), device=DEV).to(d) for _ in range(2))
        before = kr2.clone()
        pos = torch.tensor([-1, 12, len(cos)], device=DEV)
        out = K.swa_decode(q.to(d), k.to(d), v.to(d), kr2, vr2, pos, cos.to(DEV), sin.to(DEV), sinks=4)
        assert bool(out[0].isnan().all()) and bool(out[2].isnan().all()) and not bool(out[1].isnan().any())
        assert torch.equal(kr2[0], before[0]) and torch.equal(kr2[2], before[2])


def test_decode_captured_and_on_another_stream():
    from utttcompanion_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(21)
    n, heads, hkv, hd, window, sinks = 4, 8, 2, 64, 2048, 4
    q, k, v = (torch.randn((n, h, hd), generator=g, device=DEV).bfloat16() for h in (heads, hkv, hkv))
    kr, vr = (torch.randn((n, hkv, window + sinks, hd), generator=g, device=DEV).bfloat16() for _ in range(2))
    pos = torch.tensor([5, 900, 2052, 7000], device=DEV)
    cos, sin = (t.to(DEV) for t in tables(7100, hd))
    out = torch.empty_like(q)
    K.swa_decode(q, k, v, kr, vr, pos, cos, sin, out=out, sinks=sinks)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.swa_decode(q, k, v, kr, vr, pos, cos, sin, out=out, sinks=sinks)
    for step in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV).bfloat16())
        pos += 1
        a, b = kr.clone(), vr.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = K.swa_decode(q, k, v, a, b, pos, cos, sin, sinks=sinks)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kr, a) and torch.equal(vr, b), step
