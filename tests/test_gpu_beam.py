"""Beam search's choice on the GPU against a plain 64-bit restatement: tokens, sources and ends equal, scores within the
half step of their type and the error of the exponentials' sum."""
import math

import pytest
import torch

import decode_reference as R
from utttcompanion_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check(logits, scores, beams, ended=None, banned=(0, 1, 3), limit=None, eos=2, pad=0, **kw):
    want = R.beams(logits.cpu(), scores.cpu(), beams, None if ended is None else ended.cpu(), banned, limit, eos, pad)
    got = K.beam_select(logits, scores, beams, ended=ended, banned=banned, active_limit=limit, eos=eos, pad=pad, **kw)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu().long(), want[1])
    assert torch.equal(got[3].cpu().long(), want[3])
    s, t = got[2].cpu().double(), want[2]
    fine = torch.isfinite(t)
    assert torch.equal(fine, torch.isfinite(s)) and (s[~fine] == -math.inf).all()
    # half a step of fp32, and 2^-22 of the sum: an exponential is off by a few units of 2^-24
    assert ((s - t).abs()[fine] <= 2.0 ** -24 * t.abs()[fine] + 2.0 ** -22).all()
    return got


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 300), (1, 4, 32000), (3, 2, 4097), (2, 32, 9001), (5, 7, 131), (1, 16, 70001),
                                                (2, 3, 1), (1, 8, 5)])
@pytest.mark.parametrize("over", [False, True])
def test_choice(groups, beams, vocab, over, dt):
    g = torch.Generator().manual_seed(groups + beams + vocab)
    rows = groups * beams
    logits = (3 * torch.randn(rows, vocab, generator=g)).to(dt).to(DEV)
    scores = (-20 + 2 * torch.randn(rows, generator=g)).to(DEV)
    ended = (torch.rand(rows, generator=g) < 0.3).to(torch.int32).to(DEV) if over else None
    check(logits, scores, beams, ended)
    check(logits, scores, beams, ended, limit=max(1, vocab * 2 // 3), banned=(), eos=None if vocab < 9 else 5, pad=vocab - 1)


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_rows_of_any_alignment(offset):
    g = torch.Generator().manual_seed(offset)
    wide = torch.randn(8, 5000, generator=g).bfloat16().to(DEV)
    scores = torch.randn(8, generator=g).to(DEV)
    check(wide[:, offset:offset + 4900], scores, 4)
    check(wide[:, offset:offset + 4900].float()[:, ::1], scores, 8)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [40, 5000, 20000])
def test_equal_logits(vocab, dt):
    """Of equal candidates the lower beam's, then the lower id: whole rows alike, -0 and 0, and beams with equal scores."""
    flat = torch.zeros(12, vocab, dtype=dt, device=DEV)
    flat[:, ::2] = -0.0
    check(flat, torch.zeros(12, device=DEV), 6)
    check(flat, -torch.arange(12, device=DEV).float() / 3, 12)
    few = torch.full((4, vocab), -2.0, dtype=dt, device=DEV)
    few[:, 7::9] = 1.0
    check(few, torch.zeros(4, device=DEV), 4)
    check(few, torch.zeros(4, device=DEV), 2, banned=(7, 16, 25))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("groups,beams,vocab", [(1, 32, 131072), (2, 32, 131072), (1, 20, 50000)])
def test_beams_of_unlike_scores(groups, beams, vocab, dt):
    """Many candidates of a few beams among the best: scores far apart, beams whose logits are alike, coarse logits."""
    g = torch.Generator().manual_seed(groups + beams + vocab)
    rows = groups * beams
    x = torch.randn(rows, vocab, generator=g)
    alike = x[:1].repeat(rows, 1)
    for logits in (x, alike, (4 * x).round() / 4):
        for spread in (0.01, 1.0, 8.0):
            scores = spread * torch.randn(rows, generator=g)
            check(logits.to(dt).to(DEV), scores.to(DEV), beams)


def test_rows_that_offer_nothing():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(8, 600, generator=g).to(DEV)
    scores = torch.randn(8, generator=g).to(DEV)
    x[0, 50], x[1, 60], x[2] = math.nan, math.inf, -math.inf
    x[3, 10:] = -math.inf
    check(x, scores, 4)
    check(x, scores, 8)
    scores[4], scores[5], scores[6] = math.nan, math.inf, -math.inf
    check(x, scores, 4, torch.tensor([1, 0, 0, 0, 1, 0, 1, 0], dtype=torch.int32, device=DEV))
    check(x, torch.full((8,), -math.inf, device=DEV), 8)
    check(x, scores, 2, limit=0)
    # the beams behind one prompt
    start = torch.full((8,), -math.inf, device=DEV)
    start[::4] = 0.0
    y = torch.randn(2, 600, generator=g).to(DEV).repeat_interleave(4, 0)
    tokens, sources, _, _ = check(y, start, 4)
    assert sources.tolist() == [0] * 4 + [4] * 4 and len(set(tokens[:4].tolist())) == 4


def test_in_place_and_captured():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(12, 3000, generator=g).bfloat16().to(DEV)
    scores, ended = torch.randn(12, generator=g).to(DEV), torch.zeros(12, dtype=torch.int32, device=DEV)
    ended[5] = 1
    out = (torch.zeros(12, dtype=torch.int64, device=DEV), torch.zeros(12, dtype=torch.int32, device=DEV), scores, ended)
    first_s, first_e = scores.clone(), ended.clone()
    want = check(x, first_s.clone(), 4, first_e.clone())
    call = lambda: K.beam_select(x, scores, 4, ended=ended, banned=(0, 1, 3), eos=2, out=out)  # noqa: E731
    assert call() is out and all(torch.equal(a, b) for a, b in zip(out, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        x.copy_(torch.randn(12, 3000, generator=g))
        scores.copy_(first_s)
        ended.copy_(first_e)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, check(x, first_s.clone(), 4, first_e.clone())))
