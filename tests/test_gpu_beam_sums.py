"""The sums behind beam search's scores where their errors are largest: rows whose mass lies far below their top, all of it at one
distance, whose roundings are one and the same."""
import math

import pytest
import torch

import decode_reference as R
from utttcompanion_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5000, 131072, 1 << 20])
def test_flat_rows(vocab, dt):
    rows = 8
    g = torch.Generator().manual_seed(vocab)
    x = torch.empty(rows, vocab)
    far = torch.linspace(1.0, math.log(vocab) + 2.0, rows) + 0.1 * torch.rand(rows, generator=g)
    x[:] = (2.0 - far)[:, None]
    x[:, 7] = 2.0
    x[:, vocab // 2] = 1.9  # the top moves within a row
    x = x.to(dt)
    scores = torch.randn(rows, generator=g)
    # one beam a group: nothing changes places, the scores are the sums'
    want = R.beams(x, scores, 1, None, (), None, -1, 0)
    tokens, sources, got, ended = K.beam_select(x.to(DEV), scores.to(DEV), 1)
    assert torch.equal(tokens.cpu(), want[0]) and torch.equal(sources.cpu().long(), want[1]) and not ended.any()
    d = torch.log(torch.tensor(float(vocab), dtype=torch.float64)) + 1
    # terms (2.25 d + 2), two sums moved (2 each), a part of sixteen (15), in half steps of fp32; then the score's own half step
    bound = 2.0 ** -24 * (2.25 * d + 2 + 4 + 15)
    assert ((got.cpu().double() - want[2]).abs() <= bound + 2.0 ** -24 * want[2].abs()).all()
