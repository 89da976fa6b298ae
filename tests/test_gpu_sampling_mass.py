"""``kernels.sample_select``: what the mass that top_p takes its share of is made of, where much of it lies far below the
largest logit."""
import math

import pytest
import torch

from test_gpu_sampling import call

pytestmark = pytest.mark.gpu
DEV = "cuda"


def heavy_tail(rows, vocab, dtype, seed):
    """One id on top, half of the others about 17 factors of two below it, the rest 40 below: of 131072 ids those 17 below
    hold a third of the mass, of 12000 a twentieth."""
    g = torch.Generator().manual_seed(seed)
    x = -17 * math.log(2) + 0.2 * torch.rand((rows, vocab), generator=g)
    x[:, 1::2] -= 23 * math.log(2)
    x[:, 5] = 0.0
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [12000, 131072])
def test_min_p_that_is_not_a_number_is_off(vocab, dtype):
    """The header's "<= 0 or NaN: all": the row's whole mass counts, not only what stands near the top."""
    n = 6
    x = heavy_tail(n, vocab, dtype, 3)
    x[3:] = 30 * x[3:]  # ordinary rows beside them: next to no mass below
    u, t, p = [0.1, 0.9, 0.995, 0.1, 0.5, 0.99], [1.0] * n, [0.8, 0.8, 0.98, 0.8, 0.9, 0.95]
    want, want_lp = call(x, u, t, p=p, m=[0.0] * n)
    for off in (math.nan, -1.0, -math.inf, -math.nan):
        got, lp = call(x, u, t, p=p, m=[off] * n)
        assert got.tolist() == want.tolist() and lp.tolist() == want_lp.tolist(), off
    assert int(want[2]) != 5  # the cut lies in the tail
    got, lp = call(x, u, t, k=[40000] * n, p=p, m=[math.nan] * n)
    want, want_lp = call(x, u, t, k=[40000] * n, p=p)
    assert got.tolist() == want.tolist() and lp.tolist() == want_lp.tolist()
