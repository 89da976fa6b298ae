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



@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [50001, 200001, 1 << 20])
def test_cuts_above_a_heavy_tail_are_the_definitions_at_any_alignment(vocab, dtype):
    """A cut among ids some 15 factors of two down, with as many ids below the first round's bins, whose masses make the
    bound: the same tokens and bits of the log-probabilities wherever the row starts in memory, and the cut of the definition.
    Weights are whole units of 2^-42, off by half a unit and 2^-42 of themselves, so masses of V ids are within V 2^-41 of
    exact: settings whose bound is nearer than that to an id's border, or whose uniform is to the token's, may take either
    side.  One id more or less moves a log-probability by 2^-15 / total; 2^-24 of it and the masses' V 2^-41 are allowed."""
    rows, room, temperature = 128, vocab * 2.0 ** -41, float(torch.tensor(1.3))
    g = torch.Generator().manual_seed(vocab)
    down = 0.2 * torch.rand(vocab, generator=g) + torch.where(torch.rand(vocab, generator=g) < 0.5, 15.3, 16.3)
    down[torch.rand(vocab, generator=g) < 0.2] = 45.0  # brings the row's mean down: the bins reach 16
    down[5] = 0.0
    x = (-temperature * math.log(2) * down).to(dtype).to(DEV)
    p = (0.3 + 0.5 * torch.rand(rows, generator=g)).float()
    if vocab < 100000:
        p = (0.6 + 0.2 * torch.rand(rows, generator=g)).float()
    u = torch.rand(rows, generator=g).float()
    runs = []
    for off in range(16 // x.element_size()):
        at = torch.empty(vocab + 8, dtype=dtype, device=DEV)[off:off + vocab]
        at.copy_(x)
        runs.append(call(at[None].expand(rows, -1), u.tolist(), [temperature] * rows, p=p.tolist()))
    tok, lp = (t.cpu() for t in runs[0])
    xs = x.cpu().double()
    order = torch.sort(xs, descending=True, stable=True).indices
    w = torch.exp((xs - xs.max()) / temperature)
    ahead = w[order].cumsum(0) - w[order]
    whole, sure, deep = float(w.sum()), 0, 0
    for r in range(rows):
        bound = float(p[r]) * whole
        if float((ahead - bound).abs().min()) <= room:
            continue
        kept = torch.zeros(vocab, dtype=torch.bool)
        kept[order[ahead <= bound]] = True
        below = torch.where(kept, w, 0.0).cumsum(0)
        total = float(below[-1])
        off = abs(float(lp[r]) - math.log(float(w[tok[r]]) / total))
        assert off <= 2.0 ** -24 * abs(float(lp[r])) + room, (r, off)
        want = int((below <= float(u[r]) * total).sum())
        if min(abs(float(below[want]) - float(u[r]) * total), abs(float(below[want] - w[want]) - float(u[r]) * total)) > room:
            assert int(tok[r]) == want, r
            sure, deep = sure + 1, deep + (1000 < int(kept.sum()) < vocab // 2)
    assert sure > rows // 2 and deep > rows // 2
    for off, (t, l) in enumerate(runs):
        assert t.tolist() == tok.tolist() and l.tolist() == lp.tolist(), off


@pytest.mark.parametrize("temperature", [2e37, 1e38, 3e38, math.inf])
def test_logits_further_apart_than_the_largest_number(temperature):
    """The differences of logits at both ends of the type do not fit it, and at such temperatures they weigh something."""
    from test_gpu_sampling import check, uniforms
    g = torch.Generator().manual_seed(21)
    x = 3.3e38 * (2 * torch.rand((4, 500), generator=g) - 1)
    x[1, ::3] = torch.finfo(torch.float32).min
    x[2, 100:] = -math.inf
    x[3] = 3.4e38 * torch.where(torch.rand(500, generator=g) < 0.5, 1.0, -1.0)
    x = x.to(DEV)
    for seed, kw in enumerate((dict(), dict(p=[0.3, 0.99, 0.7, 0.9]), dict(k=[400, 40, 3, 300]), dict(m=[0.01, 0.2, 0.0, 0.5]),
                               dict(k=[450, 7, 90, 400], p=[0.999, 0.9, 0.95, 0.8]))):
        check(x, uniforms(4, 40 + seed), [temperature] * 4, **kw)
