"""``kernels.sample_select`` against the 64-bit definition: cuts by count and mass, ties, odd sizes and strides, rows whose
logits are not finite, captured calls."""
import math

import pytest
import torch

from serve_reference import sample_row

pytestmark = pytest.mark.gpu
DEV = "cuda"


def call(x, u, t, k=None, p=None, m=None, **kw):
    from utttcompanion_amd import kernels as K
    f = lambda v, dt: None if v is None else torch.tensor(v, dtype=dt, device=DEV)  # noqa: E731
    return K.sample_select(x, f(u, torch.float32), f(t, torch.float32), f(k, torch.int32), f(p, torch.float32),
                           f(m, torch.float32), **kw)


def check(x, u, t, k=None, p=None, m=None, banned=(), limit=None, sure=True):
    """Tokens equal the definition's and log-probabilities are within their rounding.  Weights are whole units of
    2^-42 of the largest one and off by half a unit and by 2^-42 of themselves, so mass sums over V ids are within
    V 2^-41 largest weights of exact: a u * total nearer than that to a border could take either side (``sure``:
    none is).  top_p's bound is a share of the whole mass, to which ids more than 16 factors of two down add by fp32
    exponentials, within 2^-36 of the largest weight each: no case here has its cut that near another id."""
    tok, lp = call(x, u, t, k, p, m, banned=banned, active_limit=limit)
    tok, lp, cpu = tok.cpu(), lp.cpu(), x.float().cpu()
    vocab = x.shape[1]
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    for r in range(x.shape[0]):
        want, wlp, near, kept = sample_row(cpu[r], f32(u[r]), f32(t[r]), 0 if k is None else k[r],
                                           1.0 if p is None else f32(p[r]), 0.0 if m is None else f32(m[r]), banned, limit)
        if near <= vocab * 2.0 ** -41:
            assert not sure, f"row {r}: the case sits on a border"
            assert kept is None or kept[tok[r]], r
            continue
        assert int(tok[r]) == want, f"row {r}: {int(tok[r])} for {want} (u {u[r]}, T {t[r]})"
        if math.isnan(wlp):
            assert math.isnan(float(lp[r])), r
        else:
            assert abs(float(lp[r]) - wlp) <= 2.0 ** -24 * abs(wlp) + vocab * 2.0 ** -41, (r, float(lp[r]), wlp)
    return tok, lp


def uniforms(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(n, generator=g).tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 63, 256, 1000, 4097, 32000])
def test_settings_of_every_row(vocab, dtype):
    rows = 24
    g = torch.Generator().manual_seed(vocab)
    x = (3 * torch.randn((rows, vocab), generator=g)).to(dtype).to(DEV)
    r = torch.rand((4, rows), generator=g)
    t = [0.0 if i % 7 == 3 else 0.3 + 1.5 * float(r[0, i]) for i in range(rows)]
    k = [0 if i % 3 == 0 else 1 + int(r[1, i] * min(vocab, 300)) for i in range(rows)]
    p = [1.0 if i % 4 == 0 else 0.05 + 0.94 * float(r[2, i]) for i in range(rows)]
    m = [0.0 if i % 2 == 0 else 0.2 * float(r[3, i]) for i in range(rows)]
    u = uniforms(rows, vocab + 1)
    check(x, u, t)
    check(x, u, t, k=k)
    check(x, u, t, p=p)
    check(x, u, t, m=m)
    check(x, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_banned_ids_limit_and_strides(dtype):
    rows, vocab = 6, 2051
    g = torch.Generator().manual_seed(5)
    wide = (3 * torch.randn((rows, vocab + 9), generator=g)).to(dtype).to(DEV)
    u, t = uniforms(rows, 6), [0.8] * rows
    for x in (wide[:, :vocab], wide[:, 1:vocab + 1], wide[::2, 3:vocab + 3]):
        n = x.shape[0]
        check(x, u[:n], t[:n], k=[40] * n, p=[0.9] * n, banned=(0, 1, 3, 70, 2000), limit=1777)
        check(x, u[:n], t[:n], banned=(0, 1, 3, 70, 2000), limit=64)
        check(x, u[:n], t[:n], limit=vocab + 5)
    # only one id left, and none
    one, lp = check(wide[:, :vocab], u, t, banned=(0,), limit=2)
    assert one.tolist() == [1] * rows and lp.tolist() == [0.0] * rows
    none, lp = call(wide[:, :vocab], u, t, banned=(0, 1), active_limit=2)
    assert none.tolist() == [0] * rows and bool(lp.isnan().all())
    none, lp = call(wide[:, :vocab], u, t, active_limit=0)
    assert none.tolist() == [0] * rows and bool(lp.isnan().all())


def test_one_row_for_several_samplers():
    g = torch.Generator().manual_seed(8)
    x = (3 * torch.randn((1, 4001), generator=g)).to(DEV)
    check(x.expand(5, -1), uniforms(5, 9), [0.0, 0.5, 0.9, 1.2, 1.2], k=[0, 0, 40, 0, 7], p=[0.9] * 5)


def test_equal_logits_share_the_mass_and_ties_go_to_the_lowest_ids():
    rows, vocab = 8, 1000
    x = torch.full((rows, vocab), -2.5, device=DEV)
    u = [0.0, 0.25, 0.4999, 0.5003, 0.75, 0.9001, 0.9901, 1 - 2.0 ** -24]
    t = [1.0] * rows
    tok, lp = call(x, u, t)
    assert tok.tolist() == [int(v * vocab) for v in u]
    assert torch.allclose(lp.cpu(), torch.full((rows,), -math.log(vocab)), atol=1e-6, rtol=0)
    tok, lp = call(x, u, t, k=[10] * rows)  # the first ten ids
    assert tok.tolist() == [int(v * 10) for v in u]
    tok, _ = call(x, u, t, p=[0.5] * rows)  # mass ahead <= 0.5: ids 0 .. 500
    assert tok.tolist() == [int(v * 501) for v in u]
    tok, _ = call(x, u, t, k=[10] * rows, p=[0.25] * rows)  # of ten: ahead 0, 0.1, 0.2
    assert tok.tolist() == [int(v * 3) for v in u]
    tok, _ = call(x, u, t, p=[0.0] * rows)
    assert tok.tolist() == [0] * rows
    # two values, the larger ones last: -0 and +0 are one value
    x = torch.zeros((rows, vocab), device=DEV)
    x[:, ::2] = -0.0
    x[:, 900:] = 1.0
    tok, _ = call(x, u, t, k=[101] * rows)  # ids 900 .. 999, then id 0
    w0 = math.exp(-1.0)
    want = [0 if v * (100 + w0) < w0 else 900 + int(v * (100 + w0) - w0) for v in u]
    assert tok.tolist() == want


def test_many_neighbouring_values_in_one_bin():
    """More ids than are ranked against each other inside one bin, all values distinct: the range of keys is divided."""
    vocab = 20000
    g = torch.Generator().manual_seed(9)
    x = (1.0 + 1e-3 * torch.rand((4, vocab), generator=g)).to(DEV)
    u, t = uniforms(4, 10), [1.0] * 4
    check(x, u, t, k=[1, 5000, 9999, 19999], sure=True)
    check(x, u, t, p=[0.1, 0.5, 0.77, 0.999], sure=True)
    check(x, u, t, k=[7000] * 4, p=[0.1, 0.5, 0.77, 0.999], sure=True)
    check(-x, u, t, k=[7000] * 4, p=[0.1, 0.5, 0.77, 0.999], sure=True)
    check(x * 1e-30, u, t, k=[7000, 1, 3, 19999], p=[0.1, 0.5, 0.77, 0.999], sure=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5000, 60000])
def test_few_and_many_ids_are_kept(vocab, dtype):
    """Cuts that keep few ids of the row, some thousands, and nearly all of it: flat and peaked rows, and rows whose
    kept ids stand in one place."""
    g = torch.Generator().manual_seed(vocab)
    rows = [s * torch.randn(vocab, generator=g) for s in (0.3, 1.0, 2.0, 4.0)]
    lump = torch.randn(vocab, generator=g) - 20
    lump[700:1900] += 20  # 1200 neighbours hold the mass
    x = torch.stack([*rows, lump, lump.flip(0)]).to(dtype).to(DEV)
    n = x.shape[0]
    for seed, (k, p) in enumerate([([0] * n, [0.02, 0.3, 0.9, 0.99, 0.9, 0.97]), ([3, 700, 2500, 4900, 1100, 1300], [1.0] * n),
                                   ([4000] * n, [0.9] * n), ([0] * n, [0.9999] * n)]):
        u = uniforms(n, 100 + seed)
        check(x, u, [0.9] * n, k, p)
        check(x, u, [1.0] * n, k, p, [0.001] * n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [4001, 70001])
def test_cuts_far_below_the_top(vocab, dtype):
    """A top_k among ids that weigh next to nothing, or nothing (more than 43 factors of two down), and a top_p near 1 of
    a row with one id far above the others, which hold most of the mass."""
    g = torch.Generator().manual_seed(vocab)
    x = (3 * torch.randn((5, vocab), generator=g)).to(dtype)
    x[2:, 17] = 30.0
    x = x.to(DEV)
    t = [0.3, 0.12, 2.5, 2.8, 3.0]
    for k, p in (([200, 900, 0, 0, 3000], None), ([200, 900, 0, 40, 3000], [0.7, 0.9, 0.995, 0.9999, 0.98]), (None, [0.9999, 0.5, 0.9, 0.99, 0.6])):
        check(x, uniforms(5, 31), t, k, p)


@pytest.mark.parametrize("temperature", [2e-5, 1e-3, 50.0, 1e4, math.inf])
def test_extreme_temperatures(temperature):
    g = torch.Generator().manual_seed(11)
    x = (4 * torch.randn((3, 3000), generator=g)).to(DEV)
    check(x, uniforms(3, 12), [temperature] * 3, k=[0, 100, 100], p=[0.9, 1.0, 0.9])


def test_rows_that_are_not_finite_take_the_greedy_choice():
    g = torch.Generator().manual_seed(13)
    x = torch.randn((7, 300), generator=g)
    x[0, 17] = math.nan
    x[1, [40, 9]] = math.inf
    x[2] = -math.inf
    x[3, 5:] = -math.inf  # some at -inf are ordinary: they have no mass
    x[4, 250] = math.nan  # out of use
    x[5] = torch.finfo(torch.float32).min
    x[6] = torch.finfo(torch.float32).min
    x[6, 77] = 0.0
    u = [0.5, 0.5, 0.5, 0.9, 0.3, 0.5, 0.7]
    tok, lp = call(x.to(DEV), u, [1.0] * 7, p=[0.9] * 7, active_limit=240)
    assert tok.tolist()[:3] == [17, 9, 0] and bool(lp[:3].isnan().all())
    assert 0 <= int(tok[3]) < 5 and not bool(lp[3:].isnan().any())
    assert int(tok[5]) == sample_row(x[5], 0.5, 1.0, top_p=float(torch.tensor(0.9)), limit=240)[0] and int(tok[6]) == 77
    tok, lp = call(x.to(DEV), u, [0.0] * 7, active_limit=240)
    from utttcompanion_amd import kernels as K
    assert torch.equal(tok, K.greedy_select(x.to(DEV), active_limit=240)) and lp.tolist() == [0.0] * 7


def test_settings_out_of_range():
    g = torch.Generator().manual_seed(15)
    x = torch.randn((5, 400), generator=g).to(DEV)
    u = uniforms(5, 16)
    plain, lp = call(x, u, [1.0] * 5)
    same, lp2 = call(x, u, [1.0] * 5, k=[0, -3, 400, 4000, 2 ** 31 - 1], p=[1.0, 1.5, math.nan, math.inf, 1.0],
                     m=[0.0, -1.0, math.nan, 0.0, -math.inf])
    assert torch.equal(plain, same) and torch.equal(lp, lp2)
    top = x.argmax(1)
    one, lp = call(x, u, [1.0] * 5, p=[0.0, -1.0, 1.0, 1.0, 1.0], m=[0.0, 0.0, 1.0, 7.0, math.inf])
    assert torch.equal(one, top) and lp.tolist() == [0.0] * 5
    cold, _ = call(x, u, [0.0, -1.0, math.nan, 1e-5, -math.inf])
    assert torch.equal(cold, top)
    edge, _ = call(x[:1].expand(4, -1).contiguous(), [math.nan, -1.0, 1.0, 5.0], [1.0] * 4)
    want = [call(x[:1], [v], [1.0])[0].item() for v in (0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24)]
    assert edge.tolist() == want


def test_large_vocabulary_rows_and_repeatability():
    g = torch.Generator(device=DEV).manual_seed(17)
    x = 3 * torch.randn((5, 131072 + 4), generator=g, device=DEV)
    u = uniforms(5, 18)
    t, k, p = [0.7, 1.0, 1.3, 1.0, 0.4], [0, 0, 200, 100000, 3], [0.9, 1.0, 0.95, 0.999, 0.5]
    tok, lp = check(x, u, t, k, p)
    for _ in range(3):
        again, lp2 = call(x, u, t, k, p)
        assert torch.equal(again.cpu(), tok) and torch.equal(lp2.cpu(), lp)
    big = torch.randn((1, 1 << 20), generator=g, device=DEV)
    check(big, [0.37], [1.0], [0], [0.5])


def test_outputs_given_advance_and_capture():
    from utttcompanion_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(19)
    rows = 9
    x = (3 * torch.randn((rows, 5000), generator=g, device=DEV)).bfloat16()
    u = torch.rand(rows, generator=g, device=DEV)
    t = torch.full((rows,), 0.9, device=DEV)
    p = torch.full((rows,), 0.9, device=DEV)
    out = torch.empty(rows, dtype=torch.int64, device=DEV)
    lp = torch.empty(rows, device=DEV)
    at = torch.arange(rows, dtype=torch.int64, device=DEV)
    got = K.sample_select(x, u, t, top_p=p, out=out, logprobs=lp, advance=at)
    assert got[0] is out and got[1] is lp and at.tolist() == list(range(1, rows + 1))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.sample_select(x, u, t, top_p=p, out=out, logprobs=lp, advance=at)
    for i in range(4):
        x.copy_((3 * torch.randn(x.shape, generator=g, device=DEV)).bfloat16())
        u.copy_(torch.rand(rows, generator=g, device=DEV))
        want, wlp = K.sample_select(x, u, t, top_p=p)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lp, wlp), i
    assert at.tolist() == list(range(5, rows + 5))


def test_distribution_over_many_draws():
    """Evenly spaced uniforms: an id's share is its probability to within the draw at each of its two borders."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5, 2.0, -3.0]])
    n = 40000
    u = ((torch.arange(n) + 0.5) / n).tolist()
    tok, _ = call(x.expand(n, -1).to(DEV).contiguous(), u, [1.0] * n, k=[5] * n)
    _, _, _, kept = sample_row(x[0], 0.5, 1.0, top_k=5)
    prob = torch.softmax(x[0].double().masked_fill(~kept, -math.inf), 0)
    share = torch.bincount(tok.cpu(), minlength=7).double() / n
    assert float((share - prob).abs().max()) <= 2.0 / n
