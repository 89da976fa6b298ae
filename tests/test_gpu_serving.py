"""The serving operators together, as a decoder uses them: attention with sinks in the model and over
the rings, sampled steps, drafted tokens verified and committed, requests forked.

Token sequences are compared exactly between ways that compute the same fp32 model (weights of
0.08 make the choices vary and keep them apart, as in test_gpu_decoder.py); the attention layer is compared
with a plain form in 64 bits.
"""
import math

import pytest
import torch

from serve_reference import rotate

pytestmark = pytest.mark.gpu
DEV = "cuda"
BASE = dict(vocab_size=256, d_model=128, n_layers=3, n_heads=2, n_kv_heads=1, d_ff_fast=192, chunk_size=16,
            sliding_window_size=24, max_seq_len=512)


def make(sinks=0, dtype=torch.float32, seed=0, slow_std=0.08):
    from utttcompanion_amd import uTTTConfig, uTTTModel
    torch.manual_seed(seed)
    model = uTTTModel(uTTTConfig(**BASE, attention_sinks=sinks)).eval()
    with torch.no_grad():
        for name, p in model.named_parameters():
            if p.dim() == 2 and "fast_weight_pool" not in name and "w_eta" not in name and "w_alpha" not in name:
                p.normal_(0, slow_std)
    model = model.to(DEV)
    if dtype != torch.float32:
        model.to(dtype)
        model.fast_weight_pool.float()
    g = torch.Generator().manual_seed(seed + 1)
    states = []
    for _ in range(4):
        st = model.init_fast_state(1, device=DEV, dtype=torch.float32, detach=True)
        for name in ("w_up", "w_gate", "w_down"):
            t = getattr(st, name)
            t.add_(0.05 * torch.randn(t.shape, generator=g).to(DEV))
        states.append(st)
    prompts = [torch.randint(6, BASE["vocab_size"], (n,), generator=g) for n in (2, 17, 30, 61)]
    return model, states, prompts


def decoder(model, states, prompts):
    from utttcompanion_amd.decoder import BatchedDecoder
    dec = BatchedDecoder(model, states)
    return dec, dec.prefill(prompts)


@pytest.mark.parametrize("sinks", [0, 1, 5])
@pytest.mark.parametrize("cuts", [(50,), (1, 2, 3, 4, 40), (25, 1, 24), (29, 1, 1, 19), (4, 46)])
def test_attention_layer_with_sinks_against_the_plain_form(sinks, cuts):
    """A sequence given in pieces through the layer's own caches.  The bound, u = 2^-24: sums of D products give
    q, k and v within D u of their sums of absolute products, a rotation adds two such terms, the scores
    then differ by at most d = (4 D + hd + 8) u A, A the largest score of absolute values, so the weights
    by 2 d relatively; weighted sums and the output product add (keys + hd + 2 D) u of theirs."""
    from utttcompanion_amd.layer import SlidingWindowAttention
    torch.manual_seed(7)
    dim, heads, hkv, win, seq = 128, 2, 1, 24, sum(cuts)
    attn = SlidingWindowAttention(dim, heads, hkv, win, max_seq_len=128, sinks=sinks).eval().to(DEV)
    x = torch.randn(2, seq, dim)
    with torch.no_grad():
        got, cache, at = [], None, 0
        for n in cuts:
            y, cache = attn(x[:, at:at + n].to(DEV), kv_cache=cache, start_pos=at)
            at += n
            got.append(y.cpu())
            assert cache[0].shape == (2, hkv, min(at, sinks + win), dim // heads)
    got = torch.cat(got, 1).double()
    hd, u = dim // heads, 2.0 ** -24
    cos, sin = (t.cpu().double() for t in attn.rope.tables(seq, torch.device(DEV)))
    xd = x.double()

    def heads_of(w, n, absolute=False):
        w = w.detach().cpu().double()
        y = (xd.abs() @ w.abs().T if absolute else xd @ w.T).view(2, seq, n, hd).transpose(1, 2)
        return y

    q, k, v = (heads_of(l.weight, n) for l, n in ((attn.wq, heads), (attn.wk, hkv), (attn.wv, hkv)))
    qa, ka, va = (heads_of(l.weight, n, True) for l, n in ((attn.wq, heads), (attn.wk, hkv), (attn.wv, hkv)))
    q, k = (rotate(t, cos[:seq], sin[:seq]) for t in (q, k))
    turn = lambda t: t + torch.cat((t[..., hd // 2:], t[..., :hd // 2]), -1)  # |cos|, |sin| <= 1
    i, j = torch.arange(seq)[:, None], torch.arange(seq)[None, :]
    seen = (j <= i) & ((i - j < win) | (j < sinks))
    w = torch.softmax((q @ k.transpose(-1, -2) / math.sqrt(hd)).masked_fill(~seen, -math.inf), -1)
    d = (4 * dim + hd + 8) * u * float((turn(qa) @ turn(ka).transpose(-1, -2)).max()) / math.sqrt(hd)
    att, weighted = w @ v, w @ va
    off = (2 * d + (seq + hd + 2 * dim) * u) * weighted
    wo = attn.wo.weight.detach().cpu().double()
    flat = lambda t: t.transpose(1, 2).reshape(2, seq, dim)
    want = flat(att) @ wo.T
    bound = flat(off + dim * u * att.abs()) @ wo.abs().T
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())
    # the cache: the first sinks and the last rows, which the next piece attends to
    rows = list(range(seq)) if seq <= sinks + win else list(range(sinks)) + list(range(seq - win, seq))
    bound_k = (4 * dim + 8) * u * turn(ka)[:, :, rows]
    assert bool(((cache[0].cpu().double() - k[:, :, rows]).abs() <= bound_k).all())
    assert bool(((cache[1].cpu().double() - v[:, :, rows]).abs() <= 2 * dim * u * va[:, :, rows]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_writing_prefill_with_sinks_in_two_parts_keeps_the_caches(dtype):
    """A prefill with writes cut at a chunk boundary gives what the whole gives: the same kernels over the same
    values, the attention's keys in other rows (other tiles, so other orders of its sums)."""
    model, states, _ = make(sinks=5, dtype=dtype, slow_std=0.02)
    ids = torch.randint(6, 256, (2, 96), generator=torch.Generator().manual_seed(3)).to(DEV)
    one = lambda: model.init_fast_state(2, device=DEV, dtype=torch.float32, detach=True)
    whole = model(ids, fast_state=one())
    first = model(ids[:, :48], fast_state=one())
    second = model(ids[:, 48:], fast_state=first.fast_state, kv_caches=first.kv_caches, start_pos=48)
    tol = dict(atol=2e-4, rtol=2e-4) if dtype == torch.float32 else dict(atol=0.015, rtol=0.025)
    torch.testing.assert_close(second.logits, whole.logits[:, 48:], **tol)
    for a, b in zip(second.kv_caches, whole.kv_caches):
        assert a[0].shape == b[0].shape == (2, 1, 29, 64)
        torch.testing.assert_close(a[0], b[0], **tol)
        torch.testing.assert_close(a[1], b[1], **tol)


def test_a_window_past_the_sequence_makes_sinks_idle():
    from utttcompanion_amd import uTTTConfig, uTTTModel
    outs = []
    for sinks in (0, 4):
        torch.manual_seed(0)
        model = uTTTModel(uTTTConfig(**dict(BASE, sliding_window_size=128), attention_sinks=sinks)).eval().to(DEV)
        ids = torch.arange(6, 106).view(1, -1).to(DEV)
        outs.append(model(ids, update_fast_weights=False).logits)
    torch.testing.assert_close(outs[0], outs[1], atol=2e-4, rtol=2e-4)


@pytest.mark.parametrize("sinks", [1, 5])
def test_decoding_with_sinks_equals_per_request_generation(sinks):
    model, states, prompts = make(sinks)
    dec, first = decoder(model, states, prompts)
    tokens = dec.generate_greedy(first, 40).cpu()
    for i, (st, ids) in enumerate(zip(states, prompts)):
        want = list(model.stream_generate(ids.view(1, -1).to(DEV), st, max_new_tokens=40, temperature=0.0,
                                          eos_token_id=None))
        assert tokens[i, :len(want)].tolist() == want, f"request {i}"
    # the rings hand back what the eager caches hold, and take it in again
    caches = [dec.export_kv_caches(i) for i in range(4)]
    again, _ = decoder(model, states, prompts)
    again.reset(caches, dec.host_positions)
    assert torch.equal(again.k_rings, dec.k_rings) and torch.equal(again.v_rings, dec.v_rings)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_steps_with_sinks_and_sampling_equal_eager_steps(dtype):
    model, states, prompts = make(5, dtype)
    runs = []
    for captured in (False, True):
        dec, first = decoder(model, states, prompts)
        dec.set_sampling([0.0, 0.7, 1.0, 1.3], top_k=[0, 0, 20, 5], top_p=[1.0, 0.9, 0.8, 1.0], min_p=[0, 0, 0.05, 0],
                         generator=torch.Generator(DEV).manual_seed(11))
        if captured:
            dec.capture()
        tokens, logprobs = dec.generate_sampled(first, 20)
        dec.set_sampling(0.9, top_p=0.5, generator=torch.Generator(DEV).manual_seed(12))  # reaches the captured step
        assert (dec._graph is not None) == captured
        logits = dec.logits.clone()
        more, more_logprobs = dec.generate_sampled(logits, 10)
        runs.append((tokens, logprobs, more, more_logprobs, dec.positions.clone()))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    assert runs[0][4].tolist() == [len(p) + 28 for p in prompts]


def test_sampled_steps_give_the_probabilities_they_were_chosen_with():
    """Temperature alone: the log-probability is log_softmax(logits / T) of the choice, the left-out ids taken out
    first.  fp32 exponentials, 2^-42 steps of the masses and a logarithm: 2^-18 absolute covers them."""
    model, states, prompts = make()
    dec, first = decoder(model, states, prompts)
    dec.set_sampling(0.8, generator=torch.Generator(DEV).manual_seed(5))
    dec.generate_sampled(first, 1)
    logits = first
    for step in range(12):
        x = logits.cpu().double()
        x[:, list(left_out())] = -math.inf
        want = torch.log_softmax(x / float(torch.tensor(0.8)), -1).gather(1, dec.tokens.cpu()[:, None])[:, 0]
        torch.testing.assert_close(dec.logprobs.cpu().double(), want, atol=2.0 ** -18, rtol=2.0 ** -18)
        logits = dec.step(dec.tokens).clone()
    dec.set_sampling(0.0)
    chosen = dec.generate_sampled(first, 1)[0]
    dec.set_sampling(None)
    assert torch.equal(chosen, dec.generate_greedy(first, 1))


def left_out():
    from utttcompanion_amd.model import BOS_ID, PAD_ID, UNK_ID
    return PAD_ID, BOS_ID, UNK_ID


def drafts(truth, given, i, rng, nodes):
    """A tree for request i: node 0 its next token, then a chain of what follows, some of it wrong, with wrong siblings
    put between.  Parents, tokens."""
    at = given
    tokens, parents, tip = [truth[i][at]], [-1], 0
    while len(tokens) < nodes:
        at += 1
        if rng.random() < 0.4:  # a wrong sibling
            tokens.append(6 + (truth[i][at] + 1) % 200)
            parents.append(tip)
            if len(tokens) == nodes:
                break
        wrong = rng.random() < 0.15
        tokens.append(6 + (truth[i][at] + 7) % 200 if wrong else truth[i][at])
        parents.append(tip)
        tip = len(tokens) - 1
    return tokens, parents


@pytest.mark.parametrize("nodes", [1, 7, 20])
@pytest.mark.parametrize("sinks", [0, 5])
def test_speculated_tokens_equal_single_steps(sinks, nodes):
    import random
    model, states, prompts = make(sinks)
    plain, first = decoder(model, states, prompts)
    truth = plain.generate_greedy(first, 100).tolist()
    dec, first = decoder(model, states, prompts)
    have = [[t[0]] for t in truth]
    rng, taken = random.Random(nodes), 0
    for round_ in range(30):
        if max(map(len, have)) > 70:
            break
        trees = [drafts(truth, len(have[i]) - 1, i, rng, nodes if i else max(1, nodes - 3)) for i in range(4)]
        counts = torch.tensor([len(t) for t, _ in trees], dtype=torch.int32)
        pad = lambda row, value: row + [value] * (nodes - len(row))
        tokens = torch.tensor([pad(t, 0) for t, _ in trees])
        parents = torch.tensor([pad(p, -1) for _, p in trees], dtype=torch.int32)
        chain = nodes == 1
        got = dec.speculate_greedy(tokens.to(DEV), None if chain else parents, None if chain else counts.to(DEV))
        for i, new in enumerate(got):
            have[i] += new
            taken += len(new) - 1
            assert have[i] == truth[i][:len(have[i])], (round_, i)
        assert dec.positions.tolist() == dec.host_positions
        assert dec.tokens.tolist() == [h[-1] for h in have]
    assert nodes == 1 or taken > 20
    # single steps go on from there
    for _ in range(5):
        dec.step(dec.tokens)
        for i, t in enumerate(dec.tokens.tolist()):
            have[i].append(t)
            assert t == truth[i][len(have[i]) - 1]


def test_of_equal_siblings_the_longer_way_is_taken():
    """Two drafts that begin alike, the first of them ending at once."""
    model, states, prompts = make()
    plain, first = decoder(model, states, prompts)
    truth = plain.generate_greedy(first, 6).tolist()
    dec, _ = decoder(model, states, prompts)
    tokens = torch.tensor([[t[0], t[1], t[1], t[2], t[3]] for t in truth])
    new = dec.speculate_greedy(tokens, torch.tensor([[-1, 0, 0, 2, 3]] * 4))
    assert new == [t[1:5] for t in truth]
    assert dec.host_positions == [len(p) + 4 for p in prompts]


@pytest.mark.parametrize("chunk", [16, 80])
def test_ragged_writes_with_sinks_equal_single_ones(chunk):
    """Requests of several lengths in one chunk loop against each alone, through the layer chain and, for chunks past
    64 tokens, one update per layer (the bound of the same comparison without sinks)."""
    from utttcompanion_amd import uTTTConfig, uTTTModel
    torch.manual_seed(0)
    model = uTTTModel(uTTTConfig(**dict(BASE, chunk_size=chunk), attention_sinks=5)).eval().to(DEV)
    g = torch.Generator().manual_seed(1)
    turns = [torch.randint(6, 256, (n,), generator=g) for n in (200, 33, 90)]
    one = lambda: model.init_fast_state(1, device=DEV, dtype=torch.float32, detach=True)
    together = model.test_time_update_batched(turns, [one() for _ in turns])
    for ids, (state, surprise, _) in zip(turns, together):
        want, want_surprise, _ = model.test_time_update(ids.view(1, -1).to(DEV), one())
        assert abs(surprise - want_surprise) <= 1e-5 * max(1.0, abs(want_surprise))
        for name in ("w_up", "w_gate", "w_down", "s_up", "s_gate", "s_down"):
            a, b = getattr(state, name).double(), getattr(want, name).double()
            assert float((a - b).norm()) <= 1e-5 * float(b.norm()), name


def test_verified_logits_equal_steps_and_leave_the_requests_alone():
    model, states, prompts = make(5, torch.bfloat16, slow_std=0.02)
    dec, first = decoder(model, states, prompts)
    rings, at = dec.k_rings.clone(), dec.positions.clone()
    drafted = torch.randint(6, 256, (4, 6), generator=torch.Generator().manual_seed(2)).to(DEV)
    logits = dec.verify(drafted)
    assert torch.equal(rings, dec.k_rings) and torch.equal(at, dec.positions)
    for t in range(6):
        # the bound that holds between this decoder's bf16 steps and eager bf16 forwards
        torch.testing.assert_close(logits[:, t].float(), dec.step(drafted[:, t]).float(), atol=0.015, rtol=0.025)


def test_forked_requests_go_on_as_their_source():
    model, states, prompts = make(5)
    dec, first = decoder(model, states, prompts)
    dec.capture()
    dec.generate_greedy(first, 6)
    logits = dec.logits.clone()
    weights = dec.w_up.clone()
    rings, held = dec.k_rings.clone(), list(dec.host_positions)
    want = dec.generate_greedy(logits, 10)
    dec, first = decoder(model, states, prompts)
    dec.capture()
    dec.generate_greedy(first, 6)
    assert torch.equal(dec.logits, logits)
    src = [3, 1, 1, 2]
    dec.fork(src)
    assert torch.equal(dec.w_up, weights[src]) and dec.host_positions == [held[s] for s in src]
    for i, s in enumerate(src):
        used = min(held[s], 29)
        assert torch.equal(dec.k_rings[:, i, :, :used], rings[:, s, :, :used])
    assert torch.equal(dec.logits, logits[src])
    assert torch.equal(dec.generate_greedy(dec.logits, 10), want[src])
    dec.set_sampling(1.0)
    dec.generate_sampled(dec.logits, 2)
    chosen, weighed = dec.tokens.clone(), dec.logprobs.clone()
    dec.fork([0, 0, 3, 2])
    assert torch.equal(dec.tokens, chosen[[0, 0, 3, 2]]) and torch.equal(dec.logprobs, weighed[[0, 0, 3, 2]])
    assert dec.matches(model, [states[src[s]] for s in (0, 0, 3, 2)])


def test_decoder_refusals():
    model, states, prompts = make()
    dec, first = decoder(model, states, prompts)
    i64 = lambda *shape: torch.ones(shape, dtype=torch.int64, device=DEV)
    for bad in ([0, 1, 2], [0, 1, 2, 4], [-1, 0, 1, 2]):
        with pytest.raises(ValueError):
            dec.fork(bad)
    for kw in (dict(temperature=-1.0), dict(temperature=[1.0] * 3), dict(temperature=float("nan")),
               dict(temperature=1.0, top_p=0.0), dict(temperature=1.0, top_p=1.5), dict(temperature=1.0, top_k=-1),
               dict(temperature=1.0, min_p=2.0), dict(temperature=float("inf"))):
        with pytest.raises(ValueError):
            dec.set_sampling(**kw)
    with pytest.raises(ValueError):
        dec.generate_sampled(first, 2)
    with pytest.raises(ValueError):
        dec.commit(i64(4, 1), i64(4))  # nothing verified
    for tokens in (i64(4), i64(3, 2), i64(4, 0), i64(4, 65)):
        with pytest.raises(ValueError):
            dec.verify(tokens)
    with pytest.raises(ValueError):
        dec.speculate_greedy(i64(4, 3), torch.tensor([[-1, 0, 2]] * 4))
    for tokens in (i64(4), i64(3, 2), i64(4, 0)):
        with pytest.raises(ValueError):
            dec.speculate_greedy(tokens)
    dec.verify(i64(4, 3))
    for nodes, counts in ((i64(4, 2) * 3, i64(4)), (i64(4, 2), i64(4) * 3), (i64(4, 2), -i64(4)), (i64(3, 2), i64(3))):
        with pytest.raises(ValueError):
            dec.commit(nodes, counts)
    dec.commit(i64(4, 2) * 0, i64(4) * 0)  # an empty path is one
    with pytest.raises(ValueError):
        dec.commit(i64(4, 2) * 0, i64(4) * 0)  # once
    dec.verify(i64(4, 3))
    dec.step(i64(4))
    with pytest.raises(ValueError):
        dec.commit(i64(4, 1) * 0, i64(4))  # the requests moved on
    dec.set_sampling(1.0)
    with pytest.raises(ValueError):
        dec.generate_greedy(first, 2)
    dec.set_sampling(None)
    dec.generate_greedy(first, 2)
