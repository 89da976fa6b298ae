"""The decoder in 4 bits and its beam search: every part that it is made of, run together.

The bound of fp32 logits, 4e-5 of the largest: both sides are fp32 forms of the same model, each within 2e-5 of it (as the
decoder's other tests hold them), which differ in the order of their sums."""
import pytest
import torch

import decode_reference as R
from test_gpu_serving import DEV, make
from utttcompanion_amd import kernels as K

pytestmark = pytest.mark.gpu


def decoder(model, states, **kw):
    from utttcompanion_amd.decoder import BatchedDecoder
    return BatchedDecoder(model, states, **kw)


def near(a, b, tol=4e-5):
    a, b = a.double(), b.double()
    assert float((a - b).abs().max()) <= tol * float(b.abs().max()), float((a - b).abs().max() / b.abs().max())


def unpacked(w, norm=None):
    """A weight as 4 bits hold it, an RMSNorm's weight in its columns."""
    w = w.detach().float() if norm is None else w.detach().float() * norm.weight.detach().float()[None]
    return R.weight_values(K.pack_weight4(w).data, *w.shape).float().to(DEV)


def held_in_four(model, states):
    """The model and states whose fp32 weights are the values that the 4-bit decoder's codes stand for."""
    import copy
    m = copy.deepcopy(model)
    with torch.no_grad():
        for block in m.layers:
            a = block.attn
            for w in (a.wq, a.wk, a.wv):
                w.weight.copy_(unpacked(w.weight, block.attn_norm))
            a.wo.weight.copy_(unpacked(a.wo.weight))
            block.uttt.w_q.weight.copy_(unpacked(block.uttt.w_q.weight, block.uttt_norm))
            block.uttt.w_o.weight.copy_(unpacked(block.uttt.w_o.weight))
            block.attn_norm.weight.fill_(1.0)
            block.uttt_norm.weight.fill_(1.0)
        # the embeddings, which may be the same tensor, stay as they are
        m.lm_head.weight = torch.nn.Parameter(unpacked(m.lm_head.weight, m.norm))
        m.norm.weight.fill_(1.0)
        got = []
        for st in states:
            new = st.clone()
            for name in ("w_up", "w_gate", "w_down"):
                t = getattr(new, name)
                t.copy_(unpacked(t[0].t()).t()[None])
            got.append(new)
    return m, got


@pytest.mark.parametrize("sinks", [0, 5])
def test_weights_in_four_bits_are_the_model_of_their_values(sinks):
    """Steps, captured steps and verified trees against the 16-bit decoder of a model that holds the same values."""
    model, states, prompts = make(sinks)
    with torch.no_grad():
        for block in model.layers:
            block.attn_norm.weight.add_(0.1 * torch.randn_like(block.attn_norm.weight))
            block.uttt_norm.weight.add_(0.1 * torch.randn_like(block.uttt_norm.weight))
    same, same_states = held_in_four(model, states)
    a, b = decoder(model, states, weight_bits=4), decoder(same, same_states)
    b.prefill(prompts)
    caches = [b.export_kv_caches(i) for i in range(4)]
    a.reset(caches, [len(p) for p in prompts])
    tok = torch.tensor([7, 8, 9, 10], device=DEV)
    for i in range(6):
        near(a.step(tok), b.step(tok))
        tok = b.next_tokens.clone()
        if i == 2:
            a.capture()
    drafts = torch.randint(6, 256, (4, 5), generator=torch.Generator().manual_seed(1))
    up = torch.tensor([[-1, 0, 0, 1, 2]] * 4, dtype=torch.int32)
    near(a.verify(drafts, up), b.verify(drafts, up))
    # requests with other fast weights taken over
    a.fork([2, 1, 0, 0])
    b.fork([2, 1, 0, 0])
    near(a.step(tok), b.step(tok))


@pytest.mark.parametrize("sinks", [0, 5])
@pytest.mark.parametrize("captured", [False, True])
def test_caches_in_four_bits_are_rings_of_their_values(sinks, captured):
    """Against rings that hold, step by step, the values that the codes stand for: prompts, steps, trees, commits, forks."""
    model, states, prompts = make(sinks)
    a, b = decoder(model, states, cache_bits=4), decoder(model, states)

    def follow():
        k, v = K.kv_values4(a.cache4, a.window, a.sinks, torch.float32)
        b.k_rings.copy_(k)
        b.v_rings.copy_(v)

    assert torch.equal(a.prefill(prompts), b.prefill(prompts))
    for i in range(4):  # the prompt's rows, quantised where they lie
        for (k, v), (rk, rv) in zip(a.export_kv_caches(i), b.export_kv_caches(i)):
            for got, want in ((k, rk), (v, rv)):
                assert torch.equal(got.double().cpu(), R.values(*R.fours(want)))
    follow()
    tok = torch.tensor([7, 8, 9, 10], device=DEV)
    if captured:
        a.capture()
        b.capture()
    for _ in range(30):  # past the window
        near(a.step(tok), b.step(tok))
        follow()
        tok = b.next_tokens.clone()
    drafts = torch.randint(6, 256, (4, 6), generator=torch.Generator().manual_seed(2))
    up = torch.tensor([[-1, 0, 1, 0, 3, 4]] * 4, dtype=torch.int32)
    near(a.verify(drafts, up), b.verify(drafts, up))
    nodes, counts = torch.tensor([[0, 1, 2], [0, 3, 4], [0, 0, 0], [0, 1, 0]]), torch.tensor([3, 3, 1, 2])
    a.commit(nodes, counts)
    b.commit(nodes, counts)
    follow()
    assert torch.equal(a.positions, b.positions) and a.host_positions == b.host_positions
    near(a.step(tok), b.step(tok))
    follow()
    a.fork([1, 1, 3, 2])
    b.fork([1, 1, 3, 2])
    near(a.step(tok), b.step(tok))
    assert torch.equal(a.positions, b.positions)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_in_four_bits(dtype):
    """Weights and caches at once, eager and captured alike bit by bit, and started again."""
    model, states, prompts = make(3, dtype)
    a = decoder(model, states, weight_bits=4, cache_bits=4)
    first = a.prefill(prompts)
    eager = a.generate_greedy(first, 12)
    logits = a.logits.clone()
    assert torch.isfinite(logits).all()
    caches = decoder(model, states)
    caches.prefill(prompts)
    caches = [caches.export_kv_caches(i) for i in range(4)]
    a.reset(caches, [len(p) for p in prompts])
    a.capture()
    assert torch.equal(a.generate_greedy(first, 12), eager) and torch.equal(a.logits, logits)
    a.reset(caches, [len(p) for p in prompts])
    a.set_sampling(0.8, top_k=20, generator=torch.Generator(device=DEV).manual_seed(3))
    tokens, logprobs = a.generate_sampled(first, 6)
    assert tokens.shape == (4, 6) and (logprobs <= 0).all()


@pytest.mark.parametrize("captured", [False, True])
def test_weights_in_four_bits_follow_the_model(captured):
    """Weights and norms changed in place between steps, eager and captured, and verified trees between captured steps."""
    model, states, prompts = make(3, torch.float32)
    a = decoder(model, states, weight_bits=4)
    first = a.prefill(prompts)
    caches = [a.export_kv_caches(i) for i in range(4)]
    if captured:
        a.capture()
    a.step(first.argmax(-1))
    with torch.no_grad():
        block = model.layers[1]
        for w in (block.attn.wk.weight, block.attn.wo.weight, block.uttt.w_q.weight, block.uttt.w_o.weight, model.lm_head.weight):
            w.mul_(1.0 + 0.5 * torch.rand(w.shape, generator=torch.Generator().manual_seed(len(w))).to(DEV))
        block.attn_norm.weight.mul_(1.25)
        model.norm.weight.mul_(0.75)
    b = decoder(model, states, weight_bits=4)
    for dec in (a, b):
        dec.reset(caches, [len(p) for p in prompts])
    tokens = first.argmax(-1)
    for i in range(3):
        if i == 1:
            tree = tokens[:, None].repeat(1, 2)
            assert torch.equal(a.verify(tree), b.verify(tree))
        x, y = a.step(tokens).clone(), b.step(tokens).clone()
        assert torch.equal(x, y)
        tokens = y.argmax(-1)


def eager_beams(model, state, prompt, beams, steps, eos):
    """Beam search by whole forwards of every hypothesis."""
    limit = model.active_vocab_limit
    held, scores, ended = [[] for _ in range(beams)], [0.0] + [-float("inf")] * (beams - 1), [0] * beams
    for _ in range(steps):
        rows = []
        for h in held:
            ids = torch.cat([prompt, torch.tensor(h, dtype=torch.int64)]).view(1, -1).to(DEV)
            rows.append(model(ids, fast_state=state, update_fast_weights=False, logits_to_keep=1).logits[0, -1].cpu())
        logits = torch.stack(rows)
        t, s, scores, ended = R.beams(logits, torch.tensor(scores), beams, torch.tensor(ended), (0, 1, 3),
                                      limit if limit < logits.shape[1] else None, eos, 0)
        held = [held[i] + [int(x)] for x, i in zip(t, s)]
        scores, ended = scores.tolist(), ended.tolist()
    return torch.tensor(held), torch.tensor(scores)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("sinks", [0, 5])
def test_beam_search_is_that_of_whole_forwards(captured, sinks):
    """Two prompts with fast weights of their own, two beams each, past the window; some beams end."""
    model, states, prompts = make(sinks)
    g0, g1 = states[0], states[2]
    dec = decoder(model, [g0, g0, g1, g1])
    first = dec.prefill([prompts[1], prompts[0], prompts[2], prompts[0]])  # the second of each is taken over
    if captured:
        dec.capture()
    steps = 12
    greedy = [eager_beams(model, st, p, 2, 4, None)[0][0] for st, p in ((g0, prompts[1]), (g1, prompts[2]))]
    eos = int(greedy[0][2])  # a token that beams do take
    with torch.no_grad():
        want = [eager_beams(model, st, p, 2, steps, eos) for st, p in ((g0, prompts[1]), (g1, prompts[2]))]
    tokens, scores = dec.beam_search(first, 2, steps, eos)
    for i, (t, s) in enumerate(want):
        assert torch.equal(tokens[i].cpu(), t)
        assert float((scores[i].cpu().double() - s).abs().max()) <= 1e-4 * steps
    assert any(eos in t.tolist()[0][:-1] or eos in t.tolist()[1][:-1] for t, _ in want)
    assert dec.host_positions == [len(prompts[1]) + steps - 1] * 2 + [len(prompts[2]) + steps - 1] * 2
    assert torch.equal(dec.tokens, tokens[:, :, -1].reshape(-1))
    # the requests go on as their beams
    after = dec.step(dec.tokens)
    with torch.no_grad():
        for r in range(4):
            ids = torch.cat([prompts[1] if r < 2 else prompts[2], tokens.view(4, -1)[r].cpu()]).view(1, -1).to(DEV)
            near(after[r], model(ids, fast_state=g0 if r < 2 else g1, update_fast_weights=False, logits_to_keep=1).logits[0, -1])


def test_beams_in_four_bits():
    """The whole of it at once: one beam is the greedy choice; eager and captured agree; more beams find no worse continuation."""
    model, states, prompts = make(2, torch.bfloat16)
    st = [states[0]] * 4
    dec = decoder(model, st, weight_bits=4, cache_bits=4)
    first = dec.prefill([prompts[2]] * 4)
    greedy = decoder(model, st[:1], weight_bits=4, cache_bits=4)
    want = greedy.generate_greedy(greedy.prefill([prompts[2]]), 10)
    one = decoder(model, st[:1], weight_bits=4, cache_bits=4)
    tokens, score = one.beam_search(one.prefill([prompts[2]]), 1, 10, None)
    assert torch.equal(tokens[0], want)
    eager = dec.beam_search(first, 4, 10, None)
    assert (eager[1][0][:-1] >= eager[1][0][1:]).all() and len({tuple(t) for t in eager[0][0].tolist()}) == 4
    again = decoder(model, st, weight_bits=4, cache_bits=4)
    again.prefill([prompts[2]] * 4)
    again.capture()
    assert all(torch.equal(a, b) for a, b in zip(again.beam_search(first, 4, 10, None), eager))


def test_refusals():
    model, states, prompts = make()
    for kw in (dict(weight_bits=8), dict(cache_bits=5)):
        with pytest.raises(ValueError, match="weight_bits and cache_bits"):
            decoder(model, states, **kw)
    dec = decoder(model, states)
    first = dec.prefill(prompts)
    for args in ((first, 3, 4), (first, 0, 4), (first, 2, 0), (first[:2], 2, 4)):
        with pytest.raises(ValueError, match="beams must be|steps must be"):
            dec.beam_search(*args)
    with pytest.raises(ValueError, match="RoPE table"):
        dec.beam_search(first, 4, dec.cos.shape[0])
    dec.set_sampling(0.7)
    with pytest.raises(ValueError, match="samples"):
        dec.beam_search(first, 2, 4)


def test_weights_whose_changes_are_not_counted_are_refused():
    import copy
    model, states, _ = make()
    with torch.inference_mode():
        other = copy.deepcopy(model)
    assert any(p.is_inference() for p in other.parameters())
    with pytest.raises(ValueError, match="inference tensors"):
        decoder(other, states, weight_bits=4)
