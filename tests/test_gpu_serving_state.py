"""What a decoder's calls leave in its state: the tokens, log-probabilities and logits that the next call goes on from."""
import pytest
import torch

from test_gpu_serving import decoder, drafts, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sinks", [0, 5])
def test_capture_keeps_what_was_chosen(sinks, dtype):
    """Recording a step between two steps changes nothing that was there: tokens, log-probabilities and logits, and the
    steps that follow are those without it."""
    model, states, prompts = make(sinks, dtype)
    runs = []
    for captured in (False, True):
        dec, first = decoder(model, states, prompts)
        dec.generate_greedy(first, 5)
        dec.set_sampling(0.9, top_p=0.8, generator=torch.Generator(DEV).manual_seed(4))
        trail = []
        for _ in range(2):  # again: over a step that is recorded already
            for _ in range(3):
                if captured:
                    held = dec.tokens.clone(), dec.logits.clone(), dec.positions.clone(), dec.k_rings.clone(), dec.v_rings.clone()
                    logprobs = dec.logprobs.clone()
                    dec.capture()
                    now = dec.tokens, dec.logits, dec.positions, dec.k_rings, dec.v_rings
                    assert all(torch.equal(a, b) for a, b in zip(now, held)) and torch.equal(dec.logprobs, logprobs)
                dec.step(dec.next_tokens)
                trail += [dec.tokens.clone(), dec.logprobs.clone(), dec.logits.clone()]
            dec.fork([1, 0, 3, 3])
            trail += [dec.tokens.clone(), dec.logprobs.clone(), dec.logits.clone()]
        dec.set_sampling(None)
        if captured:
            dec.capture()
        for _ in range(3):
            dec.step(dec.tokens)
            trail += [dec.tokens.clone(), dec.logits.clone()]
        runs.append(trail)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_capture_before_the_first_step_leaves_no_logits():
    model, states, prompts = make()
    dec, first = decoder(model, states, prompts)
    dec.capture()
    assert dec.logits is None and dec.next_tokens is None and dec.tokens.tolist() == [0] * 4
    twin, _ = decoder(model, states, prompts)
    token = first.argmax(1)
    assert torch.equal(dec.step(token), twin.step(token)) and torch.equal(dec.next_tokens, twin.next_tokens)
    assert dec.next_tokens.data_ptr() == dec.tokens.data_ptr()


def test_speculation_is_refused_while_the_decoder_samples():
    """As greedy generation is: a round would take greedy choices, whatever the settings.  Nothing has changed then."""
    model, states, prompts = make()
    dec, first = decoder(model, states, prompts)
    dec.set_sampling(0.8)
    dec.generate_sampled(first, 3)
    held = dec.tokens.clone(), dec.positions.clone(), dec.k_rings.clone(), dec.logprobs.clone()
    with pytest.raises(ValueError, match="samples"):
        dec.speculate_greedy(dec.tokens[:, None])
    with pytest.raises(ValueError, match="samples"):
        dec.speculate_greedy(torch.ones(4, 3, dtype=torch.int64), torch.tensor([[-1, 0, 0]] * 4))
    assert all(torch.equal(a, b) for a, b in zip((dec.tokens, dec.positions, dec.k_rings, dec.logprobs), held))
    dec.set_sampling(None)
    dec.speculate_greedy(dec.tokens[:, None])


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("sinks", [0, 5])
def test_speculation_leaves_the_logits_behind_its_last_token(sinks, captured):
    """As a step does: generating from ``logits``, stepping on, and forks of the requests go on as single steps would."""
    import random
    model, states, prompts = make(sinks)
    plain, first = decoder(model, states, prompts)
    truth = plain.generate_greedy(first, 40).tolist()
    for after in ("generate", "step", "fork"):
        dec, first = decoder(model, states, prompts)
        if captured:
            dec.capture()
        rng, have = random.Random(3), [[t[0]] for t in truth]
        for _ in range(3):
            trees = [drafts(truth, len(have[i]) - 1, i, rng, 5) for i in range(4)]
            tokens, parents = torch.tensor([t for t, _ in trees]), torch.tensor([p for _, p in trees], dtype=torch.int32)
            verified = dec.verify(tokens, parents)
            new = dec.speculate_greedy(tokens, parents)
            for i, row in enumerate(new):
                node = 0  # the last one taken
                for token in row[:-1]:
                    node = next(j for j in range(5) if parents[i, j] == node and tokens[i, j] == token)
                assert torch.equal(dec.logits[i], verified[i, node]), i
                have[i] += row
            assert dec.next_tokens.tolist() == dec.tokens.tolist() == [h[-1] for h in have]
            if captured:  # a replay between the rounds
                dec.step(dec.next_tokens)
                for h, t in zip(have, dec.tokens.tolist()):
                    h.append(t)
        assert have == [t[:len(h)] for t, h in zip(truth, have)]
        src = [0, 1, 2, 3]
        if after == "step":
            dec.step(dec.tokens)
            have = [h + [t] for h, t in zip(have, dec.tokens.tolist())]
        elif after == "fork":
            src = [2, 2, 0, 1]
            dec.fork(src)
        got = dec.generate_greedy(dec.logits, 6).tolist()
        # the first token from the logits is the last one chosen
        assert got == [truth[s][len(have[s]) - 1:len(have[s]) + 5] for s in src], after


@pytest.mark.parametrize("sinks", [0, 5])
def test_committed_bf16_nodes_are_the_steps_up_to_their_roundings(sinks):
    """The same tokens stepped one by one, and verified and committed at once.  Of the first layer, whose inputs are equal,
    with u = 2^-8: the projections are within one rounding on each side, 2 u of a key's element; the rotation rounds once in
    the tree and, without sinks, three times in a step: of each product (together at most sqrt 2 of the pair's length h) and
    of the sum.  So the keys are within (2 sqrt 2 + sqrt 2 + 2) u h and the values within 2 u, and 2^-16 for the fp32 sums of
    128 products of about 2 in all; what follows, within the bound that holds between bf16 steps and eager bf16 forwards."""
    model, states, prompts = make(sinks, torch.bfloat16, slow_std=0.02)
    stepped, _ = decoder(model, states, prompts)
    drafted, _ = decoder(model, states, prompts)
    ids = torch.randint(6, 256, (4, 8), generator=torch.Generator().manual_seed(5)).to(DEV)
    for t in range(8):
        logits = stepped.step(ids[:, t])
    verified = drafted.verify(ids)
    drafted.commit(torch.arange(8).expand(4, -1), torch.full((4,), 8))
    assert drafted.host_positions == stepped.host_positions and torch.equal(drafted.positions, stepped.positions)
    torch.testing.assert_close(verified[:, -1].float(), logits.float(), atol=0.015, rtol=0.025)
    a, b = stepped.k_rings[0].double(), drafted.k_rings[0].double()
    lo, hi = a.chunk(2, -1)
    length = torch.hypot(lo, hi).repeat(1, 1, 1, 2)
    u, root = 2.0 ** -8, 2.0 ** 0.5
    assert bool(((a - b).abs() <= (3 * root + 2) * u * length + 2.0 ** -16).all())
    a, b = stepped.v_rings[0].double(), drafted.v_rings[0].double()
    assert bool(((a - b).abs() <= 2 * u * torch.maximum(a.abs(), b.abs()) + 2.0 ** -16).all())
    for x, y in ((stepped.k_rings, drafted.k_rings), (stepped.v_rings, drafted.v_rings)):
        torch.testing.assert_close(x, y, atol=0.015, rtol=0.025)
    more = torch.randint(6, 256, (4,), generator=torch.Generator().manual_seed(6)).to(DEV)
    torch.testing.assert_close(stepped.step(more).float(), drafted.step(more).float(), atol=0.015, rtol=0.025)


@pytest.mark.parametrize("sinks", [0, 5])
def test_nodes_that_were_not_computed_are_loud_when_committed(sinks):
    """A request whose parents are no earlier nodes has NaN logits, and nodes behind ``counts`` do not exist: neither has keys
    or values, and committing one all the same puts NaN into that request's cache, not whatever memory held."""
    model, states, prompts = make(sinks)
    dec, _ = decoder(model, states, prompts)
    twin, _ = decoder(model, states, prompts)
    at = list(dec.host_positions)
    tokens = torch.randint(6, 256, (4, 3), generator=torch.Generator().manual_seed(8))
    parents = torch.tensor([[-1, 0, 1]] * 4, dtype=torch.int32)
    want = twin.verify(tokens, parents)
    bad = parents.clone()
    bad[2, 1] = 2
    counts = torch.tensor([3, 2, 3, 3], dtype=torch.int32)
    logits = dec.verify(tokens, bad, counts)
    assert bool(logits[2].isnan().all()) and torch.equal(logits[[0, 3]], want[[0, 3]]) and torch.equal(logits[1, :2], want[1, :2])
    path = torch.tensor([[0, 1, 2]] * 4)
    dec.commit(path, torch.tensor([3, 3, 2, 3]))
    twin.commit(path, torch.tensor([3, 3, 2, 3]))
    slots = lambda i, n: dec._cached_slots(min(at[i] + n, dec.slots), at[i] + n)[-n:]  # noqa: E731
    for mine, theirs in ((dec.k_rings, twin.k_rings), (dec.v_rings, twin.v_rings)):
        assert torch.equal(mine[:, [0, 3]], theirs[:, [0, 3]])
        assert bool(mine[:, 2].index_select(2, slots(2, 2)).isnan().all())
        new = mine[:, 1].index_select(2, slots(1, 3))
        assert bool(new[:, :, 2].isnan().all()) and torch.equal(new[:, :, :2], theirs[:, 1].index_select(2, slots(1, 3))[:, :, :2])
