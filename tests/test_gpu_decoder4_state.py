"""Decoders in 4 bits, and beside them in 16, in and out of inference mode."""
import pytest
import torch

from test_gpu_serving import DEV, make

pytestmark = pytest.mark.gpu


def decoder(model, states, **kw):
    from utttcompanion_amd.decoder import BatchedDecoder
    return BatchedDecoder(model, states, **kw)


def run(dec, prompts):
    first = dec.prefill(prompts)
    out = [first.clone(), dec.step(first.argmax(-1)).clone()]
    out.append(dec.verify(torch.tensor([[9, 10, 11]] * 4)).clone())
    dec.commit(torch.tensor([[0, 1]] * 4), torch.tensor([2, 1, 0, 2]))
    dec.capture()
    out += [dec.step(torch.tensor([7, 8, 9, 10], device=DEV)).clone() for _ in range(2)]
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [(16, 16), (4, 16), (4, 4)])
def test_inference_mode(bits, dtype):
    """Made outside and run inside, all of it inside, and made behind an eager forward inside: as without inference mode."""
    kw = dict(weight_bits=bits[0], cache_bits=bits[1])
    model, states, prompts = make(3, dtype)
    with torch.no_grad():
        want = run(decoder(model, states, **kw), prompts)
    for before, inside in ((False, True), (False, False), (True, False)):
        model, states, prompts = make(3, dtype)
        if before:
            with torch.inference_mode():
                model(prompts[1].view(1, -1).to(DEV), fast_state=states[1], update_fast_weights=False)
        dec = None if inside else decoder(model, states, **kw)
        with torch.inference_mode(not before):
            dec = dec or decoder(model, states, **kw)
            got = run(dec, prompts)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_packs_made_in_inference_mode_follow_outside():
    model, states, prompts = make(0)
    dec = decoder(model, states, weight_bits=4)
    with torch.inference_mode():
        first = dec.prefill(prompts)
        dec.step(first.argmax(-1))
        caches = [dec.export_kv_caches(i) for i in range(4)]
    with torch.no_grad():
        model.layers[0].attn.wv.weight.mul_(1.5)
        model.norm.weight.mul_(0.75)
    other = decoder(model, states, weight_bits=4)
    tok = torch.tensor([7, 8, 9, 10], device=DEV)
    for d in (dec, other):
        d.reset(caches, [len(p) + 1 for p in prompts])
    assert torch.equal(dec.step(tok), other.step(tok))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [(16, 4), (4, 4), (4, 16)])
def test_beams_hold_what_their_tokens_lead_to(bits, dtype):
    """The scores of beam search over caches that are reordered at every step, against the sums of log-probabilities of each
    hypothesis stepped through caches of its own, among as many requests: the logits are the same bit by bit."""
    kw = dict(weight_bits=bits[0], cache_bits=bits[1])
    model, states, prompts = make(2, dtype)
    st = [states[0]] * 4 + [states[1]] * 4
    prompt = [prompts[2]] * 4 + [prompts[1]] * 4
    dec = decoder(model, st, **kw)
    steps = 12
    tokens, scores = dec.beam_search(dec.prefill(prompt), 4, steps, None)
    again = decoder(model, st, **kw)
    logits, total = again.prefill(prompt), torch.zeros(8, dtype=torch.float64)
    allowed = torch.full((model.config.vocab_size,), True)
    allowed[[0, 1, 3]] = False
    allowed[model.active_vocab_limit:] = False
    flat = tokens.view(8, steps)
    for i in range(steps):
        x = logits.double().cpu().masked_fill(~allowed, -torch.inf)
        total += torch.log_softmax(x, 1).gather(1, flat[:, i:i + 1].cpu())[:, 0]
        logits = again.step(flat[:, i].contiguous())
    assert any(len(set(map(tuple, g))) == 4 for g in tokens.tolist())
    # per step a sum's error (2.25 log(256) + 2 + 15 half steps, the top moved once: 2 more) and the score's own half step
    got = scores.view(8).double().cpu()
    assert ((got - total).abs() <= steps * 2.0 ** -24 * (2.25 * 5.6 + 19 + got.abs())).all(), (got - total).abs().max()
    # the requests stand where their beams do: the last token's step gives the logits that the hypothesis' own gave
    assert torch.equal(dec.step(dec.tokens), logits) and dec.host_positions == again.host_positions
