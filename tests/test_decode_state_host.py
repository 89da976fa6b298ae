"""What a decoder in 4 bits keeps of the model's weights, on the CPU: packs made and followed in and out of inference mode."""
import torch

from utttcompanion_amd import SlidingWindowAttention, uTTTConfig, uTTTModel
from utttcompanion_amd import kernels as K
from utttcompanion_amd.decoder import BatchedDecoder

TINY = dict(vocab_size=64, d_model=64, n_layers=2, n_heads=2, n_kv_heads=1, d_ff_fast=64, chunk_size=16,
            sliding_window_size=16)


def packs(model):
    """The part of a decoder that holds slow weights in 4 bits."""
    dec = BatchedDecoder.__new__(BatchedDecoder)
    dec.model, dec.dtype, dec.weight_bits, dec._fours = model, torch.float32, 4, {}
    return dec


def test_the_packed_qkv_is_an_ordinary_tensor_in_any_mode():
    attn = SlidingWindowAttention(64, 2, 1).eval()
    with torch.inference_mode():
        packed = attn.packed_qkv()
        attn.prepare_for_inference()
    assert not packed.is_inference() and attn.packed_qkv() is packed and packed._version == 0
    assert torch.equal(packed, torch.cat([attn.wq.weight, attn.wk.weight, attn.wv.weight]))


def test_weights_in_four_bits_follow_the_model_in_any_mode():
    """Packed first in inference mode, changed in either mode, packed again in place in either mode."""
    torch.manual_seed(0)
    model = uTTTModel(uTTTConfig(**TINY)).eval()
    dec = packs(model)
    with torch.inference_mode():
        model.prepare_for_inference()
        dec._refresh4()
    held = {name: hit[1].data for name, hit in dec._fours.items()}
    assert len(held) == 4 * 2 + 1 and not any(t.is_inference() for t in held.values())

    def same():
        for li, block in enumerate(model.layers):
            w = torch.cat([block.attn.wq.weight, block.attn.wk.weight, block.attn.wv.weight])
            for kind, w, norm in (("qkv", w, block.attn_norm), ("wo", block.attn.wo.weight, None),
                                  ("q", block.uttt.w_q.weight, block.uttt_norm), ("o", block.uttt.w_o.weight, None)):
                w = w if norm is None else w * norm.weight[None]
                assert torch.equal(held[kind, li], K.pack_weight4(w).data), (kind, li)
        assert torch.equal(held["head",], K.pack_weight4(model.lm_head.weight * model.norm.weight[None]).data)

    same()
    for change, refresh in ((True, False), (False, True), (True, True), (False, False)):
        with torch.inference_mode(change), torch.no_grad():
            block = model.layers[1]
            for w in (block.attn.wk.weight, block.attn.wo.weight, block.uttt.w_o.weight, model.lm_head.weight,
                      block.uttt_norm.weight):
                w.mul_(1.0 + 0.5 * torch.rand(w.shape))
        with torch.inference_mode(refresh), torch.no_grad():
            dec._refresh4()
        assert all(dec._fours[name][1].data is t for name, t in held.items())
        same()
