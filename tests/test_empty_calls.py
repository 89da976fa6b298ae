"""Calls in 4 bits without a row, on the CPU: nothing is launched and nothing is wrong with them."""
import pytest
import torch

from utttcompanion_amd import kernels as K


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(K, "_gpu_index", lambda *tensors: 0)
    monkeypatch.setattr(K, "_serve_call", lambda *args: pytest.fail("launched"))


def test_linear_without_rows(no_launch):
    """Empty tensors have no address that tells them apart."""
    p = K.pack_weight4(torch.ones(8, 40))
    for out in (None, torch.empty(0, 8)):
        for residual in (None, torch.empty(0, 8), out):
            assert K.linear4(torch.empty(0, 40), p, out=out, residual=residual).shape == (0, 8)


def test_readout_without_rows(no_launch):
    up, down, ln = K.pack_weight4(torch.ones(128, 64)), K.pack_weight4(torch.ones(64, 128)), torch.ones(64)
    for shape in ((0, 1, 64), (2, 0, 64)):
        for out in (None, torch.empty(shape)):
            assert K.readout4(torch.empty(shape), up, up, down, ln, ln, out=out).shape == shape


def test_caches_without_requests(no_launch):
    c = K.kv_cache4(2, 0, 1, window=40, sinks=2, head_dim=64, device=torch.device("cpu"))
    pos, ids = torch.zeros(0, dtype=torch.int64), torch.zeros(0, dtype=torch.int32)
    k = torch.empty(2, 0, 3, 1, 64)
    K.kv_commit4(k, k, None, None, c, pos, 40, 2)
    K.kv_fork4(c, ids, pos, 40, 2)
    assert K.kv_values4(c, 40, 2)[0].shape == (2, 0, 1, 42, 64)
    q, new = torch.empty(0, 3, 4, 64), torch.empty(0, 3, 1, 64)
    for nodes in (None, (torch.empty_like(new), torch.empty_like(new))):
        out, kn, vn = K.swa_tree4(q, new, new, c[0], pos, 40, sinks=2, node_outputs=nodes)
        assert out.shape == q.shape and kn.shape == vn.shape == new.shape


def test_beams_without_rows(no_launch):
    tokens, sources, scores, ended = K.beam_select(torch.empty(0, 100), torch.empty(0), 3)
    assert len(tokens) == len(sources) == len(scores) == len(ended) == 0
