"""Workspaces that do not lie together are refused before any launch (no GPU needed: the device check is passed over, and a launch
would fail the test)."""
import pytest
import torch

from utttcompanion_amd import kernels as K


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(K, "_gpu_index", lambda *tensors: 0)
    monkeypatch.setattr(K, "_serve_call", lambda *args: pytest.fail("launched"))


def trees(n=2, t=3, hkv=1, hd=64, window=4096):
    q = torch.zeros(n, t, 4 * hkv, hd)
    new = torch.zeros(n, t, hkv, hd)
    return q, new, torch.zeros(n, dtype=torch.int64), window


def test_tree_over_a_cache_in_four_bits(no_launch):
    q, new, pos, window = trees()
    cache = K.kv_cache4(2, 1, window=window, sinks=0, head_dim=64, device=torch.device("cpu"))
    nbytes = K._tree4_workspace(2, 4, 1, 3, 64, window, 0)
    assert nbytes > 16
    for bad in (torch.zeros(2 * nbytes, dtype=torch.uint8)[::2], torch.zeros(nbytes, 2, dtype=torch.uint8)[:, 0],
                torch.zeros(nbytes - 1, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="contiguous bytes"):
            K.swa_tree4(q, new, new, cache, pos, window, workspace=bad)


def test_tree_over_rings(no_launch):
    q, new, pos, window = trees()
    ring = torch.zeros(2, 1, window, 64)
    nbytes = K._tree_workspace(2, 4, 1, 3, 64, window, 0)
    assert nbytes > 16
    for bad in (torch.zeros(2 * nbytes, dtype=torch.uint8)[::2], torch.zeros(nbytes - 1, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="contiguous bytes"):
            K.swa_tree(q, new, new, ring, ring.clone(), pos, workspace=bad)
