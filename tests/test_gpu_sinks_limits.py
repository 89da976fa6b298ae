"""``kernels.swa_prefill(sinks=)``: numbers of sinks that no prompt has."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,tq,hist", [(64, 200, 0), (128, 77, 300)])
def test_more_sinks_than_keys_are_all_keys(hd, tq, hist, dtype):
    """Any number past the last key makes every earlier key visible, as does the number of keys itself
    (which test_gpu_sinks.py compares with the definition)."""
    from utttcompanion_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(hd + tq)
    q = torch.randn((2, 4, tq, hd), generator=g, device=DEV).to(dtype)
    k, v = (torch.randn((2, 2, hist + tq, hd), generator=g, device=DEV).to(dtype) for _ in range(2))
    want = K.swa_prefill(q, k, v, 16, hist, sinks=hist + tq)
    for sinks in (2 ** 31 - 1, 2 ** 31, 2 ** 31 + 40, 2 ** 32, 2 ** 32 + 1, 2 ** 40, 2 ** 63 - 1):
        same = torch.equal(K.swa_prefill(q, k, v, 16, hist, sinks=sinks), want)
        assert same, sinks
