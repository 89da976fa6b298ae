"""Refusals of the serving wrappers that need no GPU: operands that ask for gradients."""
import pytest
import torch

from utttcompanion_amd import kernels as K


def test_sampling_refuses_operands_that_ask_for_gradients():
    """Its log-probabilities have none, so they are refused, as the other serving calls' are; under no_grad they pass on."""
    x, u = torch.zeros(2, 100), torch.ones(2)
    asks = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda: K.sample_select(asks(x), u, u), lambda: K.sample_select(x, u, asks(u)),
             lambda: K.sample_select(x, u, u, top_p=asks(u)), lambda: K.sample_select(x, u, u, min_p=asks(u)),
             lambda: K.sample_select(asks(x)[:, 1:], u, u)]
    for call in calls:
        with pytest.raises(ValueError, match="forward-only"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
            call()


@pytest.mark.parametrize("ids", [(-1,), (3, 2 ** 31), (2 ** 40,)])
def test_sampling_refuses_banned_ids_that_are_none(ids):
    x, u = torch.zeros(2, 100), torch.ones(2)
    with pytest.raises(ValueError, match="excluded ids"):
        K.sample_select(x, u, u, banned=ids)
