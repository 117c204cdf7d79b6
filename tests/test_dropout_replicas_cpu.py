"""Dropout masks that have to be independent of each other: of two modules and of the replicas of a model."""
import torch

from spiky_b200 import residual


def test_modules_have_seeds_of_their_own():
    torch.manual_seed(5)
    one, two = residual.CounterDropout(0.5), residual.CounterDropout(0.5)
    torch.manual_seed(5)
    again = residual.CounterDropout(0.5)
    assert one.state[0] != two.state[0] and torch.equal(one.state, again.state)
    assert residual.CounterDropout(0.5, 9).state.tolist() == [9, 0] and residual.CounterDropout(0.5, seed=0).state.tolist() == [0, 0]
    with torch.device("meta"):
        assert residual.CounterDropout(0.5).state.is_meta
