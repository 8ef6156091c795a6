"""What `provider.decode` takes for a call that autograd would have to follow."""

import torch
import torch.autograd.forward_ad as forward_ad

from mlops_b200 import provider
from mlops_b200.weights import BlockFP8Weight


def test_gradients_and_tangents_are_seen_and_containers_in_an_open_level_pass():
    x, leaf = torch.zeros(2, 128), torch.nn.Parameter(torch.zeros(2))
    weight = BlockFP8Weight(torch.zeros(2, 128, 128).to(torch.float8_e4m3fn), torch.ones(2, 1, 1))
    asks = provider._would_be_differentiated
    assert not asks(x, None, weight) and asks(x, leaf)
    with torch.no_grad():
        assert not asks(x, leaf, weight)
    with forward_ad.dual_level():
        assert not asks(x, weight)  # a level alone changes nothing, and a container has no tangent
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert asks(weight, dual)
        with torch.no_grad():
            assert asks(dual, leaf) and not asks(leaf)
