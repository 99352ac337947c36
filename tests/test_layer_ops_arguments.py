"""Arguments of scored routing that no kernel sees: each is refused as what it is, before anything is packed."""

import numpy as np
import pytest
import torch

from moe_dispatch import autograd, route_scored, route_scored_backward


def test_numbers_that_are_none():
    logits, ids = torch.zeros(4, 16), torch.zeros(4, 2, dtype=torch.int32)
    for scale in (None, "2", [1.0], 1j):
        with pytest.raises(TypeError, match="scale"):
            route_scored(logits, 2, scale=scale)
        with pytest.raises(TypeError, match="scale"):
            route_scored_backward(torch.zeros(4, 2), logits, ids, scale=scale)
    for best in (2.0, 1.0, "1", None):
        with pytest.raises(ValueError, match="group_best"):
            route_scored(logits, 2, groups=4, top_groups=2, group_best=best)


def test_a_bias_that_is_no_tensor():
    for call in (route_scored, autograd.route_scored):
        for bias in ([0.0] * 16, 0.5):
            with pytest.raises(TypeError, match="bias must be a tensor"):
                call(torch.zeros(4, 16), 2, bias=bias)


def test_numbers_of_other_kinds_pass():
    """Whatever packs as a number stays one: the next check is the GPU's."""
    if torch.cuda.is_available():
        pytest.skip("checks come before the GPU's presence here")
    for scale in (2, True, np.float32(1.5), np.float64(1.5), torch.tensor(1.5)):
        with pytest.raises(RuntimeError, match="GPU"):
            route_scored(torch.zeros(4, 16), 2, scale=scale)
    for best in (1, np.int64(2)):
        with pytest.raises(RuntimeError, match="GPU"):
            route_scored(torch.zeros(4, 16), 2, groups=4, top_groups=2, group_best=best)
