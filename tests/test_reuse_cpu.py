"""Buffers that are used again: what the operators refuse, checked where no kernel can launch."""

import pytest
import torch

from moe_dispatch import AdapterGroups, autograd, combine_backward, dispatch_backward
from moe_dispatch.ops import PackedTokens


class _Workspace:
    shape, dtype, device = (4, 16, 8, 2), torch.float32, torch.device("cpu")

    def __init__(self):
        self.dispatches = 1


def test_gradients_refuse_a_batch_whose_workspace_was_dispatched_again():
    workspace = _Workspace()
    indices = [torch.zeros(shape, dtype=torch.int32) for shape in ((4, 2), (8,), (9,))]
    batch = PackedTokens(torch.zeros(8, 16), *indices, workspace)
    batch.require_current()
    workspace.dispatches += 1
    y, w = torch.zeros(8, 16), torch.zeros(4, 2)
    for call in (lambda: combine_backward(torch.zeros(4, 16), y, batch, w), lambda: dispatch_backward(y, batch),
                 lambda: autograd.combine(y, batch, w)):
        with pytest.raises(RuntimeError, match="dispatched again"):
            call()
    # A batch formed after that dispatch is current.
    PackedTokens(torch.zeros(8, 16), *indices, workspace).require_current()


def test_the_first_assignment_is_not_captured(monkeypatch):
    groups = object.__new__(AdapterGroups)
    groups.tokens, groups.device, groups.assignment = 4, torch.device("cpu"), 0
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        groups.assign(torch.zeros(4, dtype=torch.int32))
    assert groups.assignment == 0


def test_route_refuses_before_its_forward_what_its_gradient_would():
    x = torch.zeros(2**21 + 1, 8, dtype=torch.bfloat16)
    w, bias = torch.zeros(4, 8, requires_grad=True), torch.zeros(4)
    with pytest.raises(ValueError, match="2.21 tokens"):
        autograd.route(x, w, bias, 2)
