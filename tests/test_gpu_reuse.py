"""Buffers that are used again between a forward and its backward pass."""

import pytest
import torch

from moe_dispatch import (AdapterGroups, MoEBlock, MoEConfig, autograd, combine_backward, dispatch, dispatch_backward,
                          low_rank_add, low_rank_backward)
from moe_dispatch.ops import PackedTokens
from tests._helpers import gpu

pytestmark = gpu

BF16 = torch.bfloat16


def _normal(g, *shape, dtype=BF16):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _ids(g, tokens, experts, topk):
    return torch.randint(0, experts, (tokens, topk), device="cuda", generator=g, dtype=torch.int32)


@pytest.mark.parametrize("again", ["ops", "workspace"])
def test_a_batch_of_an_earlier_dispatch_gets_no_gradients(again):
    """The second dispatch has put its own rows where the first batch's views look."""
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens, hidden, experts, topk = 50, 64, 4, 2
    x = _normal(g, tokens, hidden).requires_grad_()
    ids, others = _ids(g, tokens, experts, topk), _ids(g, tokens, experts, topk)
    weights = torch.rand(tokens, topk, device="cuda", generator=g).requires_grad_()
    packed, batch = autograd.dispatch(x, ids, experts)
    out = autograd.combine(packed * 2, batch, weights)
    y, dout = _normal(g, *batch.packed.shape), _normal(g, tokens, hidden)
    want = combine_backward(dout, y, batch, weights.detach())
    if again == "ops":
        second = dispatch(x.detach(), others, experts, workspace=batch.workspace)
    else:
        workspace = batch.workspace
        workspace.dispatch(x.detach(), others)
        second = PackedTokens(workspace.packed, workspace.inverse, workspace.counts, workspace.offsets, workspace)
    for call in (lambda: out.sum().backward(), lambda: packed.float().sum().backward(),
                 lambda: combine_backward(dout, y, batch, weights.detach()), lambda: dispatch_backward(y, batch),
                 lambda: autograd.combine(packed, batch, weights)):
        with pytest.raises(RuntimeError, match="dispatched again"):
            call()
    # The second batch is current; dispatched as the first was, so is a third.
    assert not torch.equal(combine_backward(dout, y, second, weights.detach())[1], want[1])
    third = dispatch(x.detach(), ids, experts, workspace=batch.workspace)
    for a, b in zip(combine_backward(dout, y, third, weights.detach()), want):
        assert torch.equal(a, b)


def test_a_batch_of_a_blocks_transport_ends_with_the_next_forward():
    """Both forms of a block's forward write its transport's index buffers."""
    g = torch.Generator(device="cuda").manual_seed(1)
    block = MoEBlock(MoEConfig(hidden=64, intermediate=128, experts=4, topk=2), device="cuda:0",
                     implementation="cuda_fused", seed=0)
    x = _normal(g, 40, 64)
    grad = None
    for _ in range(3):  # validated, then by one native call
        block(x)
        t = block.workspace(x).transport
        batch = PackedTokens(t.packed, t.inverse, t.counts, t.offsets, t)
        grad = _normal(g, *t.packed.shape)
        dispatch_backward(grad, batch)
        block(x)
        with pytest.raises(RuntimeError, match="dispatched again"):
            dispatch_backward(grad, batch)


def test_a_captured_assignment_takes_effect_when_it_is_replayed():
    """Between capture and replay the groups are those of the last assignment that ran."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x, base = _normal(g, 70, 64), _normal(g, 70, 72)
    down, up = _normal(g, 3, 8, 64), _normal(g, 3, 8, 72)
    first, second = (torch.randint(-1, 3, (70,), device="cuda", generator=g, dtype=torch.int32) for _ in range(2))

    def alone(ids):
        groups = AdapterGroups(70, 3)
        groups.assign(ids)
        return low_rank_add(base, x, down, up, groups)

    want = alone(first), alone(second)
    assert not torch.equal(*want)
    groups = AdapterGroups(70, 3)
    groups.assign(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        groups.assign(second)
        captured = low_rank_add(base, x, down, up, groups)
    assert torch.equal(low_rank_add(base, x, down, up, groups), want[0])
    for _ in range(3):
        captured.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want[1])
        assert torch.equal(low_rank_add(base, x, down, up, groups), want[1])
        groups.assign(first)
        assert torch.equal(low_rank_add(base, x, down, up, groups), want[0])


def test_the_gradient_of_x_alone_takes_no_memory_of_the_others():
    """Frozen adapters: no scratch of the size of their gradients."""
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens, hidden, rank, adapters = 4096, 1024, 16, 64
    x, grad = _normal(g, tokens, hidden), _normal(g, tokens, hidden)
    down, up = _normal(g, adapters, rank, hidden), _normal(g, adapters, rank, hidden)
    groups = AdapterGroups(tokens, adapters)
    groups.assign(torch.randint(0, adapters, (tokens,), device="cuda", generator=g, dtype=torch.int32))
    _, kept = low_rank_add(None, x, down, up, groups, return_hidden=True)
    want = low_rank_backward(grad, x, down, up, groups, hidden=kept)[0]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got, _, _ = low_rank_backward(grad, x, down, up, groups, hidden=kept, gradients=(True, False, False))
    peak = torch.cuda.max_memory_allocated() - before
    assert torch.equal(got, want)
    # The result, dh and up to sixteen slices' sums of it, and the allocator's 512-byte steps.
    assert peak <= tokens * hidden * 2 + 17 * tokens * rank * 4 + 4096
