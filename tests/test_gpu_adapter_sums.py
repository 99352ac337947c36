"""Adapter gradients in whole numbers: every sum has one value, whatever its order."""

import pytest
import torch

from moe_dispatch import AdapterGroups, low_rank_add, low_rank_backward
from tests._helpers import gpu

pytestmark = gpu


@pytest.mark.parametrize("sizes", [
    (0, 1, 127, 128, 129, 0, 255, 256, 257, 130, 17), (129,) * 7 + (121,), (1024,), (128,) * 8, (0, 0, 300, 0, 300, 1),
    (256, 257, 255, 512, 0, 513, 1, 254, 700)])
@pytest.mark.parametrize("rank", [5, 40])
def test_adapter_gradients_on_either_side_of_a_split(sizes, rank):
    """Whole-number factors: sums are exact, so that a split or an adapter in another's place
    shows. Splits are of 128 rows up to 1024 rows, of 256 up to 2048, and of 512 behind."""
    g = torch.Generator(device="cuda").manual_seed(sum(sizes) + rank)
    tokens, hidden, width = sum(sizes), 136, 72
    ids = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), torch.tensor(sizes, device="cuda")).int()
    ids = ids[torch.randperm(tokens, device="cuda", generator=g)].contiguous()

    def whole(*shape):
        return torch.randint(-2, 3, shape, device="cuda", generator=g).bfloat16()

    x, grad, down, up = whole(tokens, hidden), whole(tokens, width), whole(len(sizes), rank, hidden), whole(len(sizes),
                                                                                                           rank, width)
    groups = AdapterGroups(tokens, len(sizes))
    groups.assign(ids)
    _, kept = low_rank_add(None, x, down, up, groups, return_hidden=True)
    _, grad_down, grad_up = low_rank_backward(grad, x, down, up, groups, hidden=kept)
    for a in range(len(sizes)):
        rows = ids == a
        h = x[rows].double() @ down[a].double().t()
        dh = grad[rows].double() @ up[a].double().t()
        assert torch.equal(grad_down[a].double(), dh.t() @ x[rows].double()), a
        assert torch.equal(grad_up[a].double(), h.t() @ grad[rows].double()), a


@pytest.mark.parametrize("rank", [4, 40])
def test_gradients_of_rows_past_two_to_the_31_elements(rank):
    """70000 rows of 32768 columns: the last 4464 lie past 2^31 elements. Whole numbers below
    2^24 throughout, so that every sum has one value, whatever its order."""
    g = torch.Generator(device="cuda").manual_seed(rank)
    tokens, width, hidden = 70000, 32768, 8

    def whole(*shape):
        return torch.randint(-1, 2, shape, device="cuda", generator=g, dtype=torch.int8).bfloat16()

    grad, x, down, up = whole(tokens, width), whole(tokens, hidden), whole(2, rank, hidden), whole(2, rank, width)
    up[:, :, torch.arange(width, device="cuda") % 512 != 3] = 0  # 64 columns: |dh| <= 64
    ids = torch.randint(0, 2, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    groups = AdapterGroups(tokens, 2)
    groups.assign(ids)
    y, kept = low_rank_add(None, x, down, up, groups, return_hidden=True)
    grad_x, grad_down, grad_up = low_rank_backward(grad, x, down, up, groups, hidden=kept)
    for a in range(2):
        rows = torch.nonzero(ids == a).squeeze(1)
        h = x[rows].float() @ down[a].float().t()
        dh = torch.zeros(rows.numel(), rank, device="cuda")
        for first in range(0, width, 4096):
            part = slice(first, first + 4096)
            wide, factor = grad[:, part][rows].float(), up[a][:, part].float()
            assert torch.equal(grad_up[a][:, part], h.t() @ wide), (a, first)
            assert torch.equal(y[:, part][rows], (h @ factor).bfloat16()), (a, first)
            dh += wide @ factor.t()
        assert torch.equal(grad_down[a], dh.t() @ x[rows].float()), a
        assert torch.equal(grad_x[rows], (dh @ down[a].float()).bfloat16()), a
