"""C entries' limits whose arithmetic could overflow, checked where no kernel can launch."""

import pytest

from moe_dispatch import _lib
from tests.test_abi import stand_in_addresses

A = 1 << 20  # never dereferenced


@stand_in_addresses
@pytest.mark.parametrize("tokens,topk", [(1 << 62, 4), (1 << 61, 8), ((1 << 63) - 1, 2), (1 << 30, 2)])
def test_tokens_times_topk_is_bounded_before_it_is_formed(tokens, topk):
    """2^62 tokens of four experts are 2^64 assignments: 0 in 64 bits, which every buffer holds."""
    lib = _lib.load_library()
    capacity = 3
    assert lib.moe_combine(A, 2, A, A, A, tokens, 64, topk, 8, None) == capacity
    assert lib.moe_combine_backward(A, A, 2, A, A, A, A, A, A, tokens, 64, 8, topk, 8, None) == capacity
    assert lib.moe_dispatch_backward(A, 2, A, A, tokens, 64, topk, 8, None) == capacity
    assert lib.moe_dispatch(A, 2, A, A, A, A, A, A, A, 1 << 40, tokens, 64, 8, topk, 1, 8, 1, None) == capacity
    assert lib.moe_dispatch_rows(A, A, A, A, A, A, A, 1 << 40, tokens, 8, topk, 1, 8, None) == capacity


def test_gradients_that_are_not_wanted_ask_for_no_scratch():
    lib = _lib.load_library()
    tokens, hidden, width, rank, adapters = 4096, 4096, 1408, 16, 8

    def need(backward):
        return lib.moe_low_rank_scratch_bytes(tokens, hidden, width, rank, adapters, backward)

    x, down, up = 2, 4, 8  # MOE_WITHOUT_GRAD_*
    assert need(1 + x + down + up) == 0
    # Without both products: dh's sums and dh, no partial sums of a whole gradient's size.
    assert tokens * rank * 4 <= need(1 + down + up) <= (16 + 1) * tokens * rank * 4
    partial_down, partial_up = need(1 + up) - need(1 + down + up), need(1 + down) - need(1 + down + up)
    assert partial_down > 0 and partial_up > 0 and partial_down * width == partial_up * hidden
    assert need(1) == need(1 + x) == need(1 + down + up) + partial_down + partial_up
    assert need(1 + x + down) == partial_up and need(1 + x + up) == need(1 + up)


@stand_in_addresses
def test_a_backward_call_is_held_to_the_scratch_of_its_gradients():
    lib = _lib.load_library()
    sizes = 4096, 4096, 1408, 40, 8
    table = lib.moe_adapter_table_bytes(4096, 8)
    for grads, without in (((A, None, None), 12), ((None, A, None), 10), ((None, None, A), 6), ((A, A, None), 8)):
        need = lib.moe_low_rank_scratch_bytes(*sizes, 1 + without)
        status = [lib.moe_low_rank_backward(A, A, A, A, A, A, table, A, A, *grads, 0, A, nbytes, *sizes, None)
                  for nbytes in (need - 1, need)]
        assert status == [4, 5]  # workspace too small; no GPU to launch on


@pytest.mark.parametrize("tokens", [1, 128, 129, 257, 1024, 1025, 4096, 8192, 8193, 100_000, 1 << 21])
@pytest.mark.parametrize("adapters", [1, 7, 256, 4096])
def test_partial_sums_are_those_of_adapters_of_several_splits(tokens, adapters):
    """Their number does not grow with the bank, and holds the worst batch: as many adapters
    as there are rows for, each one row past a split."""
    lib = _lib.load_library()
    rank, width = 16, 64
    split = 128
    while split < 1024 and split * 8 < tokens:
        split *= 2
    size = lib.moe_low_rank_scratch_bytes(tokens, width, width, rank, adapters, 1 + 2 + 4)
    assert size % (rank * width * 4) == 0
    bound = size // (rank * width * 4)
    assert bound <= 2 * tokens / split
    for rows in (split + 1, split + 2, 2 * split, 2 * split + 1, tokens):
        whole = min(tokens // rows, adapters) if rows <= tokens else 0
        rest = tokens - whole * rows if whole < adapters else 0
        partials = whole * -(-rows // split) if rows > split else 0
        if rest > split:
            partials += -(-rest // split)
        assert partials <= bound, rows
