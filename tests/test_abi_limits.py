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
