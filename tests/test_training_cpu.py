"""Refusals of the training and adapter operators, checked where no kernel can launch."""

from types import SimpleNamespace

import pytest
import torch

from moe_dispatch import (AdapterGroups, RouterLoss, _lib, combine_backward, dispatch_backward, low_rank_add,
                          low_rank_backward, route_backward, route_logits_backward, router_loss)
from moe_dispatch.adapters import LowRankHidden
from moe_dispatch.ops import PackedTokens
from tests.test_abi import stand_in_addresses

BF16 = torch.bfloat16


def _routed(tokens=4, experts=8, topk=2):
    return torch.zeros(tokens, experts), torch.zeros(tokens, topk, dtype=torch.int32), torch.zeros(experts)


def test_router_loss_refuses_bad_tensors():
    logits, ids, bias = _routed()
    with pytest.raises(TypeError, match="logits"):
        router_loss(logits.to(BF16), ids, bias)
    with pytest.raises(TypeError, match="expert_ids"):
        router_loss(logits, ids.long(), bias)
    with pytest.raises(TypeError, match="mask"):
        router_loss(logits, ids, bias, mask=torch.ones(4))
    with pytest.raises(ValueError, match="expert_ids"):
        router_loss(logits, ids[:3].contiguous(), bias)
    with pytest.raises(ValueError, match="bias"):
        router_loss(logits, ids, bias[:7].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        router_loss(torch.zeros(8, 4).t(), ids, bias)
    with pytest.raises(ValueError, match="1..64"):
        router_loss(torch.zeros(4, 65), ids)
    with pytest.raises(ValueError, match="1..8"):
        router_loss(logits, torch.zeros(4, 9, dtype=torch.int32))
    with pytest.raises(ValueError, match="mask"):
        router_loss(logits, ids, mask=torch.ones(5, dtype=torch.bool))


def test_route_gradients_refuse_bad_tensors():
    logits, ids, bias = _routed()
    with pytest.raises(TypeError, match="RouterLoss"):
        route_logits_backward(logits, ids, bias, grad_losses=torch.zeros(2))
    loss = RouterLoss(torch.zeros(2), torch.zeros(9, dtype=torch.int32))
    with pytest.raises(ValueError, match="grad_losses"):
        route_logits_backward(logits, ids, bias, loss=loss, grad_losses=torch.zeros(3))
    short = RouterLoss(torch.zeros(2), torch.zeros(8, dtype=torch.int32))
    with pytest.raises(ValueError, match="stats"):
        route_logits_backward(logits, ids, bias, loss=short, grad_losses=torch.zeros(2))
    with pytest.raises(ValueError, match="grad_weights"):
        route_logits_backward(logits, ids, bias, grad_weights=torch.zeros(4, 3))
    x, w = torch.zeros(4, 64, dtype=BF16), torch.zeros(8, 64)
    with pytest.raises(TypeError, match="x must be"):
        route_backward(x.float(), w, logits, ids)
    with pytest.raises(ValueError, match="router_weight"):
        route_backward(x, w[:, :32].contiguous(), logits, ids)
    with pytest.raises(ValueError, match="multiple of 8"):
        route_backward(torch.zeros(4, 12, dtype=BF16), torch.zeros(8, 12), logits, ids)
    with pytest.raises(ValueError, match="grad_x"):
        route_backward(x, w, logits, ids, grad_x=x[:3])


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU error path")
def test_operators_need_a_gpu():
    logits, ids, bias = _routed()
    with pytest.raises(RuntimeError, match="GPU"):
        router_loss(logits, ids, bias)
    with pytest.raises(RuntimeError, match="GPU"):
        route_logits_backward(logits, ids, bias)
    with pytest.raises(RuntimeError, match="GPU"):
        route_backward(torch.zeros(4, 64, dtype=BF16), torch.zeros(8, 64), logits, ids)
    with pytest.raises(RuntimeError, match="GPU"):
        AdapterGroups(4, 2)


class _Workspace:
    shape, dtype, device = (4, 16, 8, 2), torch.float32, torch.device("cpu")


def _batch():
    return PackedTokens(torch.zeros(8, 16), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32),
                        torch.zeros(9, dtype=torch.int32), _Workspace())


def test_transport_gradients_refuse_bad_tensors():
    batch = _batch()
    y, w = torch.zeros(8, 16), torch.zeros(4, 2)
    with pytest.raises(TypeError, match="grad_output"):
        combine_backward(torch.zeros(4, 16, dtype=BF16), y, batch, w)
    with pytest.raises(ValueError, match="grad_output"):
        combine_backward(torch.zeros(3, 16), y, batch, w)
    with pytest.raises(ValueError, match="expert_output"):
        combine_backward(torch.zeros(4, 16), torch.zeros(9, 16), batch, w)
    with pytest.raises(TypeError, match="weights"):
        combine_backward(torch.zeros(4, 16), y, batch, w.double())
    with pytest.raises(ValueError, match="grad_packed"):
        dispatch_backward(torch.zeros(8, 15), batch)


def _groups(tokens=4, adapters=3, assigned=True):
    groups = object.__new__(AdapterGroups)
    groups.tokens, groups.adapters, groups.device = tokens, adapters, torch.device("cpu")
    groups.assignment, groups.table_bytes, groups._sizes = int(assigned), 0, {}
    groups.extension = SimpleNamespace(lib=_lib.load_library())
    return groups


def _operands(tokens=4, hidden=64, width=32, rank=8, adapters=3):
    def zeros(*shape):
        return torch.zeros(shape, dtype=BF16)

    return zeros(tokens, width), zeros(tokens, hidden), zeros(adapters, rank, hidden), zeros(adapters, rank, width)


def test_groups_refuse_bad_sizes():
    for tokens, adapters in ((-1, 2), (2**21 + 1, 2), (4.0, 2), (4, 0), (4, 4097)):
        with pytest.raises(ValueError):
            AdapterGroups(tokens, adapters)
    with pytest.raises(RuntimeError):
        AdapterGroups(4, 2, device="cpu")
    groups = _groups()
    with pytest.raises(TypeError, match="ids"):
        groups.assign(torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="ids"):
        groups.assign(torch.zeros(5, dtype=torch.int32))


def test_low_rank_add_refuses_bad_tensors():
    base, x, down, up = _operands()
    groups = _groups()
    with pytest.raises(TypeError, match="groups"):
        low_rank_add(base, x, down, up, None)
    with pytest.raises(RuntimeError, match="assign"):
        low_rank_add(base, x, down, up, _groups(assigned=False))
    with pytest.raises(TypeError, match="x must be"):
        low_rank_add(base, x.float(), down, up, groups)
    with pytest.raises(ValueError, match="x:"):
        low_rank_add(base, x[:3], down, up, groups)
    with pytest.raises(ValueError, match="down"):
        low_rank_add(base, x, down[:2], up, groups)
    with pytest.raises(ValueError, match="up"):
        low_rank_add(base, x, down, up[:, :7].contiguous(), groups)
    with pytest.raises(ValueError, match="base"):
        low_rank_add(base[:, :24].contiguous(), x, down, up, groups)
    with pytest.raises(ValueError, match="scales"):
        low_rank_add(base, x, down, up, groups, scales=torch.ones(4))
    with pytest.raises(TypeError, match="scales"):
        low_rank_add(base, x, down, up, groups, scales=torch.ones(3, dtype=BF16))
    with pytest.raises(ValueError, match="multiple of 8"):
        low_rank_add(*_operands(hidden=60), groups)
    with pytest.raises(ValueError, match="multiple of 8"):
        low_rank_add(*_operands(width=36), groups)
    with pytest.raises(ValueError, match="1..128"):
        low_rank_add(*_operands(rank=129), groups)
    square = _operands(width=64)
    with pytest.raises(ValueError, match="overlap"):
        low_rank_add(*square, groups, output=square[1])
    storage = torch.zeros(4 * 32 + 32, dtype=BF16)
    with pytest.raises(ValueError, match="overlap"):
        low_rank_add(storage[:128].view(4, 32), x, down, up, groups, output=storage[32:].view(4, 32))
    with pytest.raises(ValueError, match="autograd"):
        low_rank_add(base, x.requires_grad_(), down, up, groups)


def test_low_rank_backward_refuses_bad_tensors():
    grad, x, down, up = _operands()
    groups = _groups()
    kept = torch.zeros(4, 8)
    hidden = LowRankHidden(kept, groups, 1)
    with pytest.raises(TypeError, match="hidden"):
        low_rank_backward(grad, x, down, up, groups, hidden=kept)
    for stale in (LowRankHidden(kept, groups, 2), LowRankHidden(kept, _groups(), 1)):
        with pytest.raises(RuntimeError, match="another assignment"):
            low_rank_backward(grad, x, down, up, groups, hidden=stale)
    with pytest.raises(ValueError, match="hidden"):
        low_rank_backward(grad, x, down, up, groups, hidden=LowRankHidden(kept[:, :7].contiguous(), groups, 1))
    with pytest.raises(ValueError, match="grad_output"):
        low_rank_backward(grad[:, :8].contiguous(), x, down, up, groups, hidden=hidden)
    with pytest.raises(ValueError, match="grad_x"):
        low_rank_backward(grad, x, down, up, groups, hidden=hidden, grad_x=grad)
    with pytest.raises(TypeError, match="grad_dtype"):
        low_rank_backward(grad, x, down, up, groups, hidden=hidden, grad_dtype=torch.float16)


@stand_in_addresses
def test_c_entries_check_their_arguments_without_launching():
    lib = _lib.load_library()
    A = 1 << 20  # never dereferenced
    big = 1 << 40
    assert lib.moe_router_loss_scratch_bytes(4, 65) == -1 and lib.moe_router_loss_scratch_bytes(-1, 8) == -1
    # logits, bias, ids, mask, losses, stats, scratch, bytes, T, E, K
    assert lib.moe_router_loss(A, A, A, None, A, A, A, big, 4, 65, 2, None) == 2
    assert lib.moe_router_loss(A, A, A, None, A, A, A, big, 4, 8, 9, None) == 2
    assert lib.moe_router_loss(None, A, A, None, A, A, A, big, 4, 8, 2, None) == 1
    assert lib.moe_router_loss(A, A, A, None, None, A, A, big, 4, 8, 2, None) == 1
    assert lib.moe_router_loss_scratch_bytes(128, 8) == 0  # one block
    need = lib.moe_router_loss_scratch_bytes(8192, 64)
    assert lib.moe_router_loss(A, A, A, None, A, A, A, need - 1, 8192, 64, 2, None) == 4
    assert lib.moe_router_loss(A, A, A, None, A, A, None, need, 8192, 64, 2, None) == 4
    assert lib.moe_router_loss(A, A, A, None, A, A, A, big, 1 << 29, 8, 2, None) == 3
    # logits, bias, ids, mask, stats, grad_losses, grad_weights, grad_logits, T, E, K
    assert lib.moe_router_logits_backward(A, A, A, None, None, A, A, A, 4, 8, 2, None) == 1
    assert b"stats" in lib.moe_last_error()
    assert lib.moe_router_logits_backward(A, A, A, None, A, A, A, None, 4, 8, 2, None) == 1
    assert lib.moe_router_logits_backward(A, A, A, None, A, A, A, A + 2, 4, 8, 2, None) == 1
    assert lib.moe_router_logits_backward(A, A, A, None, A, A, A, A, 0, 8, 2, None) == 0
    need = lib.moe_route_backward_scratch_bytes(4, 64, 8)
    assert need > 0 and lib.moe_route_backward_scratch_bytes(4, 60, 8) == -1

    def route(x=A, w=A, gx=A, gw=A, nbytes=need, tokens=4, hidden=64):
        return lib.moe_route_backward(x, w, A, A, A, None, A, A, A, A, gx, gw, A, A, nbytes, tokens, hidden, 8, 2, None)

    assert route(hidden=60) == 2 and route(nbytes=need - 1) == 4 and route(tokens=0) == 3
    assert route(x=None) == 1 and route(w=None) == 1 and route(x=A + 8) == 1 and route(gx=A + 8) == 1
    # grad_output, expert_output, dtype, inverse, weights, counts, offsets, gy, gw, T, H, E, K, R
    assert lib.moe_combine_backward(A, A, 7, A, A, A, A, A, A, 4, 64, 8, 2, 8, None) == 1
    assert lib.moe_combine_backward(A, A, 2, A, A, A, A, A, A, 4, 64, 8, 2, 7, None) == 1
    assert lib.moe_combine_backward(A, A, 2, A, A, None, A, A, A, 4, 64, 8, 2, 8, None) == 1
    assert lib.moe_combine_backward(A, A, 2, A, A, A, A, A, A, 4, 64, 65, 2, 8, None) == 2
    assert lib.moe_combine_backward(A + 1, A, 2, A, A, A, A, A, A, 4, 64, 8, 2, 8, None) == 1
    assert lib.moe_combine_backward(A, A, 2, A, A, A, A, A, A, 0, 64, 8, 2, 0, None) == 0
    assert lib.moe_dispatch_backward(A, 2, A, A, 4, 64, 9, 36, None) == 2
    assert lib.moe_dispatch_backward(A, 2, None, A, 4, 64, 2, 8, None) == 1
    assert lib.moe_dispatch_backward(A, 2, A, A, 4, 64, 2, 7, None) == 1
    assert lib.moe_dispatch_backward(A, 2, A, A, 0, 64, 2, 0, None) == 0
    table = lib.moe_adapter_table_bytes(4, 3)
    assert table > 0 and lib.moe_adapter_table_bytes(4, 4097) == -1 and lib.moe_adapter_table_bytes(1 << 25, 3) == -1
    assert lib.moe_adapter_group(A, A, table - 1, 4, 3, None) == 4
    assert lib.moe_adapter_group(None, A, table, 4, 3, None) == 1
    assert lib.moe_adapter_group(A, A + 4, table, 4, 3, None) == 1
    assert lib.moe_adapter_group(A, A, table, 4, 0, None) == 2
    assert lib.moe_low_rank_scratch_bytes(4, 64, 32, 129, 3, 0) == -1
    assert lib.moe_low_rank_scratch_bytes(4, 64, 32, 8, 3, 0) == 0  # a small batch: one launch, nothing handed over
    need = lib.moe_low_rank_scratch_bytes(4, 64, 32, 40, 3, 0)
    assert need == 4 * 40 * 4  # one slice of 64: tokens * rank sums

    def add(x=A, base=A, out=A, nbytes=need, table_bytes=table, hidden=64, width=32, rank=40, tokens=4):
        return lib.moe_low_rank_add(x, A, A, A, A, table_bytes, base, out, None, A, nbytes, tokens, hidden, width, rank,
                                    3, None)

    assert add(hidden=60) == 2 and add(width=36) == 2 and add(rank=0) == 2 and add(rank=129) == 2
    assert add(nbytes=need - 1) == 4 and add(table_bytes=table - 4) == 4
    assert add(x=None) == 1 and add(out=None) == 1 and add(x=A + 8) == 1 and add(base=A + 8) == 1
    need = lib.moe_low_rank_scratch_bytes(4, 64, 32, 8, 3, 1)

    def back(hidden_in=A, dtype=0, nbytes=need, grad=A, gx=A):
        return lib.moe_low_rank_backward(grad, A, A, A, A, A, table, hidden_in, A, gx, A, A, dtype, A, nbytes, 4, 64, 32,
                                         8, 3, None)

    assert back(dtype=1) == 1 and back(hidden_in=None) == 1 and back(nbytes=need - 1) == 4
    assert back(grad=None) == 1 and back(gx=A + 8) == 1
