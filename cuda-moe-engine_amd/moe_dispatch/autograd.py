"""The training operators as differentiable functions, for ``loss.backward()``.

``route``, ``dispatch``, ``combine``, ``low_rank_add``, ``rms_norm`` and ``route_scored`` run
the forward kernels and record the gradients of ``training``, ``adapters``, ``norms`` and
``scored``. Each returns new tensors, so that several layers and micro-batches may be in
flight; none keeps a buffer for the next call.
Gradients are first order (a second differentiation raises).

They are eager: under graph capture they raise, since a backward pass recorded beside a
live eager graph of the same leaves is more than torch survives. Capture the plain calls
of those modules instead; they take buffers in and give gradients out.
"""

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import adapters as _adapters
from . import norms as _norms
from . import ops as _ops
from . import scored as _scored
from . import training as _training
from ._extension import get_extension


def _eager_only():
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("moe_dispatch.autograd is eager: capture the calls of moe_dispatch.training and "
                           "moe_dispatch.adapters (or norms, scored) instead")


def _rows(grad):
    """A gradient as the kernels take it: contiguous, and 16-byte aligned where it was cut
    out of a larger one."""
    grad = grad.contiguous()
    return grad if grad.data_ptr() % 16 == 0 else grad.clone()


class Routed(NamedTuple):
    """``weights`` fp32 [T, K] and ``losses`` fp32 [2] (balance, z) carry gradients;
    ``ids`` int32 [T, K], ``counts`` int32 [E] do not."""

    weights: torch.Tensor
    losses: torch.Tensor
    ids: torch.Tensor
    counts: torch.Tensor


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, router_weight, bias, topk, mask):
        tokens, experts = x.shape[0], router_weight.shape[0]
        shape = (tokens, topk)
        ids = torch.empty(shape, dtype=torch.int32, device=x.device)
        weights = torch.empty(shape, dtype=torch.float32, device=x.device)
        logits = torch.empty((tokens, experts), dtype=torch.float32, device=x.device)
        with _training.on_device(x.device):
            get_extension().router_fused_out(x, router_weight, bias, ids, None, weights, logits=logits)
        loss = _training.router_loss(logits, ids, bias, mask=mask)
        ctx.save_for_backward(x, router_weight, bias, logits, ids, mask, loss.stats)
        ctx.mark_non_differentiable(ids, loss.stats)
        ctx.set_materialize_grads(False)
        return weights, loss.losses, ids, loss.stats

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_weights, grad_losses, _ids, _stats):
        _eager_only()
        if grad_weights is None and grad_losses is None:
            return None, None, None, None, None
        x, router_weight, bias, logits, ids, mask, stats = ctx.saved_tensors
        grads = _training.route_backward(
            x, router_weight, logits, ids, bias, mask=mask, loss=_training.RouterLoss(None, stats),
            grad_losses=None if grad_losses is None else grad_losses.contiguous(),
            grad_weights=None if grad_weights is None else grad_weights.contiguous(),
            gradients=ctx.needs_input_grad[:3])
        return (*grads, None, None)


def route(x, router_weight, bias, topk, *, mask=None):
    """Routes x bf16 [T, H] by router_weight fp32 [E, H] and bias fp32 [E] through the fused
    router, with the losses of ``training.router_loss``: ``Routed``. T is at least 1, and up to
    2^21 where a gradient is recorded. ``mask`` bool [T] is false for padding tokens: they count
    in no loss and pass no gradient on, though they get ids and weights as any token."""
    _eager_only()
    _training.shape_of(x, "x", 2)
    experts = _training.shape_of(router_weight, "router_weight", 2)[0]
    if x.shape[0] == 0:
        raise ValueError("route needs at least one token")
    if x.shape[0] > _training.MAX_ROUTED and torch.is_grad_enabled() and any(
            isinstance(t, torch.Tensor) and t.requires_grad for t in (x, router_weight, bias)):
        raise ValueError("route records gradients of up to 2^21 tokens")
    if not isinstance(topk, int) or not 1 <= topk <= min(experts, _training.MAX_TOPK):
        raise ValueError("topk must be in 1..min(experts, 8)")
    weights, losses, ids, stats = _Route.apply(x, router_weight, bias, topk, mask)
    return Routed(weights, losses, ids, stats[:-1])


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, batch):
        ctx.batch = batch
        return batch.packed.detach()

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_packed):
        _eager_only()
        return _training.dispatch_backward(grad_packed.contiguous(), ctx.batch), None


def dispatch(x, expert_ids, experts, *, alignment=1):
    """``ops.dispatch`` into a workspace of its own: ``(packed, batch)``, packed rows with
    their gradient to x and the ``PackedTokens`` for ``combine``. Rows without an assignment
    are zero. As there, the id range is checked on the host, which waits for the stream."""
    _eager_only()
    x_data = x.detach()
    with torch.no_grad():
        _ops.validate_inputs(x_data, expert_ids, experts)
        if not x.is_cuda:
            raise RuntimeError("dispatch requires a GPU")
        workspace = _ops.CudaWorkspace(x.shape[0], x.shape[1], experts, expert_ids.shape[1], x.dtype, device=x.device,
                                       alignment=alignment)
        # Rows behind the last span: a program's experts may run over all of them.
        if workspace.capacity_rows > expert_ids.numel():
            workspace.packed.zero_()
    batch = _ops.dispatch(x_data, expert_ids, experts, workspace=workspace)
    return _Dispatch.apply(x, batch), batch


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, expert_output, weights, batch):
        tokens, hidden, _, _ = batch.workspace.shape
        output = expert_output.new_empty((tokens, hidden))
        with _training.on_device(expert_output.device):
            batch.workspace.extension.combine_out(expert_output, batch.inverse, weights, output)
        ctx.save_for_backward(expert_output, weights)
        ctx.batch = batch
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        _eager_only()
        expert_output, weights = ctx.saved_tensors
        grads = _training.combine_backward(grad_output.contiguous(), expert_output, ctx.batch, weights)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None)


def combine(expert_output, batch, weights):
    """The weighted combine of ``batch``'s packed rows, [T, H], with gradients to the rows
    and to the fp32 weights [T, K]. The batch's workspace must not be dispatched again before
    the backward pass has run (``RuntimeError``)."""
    _eager_only()
    batch.require_current()
    _training.require_tensor(expert_output, "expert_output", batch.packed.shape, batch.workspace.dtype,
                             batch.workspace.device)
    _training.require_tensor(weights, "weights", batch.inverse.shape, torch.float32, batch.workspace.device)
    return _Combine.apply(expert_output, weights, batch)


class _LowRankAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, base, x, down, up, groups, scales):
        output, hidden = _adapters.low_rank_add(base, x, down, up, groups, scales=scales, return_hidden=True)
        ctx.save_for_backward(x, down, up, hidden.values, scales)
        ctx.groups, ctx.assignment = groups, hidden.assignment
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        _eager_only()
        x, down, up, values, scales = ctx.saved_tensors
        _, need_x, need_down, need_up, _, _ = ctx.needs_input_grad
        grads = None, None, None
        if need_x or need_down or need_up:
            hidden = _adapters.LowRankHidden(values, ctx.groups, ctx.assignment)
            grads = _adapters.low_rank_backward(_rows(grad_output), x, down, up, ctx.groups, scales=scales,
                                                hidden=hidden, grad_dtype=down.dtype,
                                                gradients=(need_x, need_down, need_up))
        return (grad_output if ctx.needs_input_grad[0] else None, *grads, None, None)


def low_rank_add(base, x, down, up, groups, *, scales=None):
    """``adapters.low_rank_add`` with gradients to base, x, down and up (bf16). The groups
    must hold the same assignment when the backward pass runs."""
    _eager_only()
    if scales is not None and scales.requires_grad:
        raise ValueError("scales get no gradient; detach them")
    return _LowRankAdd.apply(base, x, down, up, groups, scales)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        normed = _norms.rms_norm(x, weight, residual=residual, eps=eps, return_rstd=True)
        ctx.save_for_backward(x if residual is None else normed.total, weight, normed.rstd)
        ctx.set_materialize_grads(False)
        return normed.output, normed.total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output, grad_total):
        _eager_only()
        total, weight, rstd = ctx.saved_tensors
        need_x, need_weight, need_residual, _ = ctx.needs_input_grad
        if grad_output is None:
            return (grad_total if need_x else None, None, grad_total if need_residual else None, None)
        grad_x, grad_weight = _norms.rms_norm_backward(
            grad_output.contiguous(), total, weight, rstd, grad_x=None if grad_total is None else grad_total.contiguous(),
            gradients=(need_x or need_residual, need_weight))
        if grad_weight is not None:
            grad_weight = grad_weight.to(weight.dtype)
        return grad_x if need_x else None, grad_weight, grad_x if need_residual else None, None


def rms_norm(x, weight=None, *, residual=None, eps=1e-6):
    """``norms.rms_norm`` with gradients to x, weight and residual: ``(output, total)``, total =
    x + residual (None without a residual), to be the next residual. The gradient takes the normed
    rows as total holds them, rounded to their type."""
    _eager_only()
    return _RmsNorm.apply(x, weight, residual, eps)


class _RouteScored(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, options, choice):
        ids, weights = _scored.route_scored(logits, topk, **options, **choice)
        ctx.save_for_backward(logits, ids)
        ctx.options = options
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    @once_differentiable
    def backward(ctx, _ids, grad_weights):
        _eager_only()
        logits, ids = ctx.saved_tensors
        return _scored.route_scored_backward(grad_weights.contiguous(), logits, ids, **ctx.options), None, None, None


def route_scored(logits, topk, *, scoring="softmax", bias=None, groups=1, top_groups=1, group_best=2,
                 renormalize=True, scale=1.0):
    """``scored.route_scored`` with the weights' gradient to the logits: ``(ids, weights)``."""
    _eager_only()
    if isinstance(bias, torch.Tensor) and bias.requires_grad:
        raise ValueError("the selection bias gets no gradient; detach it")
    return _RouteScored.apply(logits, topk, {"scoring": scoring, "renormalize": renormalize, "scale": scale},
                              {"bias": bias, "groups": groups, "top_groups": top_groups, "group_best": group_best})
