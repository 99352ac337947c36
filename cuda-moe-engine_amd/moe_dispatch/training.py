"""The router's training losses, and the gradients of the router and the transport.

The forward path's kernels (``MoEBlock.route``, ``ops.dispatch``, ``ops.combine``) record
no autograd graph. These operators are their training side, on the kernels of
``libmoe_hip.so``, as plain calls on tensors:

* ``router_loss``: balance loss, z loss and per-expert counts of a routed batch;
* ``route_logits_backward``: the gradient of the logits, from the losses' and the
  routing weights' gradients;
* ``route_backward``: that, and behind it the gradients of x, router weight and bias;
* ``combine_backward`` and ``dispatch_backward``: the transport's gradients.

``moe_dispatch.autograd`` wraps them for ``loss.backward()``. Nothing here has a
counterpart in the reference, which is forward-only.

Each call checks its tensors on the host (``ValueError`` for shapes, devices and layouts,
``TypeError`` for dtypes, ``RuntimeError`` without a GPU), launches on the current stream
of the tensors' device and does not synchronise. Results are new tensors. Every sum has
one order: results do not vary from call to call.
"""

from contextlib import nullcontext
from functools import lru_cache
from typing import NamedTuple

import torch

from ._extension import DTYPE_CODES, current_stream_handle, get_extension
from .workspace import MAX_EXPERTS, MAX_TOPK

MAX_ROUTED = 2**21  # tokens of route_backward

_CURRENT = nullcontext()
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def on_device(device):
    """Makes ``device`` current where it is not: streams and launches go by the current device."""
    return _CURRENT if device.index == _current_device() else torch.cuda.device(device)


def require_tensor(t, name, shape, dtype, device):
    """The checks every operand shares. A call on small tensors is host work first: the
    passing case is a few comparisons, and only a failing one finds out what to say."""
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device
            and t.is_contiguous()):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {list(shape)}, got {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    raise ValueError(f"{name} must be contiguous")


def shape_of(t, name, dims):
    shape = t.shape if isinstance(t, torch.Tensor) else None
    if shape is None:
        raise TypeError(f"{name} must be a tensor")
    if len(shape) != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got shape {list(shape)}")
    return shape


def refuse_autograd(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("this operator records no autograd graph: detach its inputs, call it under no_grad, "
                                 "or use moe_dispatch.autograd")


def require_gpu(t):
    if not t.is_cuda:
        raise RuntimeError("training operators require an AMD GPU")


def _ptr(t):
    return None if t is None else t.data_ptr()


@lru_cache(maxsize=1024)
def _loss_scratch_bytes(tokens, experts):
    return get_extension().lib.moe_router_loss_scratch_bytes(tokens, experts)


@lru_cache(maxsize=1024)
def _route_scratch_bytes(tokens, hidden, experts):
    return get_extension().lib.moe_route_backward_scratch_bytes(tokens, hidden, experts)


class RouterLoss(NamedTuple):
    """``losses`` fp32 [2] (balance, z) and ``stats`` int32 [E + 1] (per-expert counts of the
    valid tokens' assignments, then the number of valid tokens)."""

    losses: torch.Tensor
    stats: torch.Tensor

    @property
    def balance(self):
        return self.losses[0]

    @property
    def z(self):
        return self.losses[1]

    @property
    def counts(self):
        return self.stats[:-1]


def _check_routed(logits, expert_ids, bias, mask):
    tokens, experts = shape_of(logits, "logits", 2)
    device = logits.device
    if logits.dtype is not torch.float32 or not logits.is_contiguous():
        require_tensor(logits, "logits", logits.shape, torch.float32, device)
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError("logits must have 1..64 experts")
    rows, topk = shape_of(expert_ids, "expert_ids", 2)
    if (rows != tokens or expert_ids.dtype is not torch.int32 or expert_ids.device != device
            or not expert_ids.is_contiguous()):
        require_tensor(expert_ids, "expert_ids", (tokens, topk), torch.int32, device)
    if not 1 <= topk <= MAX_TOPK:
        raise ValueError("topk must be in 1..8")
    if tokens * max(experts, topk) > 2**31 - 1:
        raise ValueError("tokens*experts and tokens*topk must fit int32")
    if bias is not None:
        require_tensor(bias, "bias", (experts,), torch.float32, device)
    if mask is not None:
        require_tensor(mask, "mask", (tokens,), torch.bool, device)
    return tokens, experts, topk, device


def router_loss(logits, expert_ids, bias=None, *, mask=None):
    """Balance loss, z loss and per-expert counts of a routed batch.

    ``logits`` fp32 [T, E] (without the bias), ``expert_ids`` int32 [T, K] as the router
    chose them on ``logits + bias``, ``mask`` bool [T] false for padding tokens. With p the
    softmax of ``logits + bias``, N the valid tokens and c_e their assignments to expert e:

    * balance = E * sum_e (c_e / (N K)) * mean_t p_te, 1 where both are uniform;
    * z = mean_t (log sum_e exp(logits + bias)_te)^2.

    Both are 0 without valid tokens. Ids out of range count nowhere. Logits may be -inf (a
    token of none but -inf adds nothing to the losses); +inf or NaN ones of a valid token
    show in the losses.
    """
    tokens, experts, topk, device = _check_routed(logits, expert_ids, bias, mask)
    require_gpu(logits)
    refuse_autograd(logits, bias)
    lib = get_extension().lib
    with on_device(device):
        losses = logits.new_empty(2)
        stats = expert_ids.new_empty(experts + 1)
        need = _loss_scratch_bytes(tokens, experts)
        scratch = logits.new_empty(need // 4) if need else None
        lib.check(lib.moe_router_loss(
            logits.data_ptr(), _ptr(bias), expert_ids.data_ptr(), _ptr(mask), losses.data_ptr(), stats.data_ptr(),
            _ptr(scratch), need, tokens, experts, topk, current_stream_handle(device.index)), "router_loss")
    return RouterLoss(losses, stats)


def _check_gradients(logits, expert_ids, loss, grad_losses, grad_weights):
    if grad_losses is not None:
        require_tensor(grad_losses, "grad_losses", (2,), torch.float32, logits.device)
        if not isinstance(loss, RouterLoss):
            raise TypeError("grad_losses needs the forward's RouterLoss as loss")
        require_tensor(loss.stats, "loss.stats", (logits.shape[1] + 1,), torch.int32, logits.device)
    if grad_weights is not None:
        require_tensor(grad_weights, "grad_weights", expert_ids.shape, torch.float32, logits.device)


def route_logits_backward(logits, expert_ids, bias=None, *, mask=None, loss=None, grad_losses=None, grad_weights=None):
    """The gradient of the logits, fp32 [T, E].

    ``grad_losses`` fp32 [2]: the gradients of ``loss.balance`` and ``loss.z``, with ``loss``
    the ``router_loss`` of the same logits, ids, bias and mask. ``grad_weights`` fp32 [T, K]:
    the routing weights' gradient. Either may be None (0). The routing weights are the
    softmax of the chosen logits (K = 1: the constant 1, without a gradient); the counts in
    the balance loss are constants. Masked tokens get 0.
    """
    tokens, experts, topk, device = _check_routed(logits, expert_ids, bias, mask)
    _check_gradients(logits, expert_ids, loss, grad_losses, grad_weights)
    require_gpu(logits)
    refuse_autograd(logits, bias, grad_losses, grad_weights)
    lib = get_extension().lib
    with on_device(device):
        grad_logits = torch.empty_like(logits)
        lib.check(lib.moe_router_logits_backward(
            logits.data_ptr(), _ptr(bias), expert_ids.data_ptr(), _ptr(mask),
            loss.stats.data_ptr() if loss is not None else None, _ptr(grad_losses), _ptr(grad_weights),
            grad_logits.data_ptr(), tokens, experts, topk,
            current_stream_handle(device.index)), "route_logits_backward")
    return grad_logits


def route_backward(x, router_weight, logits, expert_ids, bias=None, *, mask=None, loss=None, grad_losses=None,
                   grad_weights=None, grad_x=None, gradients=(True, True, True)):
    """Gradients of x, router weight and bias: ``(grad_x, grad_router_weight, grad_bias)``.

    x bf16 [T, H] and router_weight fp32 [E, H] are the router's inputs (H a multiple of 8),
    T is up to 2^21, the rest is ``route_logits_backward``'s. ``grad_x`` bf16 [T, H] is x's gradient along its
    other paths: the result is the sum, rounded once. grad_router_weight [E, H] and grad_bias
    [E] are fp32. A masked token's row of x may hold anything. ``gradients``: which of the
    three are wanted; the others are None and are not computed.
    """
    tokens, experts, topk, device = _check_routed(logits, expert_ids, bias, mask)
    _check_gradients(logits, expert_ids, loss, grad_losses, grad_weights)
    hidden = shape_of(x, "x", 2)[1]
    require_tensor(x, "x", (tokens, hidden), torch.bfloat16, device)
    if hidden < 8 or hidden % 8 or hidden > 2**20:
        raise ValueError("hidden must be a multiple of 8 up to 2^20")
    if tokens > MAX_ROUTED:
        raise ValueError("route_backward takes up to 2^21 tokens")
    require_tensor(router_weight, "router_weight", (experts, hidden), torch.float32, device)
    if grad_x is not None:
        require_tensor(grad_x, "grad_x", (tokens, hidden), torch.bfloat16, device)
    require_gpu(x)
    refuse_autograd(x, router_weight, logits, bias, grad_losses, grad_weights, grad_x)
    lib = get_extension().lib
    with on_device(device):
        want_x, want_weight, want_bias = gradients
        out_x = torch.empty_like(x) if want_x else None
        grad_router_weight = torch.empty_like(router_weight) if want_weight else None
        grad_bias = logits.new_empty(experts) if want_bias else None
        if tokens == 0:
            for t in (grad_router_weight, grad_bias):
                if t is not None:
                    t.zero_()
            return out_x, grad_router_weight, grad_bias
        need = _route_scratch_bytes(tokens, hidden, experts)
        scratch = logits.new_empty(need // 4)
        lib.check(lib.moe_route_backward(
            x.data_ptr(), router_weight.data_ptr(), logits.data_ptr(), _ptr(bias), expert_ids.data_ptr(), _ptr(mask),
            loss.stats.data_ptr() if loss is not None else None, _ptr(grad_losses), _ptr(grad_weights), _ptr(grad_x),
            _ptr(out_x), _ptr(grad_router_weight), _ptr(grad_bias), scratch.data_ptr(), need, tokens,
            hidden, experts, topk, current_stream_handle(device.index)), "route_backward")
    return out_x, grad_router_weight, grad_bias


def combine_backward(grad_output, expert_output, batch, weights):
    """Gradients of ``combine(expert_output, batch, weights)``: ``(grad_expert_output, grad_weights)``.

    ``batch`` is the ``PackedTokens`` of the dispatch, its workspace not dispatched again
    since (``RuntimeError``). grad_expert_output has the packed rows' shape and dtype; rows that hold no
    assignment (padding) are zero. grad_weights is fp32 [T, K].
    """
    batch.require_current()
    workspace = batch.workspace
    tokens, hidden, experts, topk = workspace.shape
    dtype, device = workspace.dtype, workspace.device
    packed = batch.packed.shape
    require_tensor(grad_output, "grad_output", (tokens, hidden), dtype, device)
    require_tensor(expert_output, "expert_output", packed, dtype, device)
    require_tensor(weights, "weights", (tokens, topk), torch.float32, device)
    refuse_autograd(grad_output, expert_output, weights)
    lib = get_extension().lib
    with on_device(device):
        grad_expert = torch.empty_like(expert_output)
        grad_weights = torch.empty_like(weights)
        lib.check(lib.moe_combine_backward(
            grad_output.data_ptr(), expert_output.data_ptr(), DTYPE_CODES[dtype], batch.inverse.data_ptr(),
            weights.data_ptr(), batch.counts.data_ptr(), batch.offsets.data_ptr(), grad_expert.data_ptr(),
            grad_weights.data_ptr(), tokens, hidden, experts, topk, packed[0], current_stream_handle(device.index)),
            "combine_backward")
    return grad_expert, grad_weights


def dispatch_backward(grad_packed, batch):
    """Gradient of ``dispatch(x, ...)``: [T, H], each token's K packed rows' gradients summed
    in fp32 in k order and rounded once. ``batch`` as in ``combine_backward``."""
    batch.require_current()
    workspace = batch.workspace
    tokens, hidden, _, topk = workspace.shape
    dtype, device = workspace.dtype, workspace.device
    packed = batch.packed.shape
    require_tensor(grad_packed, "grad_packed", packed, dtype, device)
    refuse_autograd(grad_packed)
    lib = get_extension().lib
    with on_device(device):
        grad_x = grad_packed.new_empty((tokens, hidden))
        lib.check(lib.moe_dispatch_backward(
            grad_packed.data_ptr(), DTYPE_CODES[dtype], batch.inverse.data_ptr(), grad_x.data_ptr(), tokens, hidden,
            topk, packed[0], current_stream_handle(device.index)), "dispatch_backward")
    return grad_x
