"""Routing by scores: softmax or sigmoid, a selection bias, groups of experts, scaled weights.

``MoEBlock`` and ``autograd.route`` choose by the logits and weigh by the softmax of the
chosen ones. ``route_scored`` is for the other routers of mixture models: it takes logits
(``router_fused_out``'s, or any other product's, of up to 512 experts), and its ids and
weights go to ``dispatch`` and ``combine`` like theirs (which take up to 64 experts);
``route_scored_backward`` gives the logits' gradient. No counterpart in the reference.

Checks, streams and errors are those of ``moe_dispatch.training``.
"""

import torch

from ._extension import current_stream_handle, get_extension
from ._lib import ROUTE_SCORED_ARGS, ROUTE_SCORED_BACKWARD_ARGS
from .training import _ptr, on_device, refuse_autograd, require_gpu, require_tensor, shape_of
from .workspace import MAX_TOPK

MAX_SCORED_EXPERTS = 512
MAX_GROUPS = 64
MAX_TOKENS = 2**21
SCORINGS = ("softmax", "sigmoid")


def _check_logits(logits, topk, scoring, scale):
    tokens, experts = shape_of(logits, "logits", 2)
    require_tensor(logits, "logits", logits.shape, torch.float32, logits.device)
    if not 1 <= experts <= MAX_SCORED_EXPERTS:
        raise ValueError("logits must have 1..512 experts")
    if tokens > MAX_TOKENS:
        raise ValueError("takes up to 2^21 tokens")
    if not isinstance(topk, int) or not 1 <= topk <= MAX_TOPK:
        raise ValueError("topk must be in 1..8")
    if scoring not in SCORINGS:
        raise ValueError("scoring must be softmax or sigmoid")
    if not (hasattr(scale, "__float__") or hasattr(scale, "__index__")):
        raise TypeError("scale must be a number")
    return tokens, experts


def _check_choice(experts, topk, groups, top_groups, group_best):
    if not isinstance(groups, int) or not 1 <= groups <= MAX_GROUPS or experts % groups:
        raise ValueError("groups must be in 1..64 and divide the experts")
    if not isinstance(top_groups, int) or not 1 <= top_groups <= groups:
        raise ValueError("top_groups must be in 1..groups")
    if topk > top_groups * (experts // groups):
        raise ValueError("topk exceeds the experts of top_groups groups")
    if not hasattr(group_best, "__index__") or group_best not in (1, 2):
        raise ValueError("group_best must be 1 or 2")


def route_scored(logits, topk, *, scoring="softmax", bias=None, groups=1, top_groups=1, group_best=2,
                 renormalize=True, scale=1.0):
    """Experts and weights of each token: ``(ids int32 [T, K], weights fp32 [T, K])``.

    ``logits`` fp32 [T, E], E up to 512. With s the softmax or sigmoid of a token's logits:

    * an expert's key is s + ``bias`` (fp32 [E], finite: what balances the experts' load; it
      takes part in the choice only);
    * with ``groups`` > 1 the experts lie in that many equal consecutive groups. A group's score
      is the sum of its ``group_best`` (1 or 2) highest keys, and experts of the
      ``top_groups`` highest groups alone are chosen;
    * ids are the K highest keys, highest first, ties to the lower index. The choice is that of
      the exact keys, however fp32 rounds them;
    * weights are ``scale * s``, with ``renormalize`` divided by the sum of the chosen s: fp32, within about
      40 + 2 |l - l_top| roundings of 2^-24 (|l| for sigmoid without ``renormalize``), 0 below 2^-126.

    A logit of -inf takes an expert out: it is chosen, with weight 0, only where the token's
    groups have nothing else left. A NaN logit is out too and makes its token's weights NaN. So does
    +inf under softmax, where in the choice the experts with +inf have equal scores and the others 0.
    """
    tokens, experts = _check_logits(logits, topk, scoring, scale)
    _check_choice(experts, topk, groups, top_groups, group_best)
    device = logits.device
    if bias is not None:
        require_tensor(bias, "bias", (experts,), torch.float32, device)
    require_gpu(logits)
    refuse_autograd(logits, bias)
    lib = get_extension().lib
    with on_device(device):
        ids = logits.new_empty((tokens, topk), dtype=torch.int32)
        weights = logits.new_empty((tokens, topk))
        status = lib.moe_route_scored(ROUTE_SCORED_ARGS(
            logits.data_ptr(), _ptr(bias) or 0, ids.data_ptr(), weights.data_ptr(), tokens, experts, topk, groups,
            top_groups, group_best, scoring == "sigmoid", bool(renormalize), scale), current_stream_handle(device.index))
        if status:
            lib.check(status, "route_scored")
    return ids, weights


def route_scored_backward(grad_weights, logits, ids, *, scoring="softmax", renormalize=True, scale=1.0):
    """The gradient of the logits, fp32 [T, E], from the weights' (``grad_weights`` fp32 [T, K]).

    ``ids`` is what ``route_scored`` gave for these logits with the same ``scoring``,
    ``renormalize`` and ``scale``; the choice itself, and so the bias, has no gradient.
    """
    tokens, topk = shape_of(ids, "ids", 2)
    _, experts = _check_logits(logits, topk, scoring, scale)
    device = logits.device
    require_tensor(ids, "ids", (logits.shape[0], topk), torch.int32, device)
    require_tensor(grad_weights, "grad_weights", ids.shape, torch.float32, device)
    require_gpu(logits)
    refuse_autograd(grad_weights, logits)
    lib = get_extension().lib
    with on_device(device):
        grad_logits = torch.empty_like(logits)
        status = lib.moe_route_scored_backward(ROUTE_SCORED_BACKWARD_ARGS(
            grad_weights.data_ptr(), logits.data_ptr(), ids.data_ptr(), grad_logits.data_ptr(), tokens, experts, topk,
            scoring == "sigmoid", bool(renormalize), scale), current_stream_handle(device.index))
        if status:
            lib.check(status, "route_scored_backward")
    return grad_logits
