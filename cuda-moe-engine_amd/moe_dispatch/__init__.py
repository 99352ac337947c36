"""MI355X-native MoE feed-forward engine with the ``moe_dispatch`` API.

Operators on hand-written gfx950 HIP kernels, loaded from the prebuilt
``libmoe_hip.so`` on first GPU use; importing the package never compiles or
touches the GPU. The forward's public names follow the reference package
(``src/moe_dispatch/__init__.py:6-23``); the router's losses, the gradients of
router and transport (``training``), the low-rank adapters (``adapters``) and what stands
around the experts (``norms``, ``scored``, ``dense``, ``clipping``) have no counterpart there.
"""

from importlib import import_module

__version__ = "0.1.0"
__all__ = ["dispatch", "combine", "PackedTokens", "CudaWorkspace", "TorchWorkspace", "MoEBlock",
           "MoEConfig", "RouterLoss", "router_loss", "route_logits_backward", "route_backward", "combine_backward",
           "dispatch_backward", "AdapterGroups", "low_rank_add", "low_rank_backward", "QuantizedRows", "rms_norm",
           "rms_norm_backward", "quantize_rows", "route_scored", "route_scored_backward", "linear", "clip_gradients"]
_EXPORTS = {
    "dispatch": (".ops", "dispatch"),
    "combine": (".ops", "combine"),
    "PackedTokens": (".ops", "PackedTokens"),
    "CudaWorkspace": (".workspace", "CudaWorkspace"),
    "TorchWorkspace": (".reference", "TorchWorkspace"),
    "MoEBlock": (".layer", "MoEBlock"),
    "MoEConfig": (".layer", "MoEConfig"),
    "RouterLoss": (".training", "RouterLoss"),
    "router_loss": (".training", "router_loss"),
    "route_logits_backward": (".training", "route_logits_backward"),
    "route_backward": (".training", "route_backward"),
    "combine_backward": (".training", "combine_backward"),
    "dispatch_backward": (".training", "dispatch_backward"),
    "AdapterGroups": (".adapters", "AdapterGroups"),
    "low_rank_add": (".adapters", "low_rank_add"),
    "low_rank_backward": (".adapters", "low_rank_backward"),
    "QuantizedRows": (".norms", "QuantizedRows"),
    "rms_norm": (".norms", "rms_norm"),
    "rms_norm_backward": (".norms", "rms_norm_backward"),
    "quantize_rows": (".norms", "quantize_rows"),
    "route_scored": (".scored", "route_scored"),
    "route_scored_backward": (".scored", "route_scored_backward"),
    "linear": (".dense", "linear"),
    "clip_gradients": (".clipping", "clip_gradients"),
}


def __getattr__(name):
    if name not in _EXPORTS:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    module, symbol = _EXPORTS[name]
    value = getattr(import_module(module, __name__), symbol)
    globals()[name] = value
    return value
