"""The global norm of a model's gradients, and clipping by it.

What the gradients of ``training``, ``adapters`` and ``autograd`` go through before an
optimizer step, whatever tensors they lie in: one norm over all of them, and one factor.
No counterpart in the reference.

Checks, streams and errors are those of ``moe_dispatch.training``.
"""

from array import array
from operator import attrgetter

import torch

from ._extension import DTYPE_CODES, current_stream_handle, get_extension
from ._lib import CLIP_ARGS, load_library
from .training import on_device, refuse_autograd

MAX_TENSORS = 2**16
MAX_ELEMENTS = 2**40
_SCRATCH_DOUBLES = 2048


_Tensor = torch.Tensor
_dtype_of, _wants_gradient = attrgetter("dtype"), attrgetter("requires_grad")


def _refuse_list(tensors, name, device):
    """Says what is wrong with a list that the quick checks did not pass."""
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}[{i}] must be a tensor")
        if t.dtype not in DTYPE_CODES:
            raise TypeError(f"{name}[{i}] must be float32, float16 or bfloat16, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name}[{i}] must be on {device}")
        if not t.is_contiguous():
            raise ValueError(f"{name}[{i}] must be contiguous")
    raise ValueError(f"{name} must be contiguous tensors on {device}")


def _describe(tensors, name, device):
    """(type codes, elements, addresses) of the tensors. A step's list is long and host work
    first: each property is one pass of a C method over it."""
    try:
        kinds = list(map(_dtype_of, tensors))
        code = DTYPE_CODES[kinds[0]]
        same = kinds.count(kinds[0]) == len(kinds)
        dtypes = array("q", [code]) * len(kinds) if same else array("q", [DTYPE_CODES[kind] for kind in kinds])
        # A tensor that is on no GPU has the index -1 (the CPU, or a device without storage).
        index = device.index if device.type == "cuda" else -1
        if list(map(_Tensor.get_device, tensors)).count(index) != len(tensors) or not all(
                map(_Tensor.is_contiguous, tensors)):
            _refuse_list(tensors, name, device)
        return dtypes, array("q", map(_Tensor.numel, tensors)), array("Q", map(_Tensor.data_ptr, tensors))
    except (KeyError, TypeError, AttributeError, RuntimeError):
        _refuse_list(tensors, name, device)


def clip_gradients(grads, max_norm, *, outputs=None):
    """Scales gradients so that their global norm is at most ``max_norm``; returns the norm
    before, fp32 [], on the device.

        norm = sqrt(sum of all squares),   g <- g * min(1, max_norm / (norm + 1e-6))

    ``grads`` is a list of contiguous fp32, fp16 or bf16 tensors of any shapes on one GPU, no
    two of which share memory; with ``outputs`` (a tensor of the same type and size for each, the
    gradient itself or apart from all others) they are read only and the results go there. Sums are 64
    bits, in an order that the sizes fix; the factor and its products are fp32, rounded once to a
    narrower type. Gradients that hold an infinity or NaN stay as they are, so that a program can
    look at the norm and skip the step. The norm of finite gradients may pass fp32 (3.4e38): it is
    returned as infinite, and the values are scaled by what it is.
    """
    grads = list(grads)
    if not grads:
        raise ValueError("clip_gradients needs at least one tensor")
    if len(grads) > MAX_TENSORS:
        raise ValueError("takes up to 2^16 tensors")
    if not max_norm > 0:
        raise ValueError("max_norm must be positive")
    first = grads[0]
    if not isinstance(first, torch.Tensor):
        raise TypeError("grads[0] must be a tensor")
    device = first.device
    dtypes, elements, addresses = _describe(grads, "grads", device)
    out_addresses = addresses
    if sum(elements) > MAX_ELEMENTS:
        raise ValueError("takes up to 2^40 elements")
    if outputs is not None:
        outputs = list(outputs)
        if len(outputs) != len(grads):
            raise ValueError("outputs must have a tensor for each gradient")
        out_dtypes, out_elements, out_addresses = _describe(outputs, "outputs", device)
        if out_dtypes != dtypes or out_elements != elements:
            raise ValueError("outputs must have their gradients' sizes and types")
    count = len(grads)
    room = array("Q", bytes(32 * count))
    pointers = [a.buffer_info()[0] for a in (addresses, out_addresses, elements, dtypes, room)]
    library = load_library()
    if library.moe_clip_overlap(*pointers, count):
        raise ValueError("gradients and outputs must not share memory (a gradient may be its own output)")
    if not first.is_cuda:
        raise RuntimeError("clip_gradients requires an AMD GPU")
    if torch.is_grad_enabled() and (any(map(_wants_gradient, grads)) or (outputs and any(map(_wants_gradient, outputs)))):
        refuse_autograd(*grads, *(outputs or ()))
    lib = get_extension().lib
    with on_device(device):
        norm = torch.empty((), dtype=torch.float32, device=device)
        scratch = torch.empty(_SCRATCH_DOUBLES, dtype=torch.float64, device=device)
        lib.check(lib.moe_clip_gradients(CLIP_ARGS(
            *pointers[:4], count, norm.data_ptr(), scratch.data_ptr(), _SCRATCH_DOUBLES * 8, float(max_norm)),
            current_stream_handle(device.index)), "clip_gradients")
    return norm
