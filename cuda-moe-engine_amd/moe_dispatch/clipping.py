"""The global norm of a model's gradients, and clipping by it.

What the gradients of ``training``, ``adapters`` and ``autograd`` go through before an
optimizer step, whatever tensors they lie in: one norm over all of them, and one factor.
No counterpart in the reference.

Checks, streams and errors are those of ``moe_dispatch.training``.
"""

from array import array

import torch

from ._extension import DTYPE_CODES, current_stream_handle, get_extension
from ._lib import CLIP_ARGS
from .training import refuse_autograd

MAX_TENSORS = 2**16
MAX_ELEMENTS = 2**40
_SCRATCH_DOUBLES = 2048


def _check_list(tensors, name, device):
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}[{i}] must be a tensor")
        if t.dtype not in DTYPE_CODES:
            raise TypeError(f"{name}[{i}] must be float32, float16 or bfloat16, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name}[{i}] must be on {device}")
        if not t.is_contiguous():
            raise ValueError(f"{name}[{i}] must be contiguous")


def clip_gradients(grads, max_norm, *, outputs=None):
    """Scales gradients so that their global norm is at most ``max_norm``; returns the norm
    before, fp32 [], on the device.

        norm = sqrt(sum of all squares),   g <- g * min(1, max_norm / (norm + 1e-6))

    ``grads`` is a list of contiguous fp32, fp16 or bf16 tensors of any shapes on one GPU, no
    two of which share memory; with ``outputs`` (tensors of the same shapes and types, each the
    gradient itself or apart from all others) they are read only and the results go there. Sums are 64
    bits, in an order that the sizes fix; a result is rounded once. A norm that is infinite
    or NaN leaves the values as they are, so that a program can look at the norm and skip the step.
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
    _check_list(grads, "grads", device)
    elements = array("q", [t.numel() for t in grads])
    if sum(elements) > MAX_ELEMENTS:
        raise ValueError("takes up to 2^40 elements")
    addresses = array("Q", [t.data_ptr() for t in grads])
    sizes = [t.element_size() for t in grads]
    ranges = [(a, a + n * s) for a, n, s in zip(addresses, elements, sizes) if n]
    if outputs is None:
        out_addresses = addresses
    else:
        outputs = list(outputs)
        if len(outputs) != len(grads):
            raise ValueError("outputs must have a tensor for each gradient")
        _check_list(outputs, "outputs", device)
        for i, (g, o) in enumerate(zip(grads, outputs)):
            if o.shape != g.shape or o.dtype is not g.dtype:
                raise ValueError(f"outputs[{i}] must have its gradient's shape and type")
        out_addresses = array("Q", [t.data_ptr() for t in outputs])
        ranges += [(a, a + n * s) for a, b, n, s in zip(out_addresses, addresses, elements, sizes) if n and a != b]
    ranges.sort()
    if any(a[1] > b[0] for a, b in zip(ranges, ranges[1:])):
        raise ValueError("gradients and outputs must not share memory (a gradient may be its own output)")
    if not first.is_cuda:
        raise RuntimeError("clip_gradients requires an AMD GPU")
    refuse_autograd(*grads, *(outputs or ()))
    dtypes = array("q", [DTYPE_CODES[t.dtype] for t in grads])
    lib = get_extension().lib
    with torch.cuda.device(device):
        norm = torch.empty((), dtype=torch.float32, device=device)
        scratch = torch.empty(_SCRATCH_DOUBLES, dtype=torch.float64, device=device)
        lib.check(lib.moe_clip_gradients(CLIP_ARGS(
            addresses.buffer_info()[0], out_addresses.buffer_info()[0], elements.buffer_info()[0],
            dtypes.buffer_info()[0], len(grads), norm.data_ptr(), scratch.data_ptr(), _SCRATCH_DOUBLES * 8,
            float(max_norm)), current_stream_handle(device.index)), "clip_gradients")
    return norm
