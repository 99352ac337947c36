"""Dense products with bias, activation and residual behind them, in bf16 and in 8 bits.

``experts.grouped_linear`` and the block's products are grouped over experts. ``linear`` is
for what stands beside them in a layer, a shared expert above all:

    gate_up = linear(normed, gate_up_weight, activation="swiglu")
    stream = linear(gate_up, down_weight, residual=routed)

with x and weight both bf16, or both ``norms.QuantizedRows`` (x as ``rms_norm(...,
quantize=True)`` or ``quantize_rows`` gives it, the weight quantized once when it is loaded).
Like the experts' products it is for inference: no gradient is recorded. No counterpart in the
reference.

Checks, streams and errors are those of ``moe_dispatch.training``.
"""

from functools import lru_cache

import torch

from ._extension import DTYPE_CODES, current_stream_handle, get_extension
from ._lib import LINEAR_ARGS
from .norms import E4M3, QuantizedRows
from .training import _ptr, on_device, refuse_autograd, require_gpu, require_tensor, shape_of

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "swiglu": 5}
MAX_TOKENS = 2**21
MAX_WIDTH = 2**20


@lru_cache(maxsize=1024)
def _scratch_bytes(tokens, hidden, width, activation, e4m3):
    return get_extension().lib.moe_linear_scratch_bytes(tokens, hidden, width, activation, e4m3)


def _row_stride(weight, name):
    """Elements from one weight row to the next: rows are contiguous and may be padded."""
    rows, hidden = weight.shape
    stride = weight.stride(0) if rows > 1 else hidden
    if (hidden > 1 and weight.stride(1) != 1) or stride < hidden or stride > 2 * MAX_WIDTH:
        raise ValueError(f"{name} must be contiguous, or have contiguous rows with padding between them")
    return stride


def linear(x, weight, bias=None, *, activation=None, residual=None, output=None):
    """``act(x weight^T + bias) + residual``: bf16 [T, N], rounded once from fp32.

    x [T, K] and weight [R, K] are bf16 or ``QuantizedRows``. ``activation`` is None, "relu",
    "silu", "gelu" (the erf form), "gelu_tanh" or "swiglu"; R is N, or for "swiglu" 2N: N gate
    rows, then N up rows, silu(gate) * up. ``bias`` fp32 or bf16 [R], ``residual`` bf16 [T, N].
    ``output``: where the result goes, ``residual`` itself included; a new tensor when None.
    K is a multiple of 8 (16 in 8 bits), N of 8; a weight may have padded rows.
    """
    e4m3 = isinstance(x, QuantizedRows)
    if e4m3 != isinstance(weight, QuantizedRows):
        raise TypeError("x and weight must both be QuantizedRows, or neither")
    x_scales = w_scales = None
    if e4m3:
        x, x_scales = x
        weight, w_scales = weight
    dtype = E4M3 if e4m3 else torch.bfloat16
    tokens, hidden = shape_of(x, "x", 2)
    rows, _ = shape_of(weight, "weight", 2)
    device = x.device
    require_tensor(x, "x", x.shape, dtype, device)
    if weight.dtype is not dtype:
        raise TypeError(f"weight must be {dtype}, got {weight.dtype}")
    if weight.shape[1] != hidden:
        raise ValueError(f"weight: expected rows of {hidden}, got shape {list(weight.shape)}")
    if weight.device != device:
        raise ValueError(f"weight must be on {device}")
    stride = _row_stride(weight, "weight")
    code = ACTIVATIONS.get(activation, -1)
    if code < 0:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}")
    if activation == "swiglu" and rows % 2:
        raise ValueError("swiglu needs an even number of weight rows")
    width = rows // 2 if activation == "swiglu" else rows
    unit = 16 if e4m3 else 8
    if hidden < unit or hidden % unit or hidden > MAX_WIDTH or stride % unit:
        raise ValueError(f"rows must be multiples of {unit} up to 2^20")
    if width < 8 or width % 8 or width > MAX_WIDTH:
        raise ValueError("the output's width must be a multiple of 8 up to 2^20")
    if tokens > MAX_TOKENS:
        raise ValueError("takes up to 2^21 rows")
    if e4m3:
        require_tensor(x_scales, "x.scales", (tokens,), torch.float32, device)
        require_tensor(w_scales, "weight.scales", (rows,), torch.float32, device)
    if bias is not None:
        if not isinstance(bias, torch.Tensor):
            raise TypeError("bias must be a tensor")
        if bias.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"bias must be float32 or bfloat16, got {bias.dtype}")
        require_tensor(bias, "bias", (rows,), bias.dtype, device)
    if residual is not None:
        require_tensor(residual, "residual", (tokens, width), torch.bfloat16, device)
    if output is not None:
        require_tensor(output, "output", (tokens, width), torch.bfloat16, device)
        same = residual is not None and output.data_ptr() == residual.data_ptr()
        if any(t is not None and _overlaps(output, t) for t in (x, weight, bias, x_scales, w_scales,
                                                                None if same else residual)):
            raise ValueError("output may be residual itself, but must not overlap another operand")
    require_gpu(x)
    refuse_autograd(x, weight, x_scales, w_scales, bias, residual, output)
    lib = get_extension().lib
    with on_device(device):
        if output is None:
            output = torch.empty((tokens, width), dtype=torch.bfloat16, device=device)
        need = _scratch_bytes(tokens, hidden, width, code, e4m3)
        scratch = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
        status = lib.moe_linear(LINEAR_ARGS(
            x.data_ptr(), weight.data_ptr(), _ptr(x_scales) or 0, _ptr(w_scales) or 0, _ptr(bias) or 0,
            _ptr(residual) or 0, output.data_ptr(), _ptr(scratch) or 0, need, tokens, hidden, width, stride,
            DTYPE_CODES[bias.dtype] if bias is not None else 0, code), current_stream_handle(device.index))
        if status:
            lib.check(status, "linear")
    return output


def _overlaps(a, b):
    """Whether the address ranges of two tensors meet (b's with the padding between its rows)."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    last = sum((n - 1) * s for n, s in zip(b.shape, b.stride())) + 1
    return a.data_ptr() < b.data_ptr() + last * b.element_size() and (
        b.data_ptr() < a.data_ptr() + a.numel() * a.element_size())
