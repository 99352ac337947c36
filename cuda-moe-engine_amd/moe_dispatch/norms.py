"""Root-mean-square norm of rows with the residual's addition, 8-bit rows, and the norm's gradients.

The norm in front of a layer's router and experts, on the kernels of ``libmoe_hip.so``:

    h = x + residual,   y = h / sqrt(mean(h^2) + eps) * weight

``rms_norm`` gives y in x's type, or as ``QuantizedRows``: e4m3 values with one scale a row,
which ``dense.linear`` takes as they are. ``quantize_rows`` gives any rows that form: the
activations between two 8-bit products, and weights when they are loaded.
``rms_norm_backward`` gives the gradients of rows and weight. No counterpart in the reference.

Checks, streams and errors are those of ``moe_dispatch.training``.
"""

from functools import lru_cache
from typing import NamedTuple

import torch

from ._extension import DTYPE_CODES, current_stream_handle, get_extension
from ._lib import RMS_NORM_ARGS
from .training import _ptr, on_device, refuse_autograd, require_gpu, require_tensor, shape_of

MAX_HIDDEN = 16384
MAX_QUANTIZED = 32768  # of quantize_rows
MAX_TOKENS = 2**21
E4M3 = torch.float8_e4m3fn


class QuantizedRows(NamedTuple):
    """Rows in 8 bits: ``values`` float8_e4m3fn [T, H] and ``scales`` fp32 [T]; row t stands for
    ``values[t] * scales[t]``."""

    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype=torch.float32):
        return (self.values.float() * self.scales.unsqueeze(-1)).to(dtype)


class Normed(NamedTuple):
    """``output`` is the normed rows (a tensor or ``QuantizedRows``), ``total`` x + residual (None
    without a residual), ``rstd`` fp32 [T] (None unless asked for)."""

    output: object
    total: torch.Tensor | None
    rstd: torch.Tensor | None


def _check_rows(x, most=MAX_HIDDEN):
    tokens, hidden = shape_of(x, "x", 2)
    if x.dtype not in DTYPE_CODES:
        raise TypeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    if not 1 <= hidden <= most:
        raise ValueError(f"rows must have 1..{most} elements")
    if tokens > MAX_TOKENS:
        raise ValueError("takes up to 2^21 rows")
    return tokens, hidden


def _check_weight(weight, x, hidden):
    if weight is None:
        return DTYPE_CODES[x.dtype]
    if not isinstance(weight, torch.Tensor):
        raise TypeError("weight must be a tensor")
    if weight.dtype is not x.dtype and weight.dtype is not torch.float32:
        raise TypeError(f"weight must be {x.dtype} or float32, got {weight.dtype}")
    require_tensor(weight, "weight", (hidden,), weight.dtype, x.device)
    return DTYPE_CODES[weight.dtype]


def rms_norm(x, weight=None, *, residual=None, eps=1e-6, quantize=False, return_rstd=False):
    """Norm of the rows of x + residual: ``Normed``.

    x [T, H] is fp32, fp16 or bf16, weight [H] of x's type or fp32 (None: 1), residual [T, H]
    of x's type (None: 0). Statistics and products are fp32, from the unrounded sum; ``output``
    is rounded once to x's type, or with ``quantize`` to e4m3 with
    ``scales[t] = max(max_j |y_tj|, 2^-100) / 448``. A NaN makes its whole row NaN (with
    ``quantize`` the scale is then the least one). An infinity makes rstd 0: its own y is NaN, the
    row's others 0, and the scale the least one as well. H is at most 16384, and values are below 1e17 (their
    squares' sum is fp32); with an eps below 1e-30 a row's largest value is above 1e-16, or all of it 0
    (of ``eps=0`` y is NaN there).
    """
    tokens, hidden = _check_rows(x)
    weight_code = _check_weight(weight, x, hidden)
    if residual is not None:
        require_tensor(residual, "residual", x.shape, x.dtype, x.device)
    if not 0 <= eps < 1e30:
        raise ValueError("eps must be finite and not negative")
    require_gpu(x)
    refuse_autograd(x, weight, residual)
    device = x.device
    lib = get_extension().lib
    with on_device(device):
        total = torch.empty_like(x) if residual is not None else None
        rstd = x.new_empty(tokens, dtype=torch.float32) if return_rstd else None
        if quantize:
            values = torch.empty_like(x, dtype=E4M3)
            scales = x.new_empty(tokens, dtype=torch.float32)
            output = QuantizedRows(values, scales)
        else:
            output = values = torch.empty_like(x)
            scales = None
        status = lib.moe_rms_norm(RMS_NORM_ARGS(
            x.data_ptr(), _ptr(residual) or 0, _ptr(weight) or 0, _ptr(total) or 0, values.data_ptr(),
            _ptr(scales) or 0, _ptr(rstd) or 0, tokens, hidden, DTYPE_CODES[x.dtype], weight_code, eps),
            current_stream_handle(device.index))
        if status:
            lib.check(status, "rms_norm")
    return Normed(output, total, rstd)


def quantize_rows(x):
    """Rows x [T, H] (fp32, fp16 or bf16, H up to 32768) as ``QuantizedRows``, with ``rms_norm``'s scales.

    A NaN stays one and has no part in the scale; a row that holds an infinity has an infinite scale,
    and all of it stands for NaN.
    """
    tokens, hidden = _check_rows(x, MAX_QUANTIZED)
    require_gpu(x)
    refuse_autograd(x)
    device = x.device
    lib = get_extension().lib
    with on_device(device):
        values = torch.empty_like(x, dtype=E4M3)
        scales = x.new_empty(tokens, dtype=torch.float32)
        lib.check(lib.moe_quantize_rows(x.data_ptr(), DTYPE_CODES[x.dtype], values.data_ptr(), scales.data_ptr(), tokens,
                                        hidden, current_stream_handle(device.index)), "quantize_rows")
    return QuantizedRows(values, scales)


@lru_cache(maxsize=1024)
def _scratch_bytes(tokens, hidden, dtype_code):
    return get_extension().lib.moe_rms_norm_backward_scratch_bytes(tokens, hidden, dtype_code)


def rms_norm_backward(grad_output, x, weight, rstd, *, grad_x=None, gradients=(True, True)):
    """Gradients of ``rms_norm``: ``(grad_x, grad_weight)``.

    x holds the normed rows (``Normed.total`` of a norm with a residual, whose gradient is
    grad_x as well), ``rstd`` is the forward's. ``grad_x`` [T, H] of x's type is the rows'
    gradient along their other paths: the result is the sum, rounded once. grad_weight is
    fp32 [H] (None without a weight). ``gradients``: which of the two are wanted; the other
    is None and is not computed.
    """
    tokens, hidden = _check_rows(x)
    weight_code = _check_weight(weight, x, hidden)
    require_tensor(grad_output, "grad_output", x.shape, x.dtype, x.device)
    require_tensor(rstd, "rstd", (tokens,), torch.float32, x.device)
    if grad_x is not None:
        require_tensor(grad_x, "grad_x", x.shape, x.dtype, x.device)
    require_gpu(x)
    refuse_autograd(grad_output, x, weight, grad_x)
    device = x.device
    lib = get_extension().lib
    want_x, want_weight = gradients
    with on_device(device):
        out_x = torch.empty_like(x) if want_x else None
        grad_weight = x.new_empty(hidden, dtype=torch.float32) if want_weight and weight is not None else None
        if tokens == 0:
            if grad_weight is not None:
                grad_weight.zero_()
            return out_x, grad_weight
        need = _scratch_bytes(tokens, hidden, DTYPE_CODES[x.dtype]) if grad_weight is not None else 0
        scratch = x.new_empty(need // 4, dtype=torch.float32) if need else None
        lib.check(lib.moe_rms_norm_backward(
            grad_output.data_ptr(), x.data_ptr(), DTYPE_CODES[x.dtype], _ptr(weight), weight_code, rstd.data_ptr(),
            _ptr(grad_x), _ptr(out_x), _ptr(grad_weight), _ptr(scratch), need, tokens, hidden,
            current_stream_handle(device.index)), "rms_norm_backward")
    return out_x, grad_weight
