"""Values of the operators around the experts where a rounding or a range decides them."""

import math

import pytest
import torch

from moe_dispatch import clip_gradients, quantize_rows, rms_norm
from tests._helpers import gpu

pytestmark = gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E4M3 = torch.float8_e4m3fn


def _quotients(y):
    """Scales and e4m3 values of fp32 rows by the definition's own two divisions, on the CPU."""
    y = y.float().cpu()
    scales = y.abs().amax(-1).clamp(min=2.0**-100) / torch.tensor(448.0)
    return scales, (y / scales.unsqueeze(-1)).clamp(-448.0, 448.0).to(E4M3)


def _same_rows(rows, y):
    scales, values = _quotients(y)
    assert torch.equal(rows.scales.cpu(), scales)
    assert torch.equal(rows.values.cpu().view(torch.uint8), values.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden", [(512, 2048), (700, 512), (37, 32768), (300, 1001)])
def test_eight_bit_rows_are_the_quotients(tokens, hidden, dtype):
    """e4m3(y / scale) bit for bit: quotients of few-bit values often lie half way between two of e4m3."""
    g = torch.Generator(device="cuda").manual_seed(hidden)
    x = (torch.randn(tokens, hidden, device="cuda", generator=g) * torch.exp2(
        torch.randint(-40, 40, (tokens, 1), device="cuda", generator=g)).float().clamp(2.0**-10, 2.0**12)).to(dtype)
    _same_rows(quantize_rows(x), x)
    if hidden <= 16384:
        weight = 1 + 0.2 * torch.randn(hidden, device="cuda", generator=g)
        x = x.float()
        _same_rows(rms_norm(x, weight, quantize=True).output, rms_norm(x, weight).output)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value,most", [(1e30, 1e-12), (1e36, 1e-6), (3e38, 1.0), (2e38, 0.5), (1e38, 1e-7), (1e30, 1e3), (1e20, 1e-30)])
def test_clip_factors_below_the_normal_range_of_fp32(value, most, dtype):
    """Large gradients and a small norm to reach, and norms past fp32 (written as infinite, the values scaled all the
    same): a factor within half a step of fp32's normal numbers, whatever its size."""
    grads = [torch.full((1000,), value, device="cuda", dtype=dtype), torch.full((333,), -value / 3, device="cuda", dtype=dtype)]
    kept = [t.double() for t in grads]
    exact = math.sqrt(math.fsum(float(t.square().sum()) for t in kept))
    outputs = [torch.empty_like(t) for t in grads]
    norm = clip_gradients(grads, most, outputs=outputs)
    assert float(norm) == (pytest.approx(exact, rel=1e-6) if exact < 3.4e38 else math.inf)
    for got, g in zip(outputs, kept):
        y = g * (most / (exact + 1e-6))
        half = torch.finfo(dtype).eps / 2
        # The factor and the product in fp32, half a step of a narrower type, and a step of the subnormals.
        steps = (half * 1.001 if dtype is not torch.float32 else 0.0) + 2.01 * 2.0**-24
        off = (got.double() - y).abs() - (y.abs() * steps + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)
        assert float(off.max()) <= 0, float(((got.double() - y) / y).abs().max())
    clip_gradients(grads, most)
    assert all(torch.equal(a, b) for a, b in zip(grads, outputs))
