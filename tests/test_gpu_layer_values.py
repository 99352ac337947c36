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


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_of_rows_that_are_no_numbers(dtype):
    """As documented: what a NaN and an infinity leave of their row and its scale, in the norm and alone."""
    g = torch.Generator(device="cuda").manual_seed(1)
    least = float(torch.tensor(2.0**-100) / torch.tensor(448.0))
    for hidden in (5, 200, 4096):
        x = torch.randn(4, hidden, device="cuda", generator=g).to(dtype)
        x[1, 2], x[2, 4] = float("nan"), float("-inf")
        rows = rms_norm(x, quantize=True).output
        assert rows.scales[1:3].tolist() == [least, least] and bool(torch.isfinite(rows.scales).all())
        back = rows.dequantize()
        assert torch.isnan(back[1]).all() and torch.isnan(back[2, 4])
        rest = torch.arange(hidden, device="cuda") != 4
        assert not back[2][rest].any() and bool(torch.isfinite(back[0]).all())
        rows = quantize_rows(x)
        back = rows.dequantize()
        assert math.isinf(float(rows.scales[2])) and torch.isnan(back[2]).all()
        rest = torch.arange(hidden, device="cuda") != 2
        assert torch.isnan(back[1, 2]) and bool(torch.isfinite(back[1][rest]).all())
        assert float(rows.scales[1]) == float((x[1].float()[rest].abs().amax().cpu() / torch.tensor(448.0)))


@pytest.mark.parametrize("hidden", [1, 65, 2048, 16384])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_of_tiny_rows_without_eps(hidden, dtype):
    """eps 0 at the end of the documented range: squares below it vanish beside the row's largest."""
    x = torch.zeros(3, hidden, device="cuda")
    x[0, 0] = 1.01e-16
    x[1] = 2e-16 * torch.linspace(-1, 1, hidden, device="cuda") if hidden > 1 else 2e-16
    x[2, -1], x[2, 0] = 1e-16 if hidden > 1 else 0.0, 3e-16
    x = x.to(dtype)
    y = rms_norm(x, eps=0.0).output.double()
    want = x.double() / x.double().square().mean(-1, keepdim=True).sqrt()
    # 70 roundings of fp32 as in the norm's own tests, squares lost below 2^-126 (16384 of them against 1e-32), half a step.
    half = torch.finfo(dtype).eps / 2 if dtype is not torch.float32 else 0.0
    lost = 16384 * 2.0**-126 / 1e-32
    assert bool(((y - want).abs() <= want.abs() * (half * 1.001 + 70 * 2.0**-24 + lost)).all())
