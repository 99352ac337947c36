"""Values of the operators around the experts where a rounding or a range decides them."""

import pytest
import torch

from moe_dispatch import quantize_rows, rms_norm
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
