"""Root-mean-square norm, 8-bit rows and the norm's gradients, against 64-bit formulas.

Tolerances count roundings: U = 2^-24 for an fp32 operation, half = eps / 2 for a result rounded
once to its type. A row's sum of squares runs over chains of at most 64 terms a lane, 6 steps
in a wave and 16 waves: under 100 roundings of a positive sum, half of which the root keeps;
with the mean, root, division and three products y is within STEPS = 70 roundings.
"""

import math

import pytest
import torch

from moe_dispatch import QuantizedRows, autograd, quantize_rows, rms_norm, rms_norm_backward
from tests._helpers import gpu

pytestmark = gpu

U = 2.0**-24
STEPS = 70
E4M3_HALF, E4M3_LEAST = 2.0**-4, 2.0**-10  # half a step: relative, and of the subnormals
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(1, 1), (3, 7), (5, 64), (4, 511), (3, 513), (6, 1000), (2, 1023), (7, 2048), (3, 2056), (2, 4097), (3, 8192),
          (2, 12345), (2, 16384), (133, 24)]


def _half(dtype):
    return torch.finfo(dtype).eps / 2 if dtype is not torch.float32 else 0.0


def _within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        i = int(torch.nonzero(bad.reshape(-1))[0])
        t = tol.reshape(-1)[i] if isinstance(tol, torch.Tensor) and tol.numel() > 1 else tol
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; [{i}] {got.reshape(-1)[i].item()!r} against "
                             f"{want.reshape(-1)[i].item()!r}, tolerance {float(t):.3g}")


def _case(tokens, hidden, dtype, weight_dtype=None, residual=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    x = (normal(tokens, hidden) * torch.exp(normal(hidden))).to(dtype)
    weight = None if weight_dtype is None else (1 + 0.2 * normal(hidden)).to(weight_dtype)
    return x, weight, normal(tokens, hidden).to(dtype) if residual else None


def _formula(x, weight, residual, eps):
    total = x.double() if residual is None else x.double() + residual.double()
    rstd = 1 / torch.sqrt(total.square().mean(-1, keepdim=True) + eps)
    return total, rstd, total * rstd * (1 if weight is None else weight.double())


def _check_quantized(rows, y, what, steps=STEPS):
    """Scales, and values by half a step of theirs; the values' scale is the one they were made with."""
    assert rows.values.dtype is torch.float8_e4m3fn and rows.scales.dtype is torch.float32
    scales = y.abs().amax(-1).clamp(min=2.0**-100) / 448
    _within(rows.scales, scales, scales * (steps + 2) * U, what + " scales")
    q = y / rows.scales.double().unsqueeze(-1)
    tol = torch.clamp(q.abs() * E4M3_HALF, min=E4M3_LEAST) * (1 + 1e-5) + q.abs() * (steps + 4) * U
    _within(rows.values.double(), q, tol, what + " values")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden", SHAPES)
def test_norm_against_the_formula(tokens, hidden, dtype):
    for i, (weight_dtype, residual) in enumerate(((dtype, True), (torch.float32, False), (None, True))):
        x, weight, add = _case(tokens, hidden, dtype, weight_dtype, residual, seed=i)
        total, rstd, y = _formula(x, weight, add, 1e-5)
        normed = rms_norm(x, weight, residual=add, eps=1e-5, return_rstd=True)
        assert normed.output.dtype is dtype
        # A sum of opposite x and residual keeps the rounding of the sum itself only.
        _within(normed.output, y, y.abs() * (_half(dtype) * 1.001 + STEPS * U) + 6e-8 * (dtype is torch.float16), "y")
        _within(normed.rstd, rstd.squeeze(-1), rstd.squeeze(-1) * STEPS * U, "rstd")
        if residual:
            _within(normed.total, total, total.abs() * (_half(dtype) * 1.001 + U) + 3e-8 * (dtype is torch.float16), "total")
        else:
            assert normed.total is None
        eight = rms_norm(x, weight, residual=add, eps=1e-5, quantize=True)
        assert eight.rstd is None
        _check_quantized(eight.output, y, f"quantized {weight_dtype} {residual}")
        if residual:
            assert torch.equal(eight.total, normed.total)
        _check_quantized(quantize_rows(x), x.double(), "rows", steps=4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hidden", [16385, 20000, 32767, 32768])
def test_wide_rows_in_8_bits(hidden, dtype):
    x = _case(5, hidden, dtype, None, False, seed=hidden)[0]
    _check_quantized(quantize_rows(x), x.double(), "wide", steps=4)


def test_rows_of_zeros_tiny_values_and_no_rows():
    x = torch.zeros(5, 96, device="cuda")
    x[1] = 1e-35  # below the least scale
    x[2, 3] = 2.0
    x[3] = -3e38
    x[4] = 1e-44
    rows = quantize_rows(x)
    least = 2.0**-100 / 448
    assert torch.isfinite(rows.scales).all() and float(rows.scales[0]) == pytest.approx(least, rel=1e-6)
    assert float(rows.scales[1]) == pytest.approx(least, rel=1e-6)
    back = rows.dequantize()
    assert torch.equal(back[0], x[0]) and float(back[2, 3]) == pytest.approx(2.0, rel=1e-6)
    assert torch.equal(back[2, :3], x[2, :3]) and float(back[3, 0]) == pytest.approx(-3e38, rel=1e-6)
    normed = rms_norm(x[:1], None, eps=1e-6)
    assert torch.equal(normed.output, x[:1])
    assert torch.isnan(rms_norm(x[:1], None, eps=0.0).output).all()  # 0 / 0
    for quantize in (False, True):
        empty = rms_norm(x[:0], None, residual=x[:0], quantize=quantize, return_rstd=True)
        assert empty.total.shape == (0, 96) and empty.rstd.shape == (0,)
    assert rms_norm_backward(x[:0], x[:0], torch.ones(96, device="cuda"), empty.rstd)[1].tolist() == [0] * 96


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan_stay_in_their_rows(dtype):
    x, weight, add = _case(6, 200, dtype, dtype, True)
    clean = rms_norm(x, weight, residual=add)
    clean8 = rms_norm(x, weight, residual=add, quantize=True).output
    bad = x.clone()
    bad[1, 7] = float("nan")
    bad[4, 199] = float("inf")
    got = rms_norm(bad, weight, residual=add)
    keep = [0, 2, 3, 5]
    assert torch.equal(got.output[keep], clean.output[keep]) and torch.isnan(got.output[1]).all()
    assert torch.isnan(got.output[4, 199]) and not torch.isfinite(got.total[4, 199])
    got8 = rms_norm(bad, weight, residual=add, quantize=True).output
    assert torch.equal(got8.dequantize()[keep], clean8.dequantize()[keep])
    assert torch.isnan(got8.dequantize()[1]).all()
    raw = quantize_rows(bad)
    assert torch.isnan(raw.dequantize()[1, 7]) and torch.isfinite(raw.dequantize()[1, :7]).all()
    assert torch.isnan(raw.dequantize()[4]).all() and not torch.isfinite(raw.scales[4])


def test_rows_at_any_element_address():
    """Views that start on one element, in each type: rows and weight off the vectors' grid."""
    for dtype in TYPES:
        for hidden in (64, 1000, 1023):
            x, weight, add = _case(4, hidden, dtype, dtype, True)
            want = rms_norm(x, weight, residual=add)
            off = [torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape) for t in (x, weight, add)]
            assert off[0].data_ptr() % 16 != 0
            got = rms_norm(off[0], off[1], residual=off[2])
            assert torch.equal(got.output, want.output) and torch.equal(got.total, want.total)
            g = x + add
            rstd = rms_norm(x, weight, return_rstd=True).rstd
            a, b = rms_norm_backward(g, x, weight, rstd), rms_norm_backward(off[2] + off[0], off[0], off[1], rstd)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden", SHAPES + [(1500, 40), (700, 2048)])
def test_gradients_against_the_formula(tokens, hidden, dtype):
    x, weight, g = _case(tokens, hidden, dtype, dtype, True, seed=3)
    base = _case(tokens, hidden, dtype, None, True, seed=4)[2]
    rstd = rms_norm(x, weight, return_rstd=True).rstd
    u, w, go = x.double() * rstd.double().unsqueeze(-1), weight.double(), g.double()
    mean = (go * w * u).mean(-1, keepdim=True)
    dx = rstd.double().unsqueeze(-1) * (go * w - u * mean)
    # u, products and the mean of a row: its terms' sizes, at most 100 + 10 roundings.
    size = rstd.double().unsqueeze(-1) * ((go * w).abs() + u.abs() * (go * w * u).abs().mean(-1, keepdim=True))
    dw = (go * u).sum(0)
    dw_size = (go * u).abs().sum(0)
    for use_base in (True, False):
        got_x, got_w = rms_norm_backward(g, x, weight, rstd, grad_x=base if use_base else None)
        want = dx + base.double() if use_base else dx
        least = 6e-8 if dtype is torch.float16 else 0.0
        _within(got_x, want, want.abs() * (_half(dtype) * 1.001 + 2 * U) + size * 110 * U + least, "dx")
        # Rows of a workgroup in one chain (tokens / 512), 64 partial sums a slice, 8 slices.
        assert got_w.dtype is torch.float32
        _within(got_w, dw, dw_size * (tokens / 512 + 64 + 12) * U, "dw")
    only_x, none = rms_norm_backward(g, x, weight, rstd, gradients=(True, False))
    none_x, only_w = rms_norm_backward(g, x, weight, rstd, gradients=(False, True))
    assert none is None and none_x is None
    assert torch.equal(only_x, got_x) and torch.equal(only_w, got_w)


def test_gradients_against_differences():
    """The directional derivative by central differences of the 64-bit definition: its error is
    h^2 / 6 of the third derivative (1e-10 of the value here) and 1e-16 / h."""
    x, weight, g = _case(9, 300, torch.float32, torch.float32, True, seed=5)
    rstd = rms_norm(x, weight, return_rstd=True).rstd
    dx, dw = rms_norm_backward(g, x, weight, rstd)
    gen = torch.Generator(device="cuda").manual_seed(6)
    vx = torch.randn(x.shape, device="cuda", generator=gen).double()
    vw = torch.randn(weight.shape, device="cuda", generator=gen).double()
    h = 1e-5

    def f(s):
        total = x.double() + s * vx
        y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + 1e-6) * (weight.double() + s * vw)
        return float((y * g.double()).sum())

    want = (f(h) - f(-h)) / (2 * h)
    got = float((dx.double() * vx).sum() + (dw.double() * vw).sum())
    size = float((dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum())
    assert abs(got - want) <= size * (200 * U + 1e-8)


def test_autograd_norm():
    for dtype in (torch.float32, torch.bfloat16):
        x, weight, add = _case(12, 520, dtype, dtype, True, seed=7)
        leaves = [t.clone().requires_grad_() for t in (x, weight, add)]
        out, total = autograd.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        g1, g2 = torch.randn_like(out), torch.randn_like(total)
        torch.autograd.backward([out, total], [g1, g2])
        rstd = rms_norm(x, weight, residual=add, return_rstd=True).rstd
        want_x, want_w = rms_norm_backward(g1, total.detach(), weight, rstd, grad_x=g2)
        assert torch.equal(leaves[0].grad, want_x) and torch.equal(leaves[2].grad, want_x)
        assert torch.equal(leaves[1].grad, want_w.to(dtype))
        # One output alone, and no residual.
        leaves = [t.clone().requires_grad_() for t in (x, weight)]
        out, total = autograd.rms_norm(*leaves)
        assert total is None
        out.backward(g1)
        rstd = rms_norm(x, weight, return_rstd=True).rstd
        assert torch.equal(leaves[0].grad, rms_norm_backward(g1, x, weight, rstd)[0])
        leaves = [t.clone().requires_grad_() for t in (x, weight, add)]
        autograd.rms_norm(leaves[0], leaves[1], residual=leaves[2])[1].backward(g2)
        assert torch.equal(leaves[0].grad, g2) and torch.equal(leaves[2].grad, g2) and leaves[1].grad is None


def test_many_rows_past_32_bit_offsets():
    """Elements past 2^31: the last rows equal those of a small call."""
    tokens, hidden = 2**17 + 3, 16384
    x = torch.empty(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    x[:] = torch.randn(1, hidden, device="cuda").bfloat16()
    x[-3:] = torch.randn(3, hidden, device="cuda").bfloat16()
    want = rms_norm(x[-3:].clone(), quantize=True).output
    got = rms_norm(x, quantize=True).output
    assert torch.equal(got.values[-3:].view(torch.uint8), want.values.view(torch.uint8))
    assert torch.equal(got.scales[-3:], want.scales)
    del got
    g = x
    rstd = rms_norm(x[-3:].clone(), return_rstd=True).rstd
    every = rstd.new_ones(tokens)
    every[-3:] = rstd
    dx, _ = rms_norm_backward(g, x, None, every)
    assert torch.equal(dx[-3:], rms_norm_backward(g[-3:].clone(), x[-3:].clone(), None, rstd)[0])


def test_norm_in_a_graph_and_on_another_stream():
    x, weight, add = _case(200, 1024, torch.bfloat16, torch.bfloat16, True)
    grad = _case(200, 1024, torch.bfloat16, None, True, seed=9)[2]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        normed = rms_norm(x, weight, residual=add, return_rstd=True)
        return (*rms_norm(normed.total, weight, quantize=True).output, normed.output,
                *rms_norm_backward(grad, normed.total, weight, normed.rstd, grad_x=grad))

    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        fresh = _case(200, 1024, torch.bfloat16, torch.bfloat16, True, seed=20 + seed)
        for t, f in zip((x, weight, add), fresh):
            t.copy_(f)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_autograd_is_refused_in_plain_calls():
    x = torch.ones(4, 64, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="autograd"):
        rms_norm(x)
    with torch.no_grad():
        assert isinstance(rms_norm(x, quantize=True).output, QuantizedRows)
    assert math.isclose(float(rms_norm(x.detach()).output[0, 0]), 1.0, rel_tol=1e-5)
