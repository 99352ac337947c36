"""Dense products with their epilogues, against 64-bit formulas.

A product's sum of K terms is within 2 K roundings of 2^-24 of the sum of the terms' sizes (twice,
for hardware that truncates; its chains are far shorter), scales and bias add 4 of theirs.
An activation passes an error on by at most its slope (1.13 is the largest of silu and gelu) and
adds its own: exp, erf or tanh and a few operations, 30 roundings of its argument. The result
is rounded once to bf16.

The 8-bit matrix instruction adds the products of eight neighbouring k at the largest one's
scale before it adds to fp32: beside a product of 2^16 one of 2^3 is kept and one of 2^2 is lost. So
each of the other seven loses less than 2^-13 of the largest, a group less than 7 * 2^-13 of its
terms' sizes, and a sum less than 7 * 2^-13 of them all. That bound is far from what happens
(losses average out), so the 2-norm over a result of at least 2000 values is held too: bf16's rounding is
at most 2^-8 of a value and uniform, 2^-8 / sqrt(3) = 2.3e-3, and nothing else may show beside it.
"""

import pytest
import torch

from moe_dispatch import QuantizedRows, linear, quantize_rows
from tests._helpers import gpu

pytestmark = gpu

U = 2.0**-24
HALF = 2.0**-8
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh", "swiglu"]


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=g) * scale


def _case(tokens, hidden, width, eight, activation=None, bias=None, residual=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = 2 * width if activation == "swiglu" else width
    x, w = _normal(g, tokens, hidden), _normal(g, rows, hidden, scale=hidden**-0.5)
    if eight:
        x, w = quantize_rows(x), quantize_rows(w)
    else:
        x, w = x.bfloat16(), w.bfloat16()
    b = None if bias is None else _normal(g, rows).to(bias)
    return x, w, b, _normal(g, tokens, width).bfloat16() if residual else None


def _wide(t):
    return t.values.double() * t.scales.double().unsqueeze(-1) if isinstance(t, QuantizedRows) else t.double()


def _formula(x, w, b, residual, activation):
    """The result, and how far one may be before its rounding to bf16."""
    eight = isinstance(x, QuantizedRows)
    x, w = _wide(x), _wide(w)
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    off = size * ((2 * x.shape[1] + 4) * U + (7 * 2.0**-13 if eight else 0.0))
    if b is not None:
        z = z + b.double()
        off = off + (b.double().abs() + z.abs()) * 2 * U
    f = torch.nn.functional
    if activation == "swiglu":
        gate, up = z.chunk(2, -1)
        dg, du = off.chunk(2, -1)
        y = f.silu(gate) * up
        off = 1.13 * dg * (up.abs() + du) + gate.abs() * du + gate.abs() * up.abs() * 30 * U
    elif activation is None:
        y = z
    elif activation == "relu":
        y = torch.relu(z)
    else:
        y = f.silu(z) if activation == "silu" else f.gelu(z, approximate="tanh" if activation == "gelu_tanh" else "none")
        off = 1.13 * off + z.abs() * 30 * U
    if residual is not None:
        y = y + residual.double()
        off = off + (y.abs() + residual.double().abs()) * U
    return y, off


def _check(got, x, w, b, residual, activation, what):
    y, off = _formula(x, w, b, residual, activation)
    assert got.dtype is torch.bfloat16 and got.shape == y.shape
    bad = ~((got.double() - y).abs() <= y.abs() * HALF * 1.001 + off * 1.01 + 1e-38)
    if bool(bad.any()):
        i = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; [{i}] {got.reshape(-1)[i].item()!r} against "
                             f"{y.reshape(-1)[i].item()!r}")
    if y.numel() >= 2000:
        assert float((got.double() - y).norm()) <= 2.3e-3 * float(y.norm()), what


# Tokens around every tile's edge, widths and depths that end inside tiles and stages.
SHAPES = [(1, 16, 8), (1, 64, 24), (1, 4096, 64), (2, 1000, 264), (3, 8192, 40), (7, 144, 136), (15, 2048, 128), (16, 512, 72),
          (17, 336, 320), (31, 1408, 256), (33, 64, 520), (48, 2048, 1408), (63, 208, 88), (64, 4096, 96), (65, 128, 64),
          (96, 720, 200), (127, 256, 256), (128, 96, 776), (129, 1040, 264), (200, 64, 1032), (255, 512, 248), (256, 128, 512),
          (257, 400, 640), (333, 1000, 344), (515, 2048, 136), (777, 272, 512), (1030, 192, 328)]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("tokens,hidden,width", SHAPES)
def test_products_against_the_formula(tokens, hidden, width, eight):
    hidden = hidden // 16 * 16 if eight else hidden
    for i, activation in enumerate(ACTS):
        bias = (None, torch.float32, torch.bfloat16)[(tokens + i) % 3]
        residual = bool((tokens + i) // 2 % 2)
        x, w, b, r = _case(tokens, hidden, width, eight, activation, bias, residual, seed=i)
        got = linear(x, w, b, activation=activation, residual=r)
        _check(got, x, w, b, r, activation, (activation, bias, residual))
        if i == 5:  # the same call again: no sum depends on timing
            assert torch.equal(got, linear(x, w, b, activation=activation, residual=r))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("tokens,hidden,width,activation", [(1, 4096, 4104, "swiglu"), (5, 14336, 2048, None),
                                                            (130, 4096, 2056, None), (1500, 1024, 2048, "swiglu"),
                                                            (2049, 4096, 1544, "silu"), (4100, 512, 4096, None)])
def test_larger_products(tokens, hidden, width, activation, eight):
    x, w, b, r = _case(tokens, hidden, width, eight, activation, torch.float32, True, seed=1)
    _check(linear(x, w, b, activation=activation, residual=r), x, w, b, r, activation, "larger")


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hidden", [112, 208, 336, 544, 1040])
@pytest.mark.parametrize("activation,extras", [(None, False), (None, True), ("gelu", True), ("swiglu", False), ("swiglu", True)])
def test_rounds_of_chained_tiles(hidden, eight, activation, extras):
    """More of the largest tiles than CUs, of one stage to seventeen: stores of one tile beside loads of the next."""
    x, w, b, r = _case(4200, hidden, 5000, eight, activation, torch.float32 if extras else None, extras, seed=hidden)
    first = linear(x, w, b, activation=activation, residual=r)
    _check(first, x, w, b, r, activation, (hidden, activation, extras))
    for _ in range(3):
        assert torch.equal(linear(x, w, b, activation=activation, residual=r), first)


def test_no_rows():
    x, w, _, _ = _case(0, 64, 16, False)
    assert linear(x, w).shape == (0, 16)
    x, w, _, _ = _case(0, 64, 16, True, "swiglu")
    assert linear(x, w, activation="swiglu").shape == (0, 16)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("tokens", [1, 20, 300])
def test_padded_weight_rows_and_what_lies_in_them(tokens, eight):
    """Rows with padding that holds NaN, among them a last stage that ends inside the padding."""
    for hidden in (1040, 2048):
        x, w, _, _ = _case(tokens, hidden, 264, eight)
        values = w.values if eight else w
        padded = torch.full((264, hidden + 64), float("nan"), device="cuda").to(values.dtype)
        padded[:, :hidden] = values
        view = padded[:, :hidden]
        other = w._replace(values=view) if eight else view
        assert torch.equal(linear(x, w), linear(x, other))


@pytest.mark.parametrize("tokens", [1, 40, 260])
def test_output_into_the_residual_and_rows_behind(tokens):
    """In place, and nothing outside the output changes."""
    x, w, b, r = _case(tokens, 512, 520, False, "gelu", torch.float32, True)
    want = linear(x, w, b, activation="gelu", residual=r)
    around = torch.full((tokens + 4, 520), 7.0, device="cuda", dtype=torch.bfloat16)
    around[2:2 + tokens] = r
    inside = around[2:2 + tokens]
    got = linear(x, w, b, activation="gelu", residual=inside, output=inside)
    assert got.data_ptr() == inside.data_ptr() and torch.equal(inside, want)
    assert bool((around[:2] == 7).all()) and bool((around[2 + tokens:] == 7).all())


@pytest.mark.parametrize("eight", [False, True])
def test_infinities_and_nan_stay_in_their_rows(eight):
    x, w, _, _ = _case(70, 1024, 136, eight)
    want = linear(x, w)
    values = (x.values if eight else x).clone()
    values[5, 100] = float("nan")
    values[69, 1023] = float("nan")
    got = linear(x._replace(values=values) if eight else values, w)
    keep = [t for t in range(70) if t not in (5, 69)]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[5]).all() and torch.isnan(got[69]).all()
    if eight:
        scales = x.scales.clone()
        scales[3] = float("inf")
        got = linear(x._replace(scales=scales), w)
        assert not torch.isfinite(got[3]).any() and torch.equal(got[4:], want[4:])
    act = linear(torch.full((1, 8), -3e38, device="cuda", dtype=torch.bfloat16),
                 torch.full((8, 8), 3e38, device="cuda", dtype=torch.bfloat16), activation="relu")
    assert torch.equal(act, torch.zeros_like(act))


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "swiglu"])
def test_activations_over_their_range(activation):
    """Products of one term: every argument from the flat ends to the middle."""
    z = torch.cat([torch.linspace(-120, 120, 4001), torch.logspace(-30, 4.5, 1000), -torch.logspace(-30, 4.5, 1000)])
    x = torch.zeros(z.numel(), 8, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = z.to(device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(16 if activation == "swiglu" else 8, 8, device="cuda", dtype=torch.bfloat16)
    w[:, 0] = 1
    _check(linear(x, w, activation=activation), x, w, None, None, activation, activation)


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("tokens", [2, 40])
def test_activations_of_infinities(tokens, activation):
    inf = float("inf")
    x = torch.zeros(tokens, 8, device="cuda", dtype=torch.bfloat16)
    values = torch.tensor([inf, -inf, float("nan"), 3e38, -3e38, 2e19, -2e19, 0.0], device="cuda")
    bias = values if activation != "swiglu" else torch.cat([values, torch.full((8,), 0.5, device="cuda")])
    w = torch.zeros(bias.numel(), 8, device="cuda", dtype=torch.bfloat16)
    got = linear(x, w, bias, activation=activation)
    f = torch.nn.functional
    # Halves of fp32 values: what the activations do to them needs no rounding but bf16's.
    want = {None: lambda z: z, "relu": torch.relu, "silu": f.silu, "gelu": f.gelu,
            "gelu_tanh": lambda z: f.gelu(z, approximate="tanh"), "swiglu": lambda z: f.silu(z) * 0.5}[activation]
    want = want(values.double().cpu()).bfloat16().expand(tokens, 8)
    assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(got.cpu().isnan(), want.isnan())


@pytest.mark.parametrize("tokens", [2, 40])
@pytest.mark.parametrize("part,factor", [(256, 1e13), (65536, 1e16)])
def test_scales_whose_product_nears_or_leaves_fp32(tokens, part, factor):
    """Results past bf16's range are infinite: from (2 - 2^-8) 2^127 on the nearest value is."""
    x, w, _, _ = _case(tokens, 64, 264, True, seed=9)
    x = x._replace(values=(x.values.float() / part).to(x.values.dtype), scales=x.scales * 1e30)
    w = w._replace(values=(w.values.float() / part).to(w.values.dtype), scales=w.scales * factor)
    got, (want, off) = linear(x, w), _formula(x, w, None, None, None)
    past = want.abs() >= (2 - HALF) * 2.0**127
    assert torch.equal(got[past].double(), want[past].sign() * float("inf"))
    bad = ~past & ~((got.double() - want).abs() <= want.abs() * HALF * 1.001 + off * 1.01)
    assert not bool(bad.any())


def test_operands_that_record_gradients_are_refused():
    x, w, b, r = _case(3, 64, 24, False, bias=torch.float32, residual=True)
    for t in (x, w, b, r):
        with pytest.raises(ValueError, match="autograd"):
            t.requires_grad_()
            try:
                linear(x, w, b, residual=r)
            finally:
                t.requires_grad_(False)
    x, w, _, _ = _case(3, 64, 24, True)
    for t in (x.scales, w.scales):
        t.requires_grad_()
        with pytest.raises(ValueError, match="autograd"):
            linear(x, w)
        with torch.no_grad():
            linear(x, w)
        t.requires_grad_(False)


def test_graph_replays_and_streams_share_nothing():
    """Two captured graphs and eager work in between: each call's scratch is its own."""
    x, w, b, r = _case(3, 4096, 1408, True, "swiglu", torch.float32, False)
    x2, w2, b2, r2 = _case(24, 1408, 2048, False, None, None, True)

    def step():
        return linear(x, w, b, activation="swiglu"), linear(x2, w2, residual=r2)

    step()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    side = torch.cuda.Stream()
    for seed in range(3):
        fresh, _, _, _ = _case(3, 4096, 1408, True, "swiglu", seed=50 + seed)
        x.values.copy_(fresh.values)
        x.scales.copy_(fresh.scales)
        x2.mul_(1.5)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            eager = step()
        torch.cuda.synchronize()
        for got in (*outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("tokens", [3, 20, 260, 700])
def test_widest_output_and_longest_rows(tokens, eight):
    """2^20 columns (a tile's rows span half a GiB) and 2^20 deep."""
    x, w, b, r = _case(tokens, 16, 2**20, eight, bias=torch.float32, residual=True)
    around = torch.full((tokens + 1, 2**20), 7.0, device="cuda", dtype=torch.bfloat16)
    got = linear(x, w, b, residual=r, output=around[:tokens])
    for part in (slice(0, 512), slice(2**19 - 256, 2**19 + 256), slice(2**20 - 512, 2**20)):
        few = QuantizedRows(w.values[part], w.scales[part]) if eight else w[part]
        _check(got[:, part], x, few, b[part], r[:, part], None, (tokens, part))
    assert bool((around[tokens] == 7).all())
    del around, got, r
    x, w, _, _ = _case(tokens, 2**20, 8, False)
    if eight:  # (longer than quantize_rows takes)
        x, w = (QuantizedRows((t.float() * s).to(torch.float8_e4m3fn), torch.full((len(t),), 1 / s, device="cuda"))
                for t, s in ((x, 64.0), (w, 2.0**16)))
    _check(linear(x, w), x, w, None, None, None, (tokens, "deep"))


def test_weights_past_two_gib():
    """Weight rows past 2^31 bytes, for one token and for a tile of them."""
    hidden, width = 16384, 2**17 - 8
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.zeros(width, hidden, device="cuda", dtype=torch.bfloat16)
    w[-64:] = _normal(g, 64, hidden).bfloat16()
    for tokens in (1, 80):
        x = _normal(g, tokens, hidden).bfloat16()
        got = linear(x, w)
        # A product of another width may split its sums elsewhere: the formula, not the bits.
        _check(got[:, -64:], x, w[-64:], None, None, None, tokens)
        assert not bool(got[:, :-64].any())
