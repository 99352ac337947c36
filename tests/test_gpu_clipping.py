"""Global gradient norm and clipping, and a layer's operators together.

The norm is 64-bit sums of exact squares: within one fp32 rounding of the formula. A clipped value is
the gradient times an fp32 factor: two roundings of 2^-24, then one to its type.
"""

import math

import pytest
import torch

from moe_dispatch import (CudaWorkspace, MoEBlock, MoEConfig, autograd, clip_gradients, linear, quantize_rows, rms_norm,
                          route_scored)
from moe_dispatch._extension import get_extension
from tests._helpers import gpu

pytestmark = gpu

U = 2.0**-24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _grads(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, device="cuda", generator=g) * scale).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def _norm(grads):
    return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in grads))


def _check(norm, got, grads, most):
    want = _norm(grads)
    assert norm.shape == () and norm.dtype is torch.float32
    assert abs(float(norm) - want) <= want * (1 + 1e-6) * U * 1.01 + 1e-45
    factor = min(1.0, most / (want + 1e-6))
    for a, g in zip(got, grads):
        if factor == 1.0:
            assert torch.equal(a, g)
            continue
        y = g.double() * factor
        half = 0.0 if g.dtype is torch.float32 else torch.finfo(g.dtype).eps / 2
        least = torch.finfo(g.dtype).smallest_normal * torch.finfo(g.dtype).eps  # one subnormal step
        assert bool(((a.double() - y).abs() <= y.abs() * (half * 1.001 + 2 * U) + least).all())


LISTS = [[1], [5], [32768], [32769, 1, 0, 7], [0], [100_003, 65536, 3], list(range(1, 120)), [17] * 113, [3000] * 300 + [70_001],
         [2_000_003, 11, 32768 * 3]]


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES])
def test_norm_and_clipped_values(sizes, dtypes):
    grads = _grads(sizes, dtypes)
    for most in (0.5, 1e6):
        outputs = [torch.full_like(t, 9) for t in grads]
        kept = [t.clone() for t in grads]
        norm = clip_gradients(grads, most, outputs=outputs)
        _check(norm, outputs, kept, most)
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))
        assert torch.equal(norm, clip_gradients(grads, most))  # in place, the same norm
        assert all(torch.equal(a, b) for a, b in zip(grads, outputs))
        grads = kept


def test_any_alignment_shape_and_half_of_the_outputs_in_place():
    whole = torch.randn(100_000, device="cuda")
    half = torch.randn(50_001, device="cuda").half()
    grads = [whole[1:30_000].view(29_999), whole[30_001:30_001 + 64 * 33].view(64, 33), half[1:], half[:1],
             torch.randn((), device="cuda")]
    kept = [t.clone() for t in grads]
    outputs = [grads[0], torch.empty_like(grads[1]), grads[2], torch.empty_like(grads[3]), grads[4]]
    before, between = whole[0].item(), whole[30_000].item()
    norm = clip_gradients(grads, 2.0, outputs=outputs)
    _check(norm, outputs, kept, 2.0)
    assert torch.equal(grads[1], kept[1]) and torch.equal(grads[3], kept[3])
    assert whole[0].item() == before and whole[30_000].item() == between


def test_values_whose_squares_leave_fp32():
    for value in (1e30, 1e-30):
        grads = [torch.full((1000,), value, device="cuda"), torch.full((500,), -value, device="cuda")]
        kept = [t.clone() for t in grads]
        norm = clip_gradients(grads, 1.0)
        assert float(norm) == pytest.approx(value * math.sqrt(1500), rel=1e-6)
        _check(norm, grads, kept, 1.0)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_norm_that_is_no_number_changes_nothing(bad):
    grads = _grads([40_000, 100], TYPES)
    grads[1][7] = bad
    kept = [t.clone() for t in grads]
    norm = clip_gradients(grads, 1e-3)
    assert not torch.isfinite(norm)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(grads, kept))


def test_zero_gradients():
    grads = [torch.zeros(100, device="cuda"), torch.zeros(7, device="cuda", dtype=torch.bfloat16)]
    assert float(clip_gradients(grads, 1.0)) == 0.0 and not any(bool(t.any()) for t in grads)


def test_more_than_2_to_the_31_elements():
    big = torch.ones(2**31 + 100, device="cuda", dtype=torch.bfloat16)
    big[-1] = 3.0
    small = torch.full((10,), 2.0, device="cuda")
    want = math.sqrt(2**31 + 99 + 9 + 40)
    assert float(clip_gradients([small, big], 1.0)) == pytest.approx(want, rel=1e-7)
    assert float(big[-1]) == pytest.approx(3 / want, rel=2**-8) and float(small[0]) == pytest.approx(2 / want, rel=1e-6)


def test_clipping_in_graphs_beside_eager_work():
    grads = _grads([5000] * 130 + [200_000], TYPES)
    outputs = [torch.empty_like(t) for t in grads]
    eager = [torch.empty_like(t) for t in grads]
    clip_gradients(grads, 1.0, outputs=outputs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(grads, 1.0, outputs=outputs)
    for k in range(3):
        grads[0].add_(0.5)
        want = clip_gradients(grads, 1.0, outputs=eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(outputs, eager))


# -- the operators of a layer together ---------------------------------------
@pytest.mark.parametrize("tokens", [1, 24, 600])
@pytest.mark.parametrize("eight", [False, True])
def test_feed_forward_half_of_a_layer(tokens, eight):
    """Norm, scored routing on the fused router's logits, the experts, a shared expert and the residual,
    against the same steps in 64 bits with the block's own roundings of the experts' part."""
    hidden, inner, shared, experts, topk = 512, 256, 384, 16, 4
    torch.manual_seed(tokens)
    config = MoEConfig(hidden=hidden, intermediate=inner, experts=experts, topk=topk)
    block = MoEBlock(config)
    stream, attention = torch.randn(2, tokens, hidden, device="cuda").bfloat16()
    weight = (1 + 0.1 * torch.randn(hidden, device="cuda")).bfloat16()
    up = (torch.randn(2 * shared, hidden, device="cuda") / hidden**0.5).bfloat16()
    down = (torch.randn(hidden, shared, device="cuda") / shared**0.5).bfloat16()
    bias = 0.05 * torch.randn(experts, device="cuda")
    route = dict(scoring="sigmoid", bias=bias, groups=4, top_groups=2, scale=1.5)

    normed = rms_norm(attention, weight, residual=stream)
    x = normed.output
    logits = torch.empty(tokens, experts, device="cuda")
    spare_ids, spare_weights = torch.empty(tokens, 1, device="cuda", dtype=torch.int32), torch.empty(tokens, 1, device="cuda")
    get_extension().router_fused_out(x, block.router_weight, block.routing_bias, spare_ids, None, spare_weights, logits=logits)
    ids, weights = route_scored(logits, topk, **route)
    state = block.workspace(x)
    assert isinstance(state.transport, CudaWorkspace)
    state.transport.dispatch(x, ids)
    routed = state.transport.combine(block.experts_forward(state), weights)
    routed = state.transport.output if routed is None else routed
    if eight:
        middle = linear(rms_norm(attention, weight, residual=stream, quantize=True).output, quantize_rows(up),
                        activation="swiglu")
        total = linear(quantize_rows(middle), quantize_rows(down), residual=routed)
    else:
        total = linear(linear(x, up, activation="swiglu"), down, residual=routed)

    want_logits = x.double() @ block.router_weight.double().t()
    assert bool(((logits.double() - want_logits).abs() <= 1e-4 * (1 + want_logits.abs())).all())
    f = torch.nn.functional
    want = torch.zeros(tokens, hidden, device="cuda", dtype=torch.float64)
    for e in range(experts):
        rows, slots = torch.nonzero(ids == e, as_tuple=True)
        if rows.numel():
            gate, part = (x[rows].double() @ block.gate_up_weight[e].double().t()).chunk(2, -1)
            y = (f.silu(gate) * part) @ block.down_weight[e].double().t()
            want.index_add_(0, rows, y * weights[rows, slots].double().unsqueeze(-1))
    gate, part = (x.double() @ up.double().t()).chunk(2, -1)
    want += (f.silu(gate) * part) @ down.double().t()
    # bf16 holds every step between: a few roundings of 2^-8 relative to the result's size; e4m3 adds
    # 2^-4 / sqrt(3) of each of x, weights and activations, averaged over the sums.
    size = float(want.square().mean().sqrt())
    off = float((total.double() - want).square().mean().sqrt()) / size
    assert off <= (0.09 if eight else 4 * 2.0**-8), off


def test_a_training_step_of_a_layer():
    """Norm, scored routing, dispatch, a program's experts, combine and the clipped gradients: against torch
    in 64 bits on the same choice."""
    tokens, hidden, experts, topk = 96, 64, 8, 2
    torch.manual_seed(5)
    x = torch.randn(tokens, hidden, device="cuda", requires_grad=True)
    residual = torch.randn(tokens, hidden, device="cuda")
    weight = (1 + 0.1 * torch.randn(hidden, device="cuda")).requires_grad_()
    router = (torch.randn(experts, hidden, device="cuda") / 8).requires_grad_()
    inner = (torch.randn(experts, hidden, hidden, device="cuda") / 8).requires_grad_()
    target = torch.randn(tokens, hidden, device="cuda")

    normed, total = autograd.rms_norm(x, weight, residual=residual)
    ids, weights = autograd.route_scored(normed @ router.t(), topk, scoring="sigmoid", groups=4, top_groups=2)
    packed, batch = autograd.dispatch(normed, ids, experts)
    bounds = batch.offsets.tolist()
    rows = torch.cat([packed[a:b] @ inner[e] for e, (a, b) in enumerate(zip(bounds, bounds[1:]))])
    out = total + autograd.combine(rows, batch, weights)
    (out * target).sum().backward()
    leaves = (x, weight, router, inner)
    grads = [t.grad.clone() for t in leaves]
    norm = clip_gradients([t.grad for t in leaves], 1.0)

    d = [t.detach().double().requires_grad_() for t in leaves]
    h = d[0] + residual.double()
    n = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * d[1]
    s = torch.sigmoid(n @ d[2].t()).gather(1, ids.long())
    w = s / s.sum(-1, keepdim=True)
    y = torch.bmm(n.unsqueeze(1).repeat_interleave(topk, 0), d[3][ids.long().reshape(-1)].contiguous()).view(tokens, topk, hidden)
    ((h + (y * w.unsqueeze(-1)).sum(1)) * target.double()).sum().backward()
    # fp32 sums of at most 96 x 64 terms in a few stages: 1e-4 of the gradient's size.
    for got, want in zip(grads, d):
        assert float((got.double() - want.grad).norm() / want.grad.norm()) <= 1e-4
    assert float(norm) == pytest.approx(_norm(grads), rel=1e-6)
    for leaf, grad in zip(leaves, grads):
        assert bool(((leaf.grad - grad / float(norm)).abs() <= grad.abs() / float(norm) * 1e-5 + 1e-12).all())
