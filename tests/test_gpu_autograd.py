"""The differentiable forms: gradients of whole steps against 64-bit autograd."""

import pytest
import torch

from moe_dispatch import AdapterGroups, autograd
from moe_dispatch.experts import grouped_linear
from tests._helpers import gpu
from tests.test_gpu_training import U, _half, _within

pytestmark = gpu

BF16 = torch.bfloat16


def _normal(g, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def test_low_rank_add_gradients():
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens, hidden, width, rank, adapters = 90, 64, 136, 8, 3
    leaves = [_normal(g, tokens, width), _normal(g, tokens, hidden), _normal(g, adapters, rank, hidden, scale=hidden**-0.5),
              _normal(g, adapters, rank, width, scale=rank**-0.5)]
    scales = torch.rand(adapters, device="cuda", generator=g) + 0.5
    ids = torch.randint(-1, adapters, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    groups = AdapterGroups(tokens, adapters)
    groups.assign(ids)
    for leaf in leaves:
        leaf.requires_grad_()
    y = autograd.low_rank_add(*leaves, groups, scales=scales)
    dy = _normal(g, tokens, width)
    y.backward(dy)
    base, x, down, up = (leaf.detach().double().requires_grad_() for leaf in leaves)
    out = base
    for a in range(adapters):
        rows = torch.nonzero(ids == a).squeeze(1)
        out = out.index_add(0, rows, (x[rows] @ down[a].t()) @ up[a] * float(scales[a]))
    out.backward(dy.double())
    assert torch.equal(leaves[0].grad, dy)
    # One rounding to bf16 each; sums of at most 90 rows and 136 columns around it.
    for got, want in zip(leaves[1:], (x, down, up)):
        size = want.grad.abs().max()
        _within(got.grad, want.grad, want.grad.abs() * _half(BF16) + size * (2.0**-16 * 8 + 400 * U), "gradient")
    # Frozen adapters: x alone gets a gradient.
    x = leaves[1].detach().clone().requires_grad_()
    autograd.low_rank_add(leaves[0].detach(), x, leaves[2].detach(), leaves[3].detach(), groups, scales=scales).backward(dy)
    assert torch.equal(x.grad, leaves[1].grad)
    y = autograd.low_rank_add(*leaves, groups, scales=scales)
    groups.assign(ids)
    with pytest.raises(RuntimeError, match="another assignment"):
        y.backward(dy)


def test_gradients_cut_out_of_a_larger_one():
    """A result joined with others behind an odd number of elements: its gradient starts there."""
    g = torch.Generator(device="cuda").manual_seed(5)
    groups = AdapterGroups(20, 2)
    groups.assign(torch.zeros(20, device="cuda", dtype=torch.int32))
    operands = [_normal(g, 20, 64), _normal(g, 2, 4, 64), _normal(g, 2, 4, 16)]
    head, dy = _normal(g, 3), _normal(g, 320)
    grads = []
    for cut in (True, False):
        leaves = [t.clone().requires_grad_() for t in operands]
        y = autograd.low_rank_add(None, *leaves, groups)
        if cut:
            torch.cat((head, y.reshape(-1))).backward(torch.cat((head, dy)))
        else:
            y.backward(dy.reshape(20, 16))
        grads.append([leaf.grad for leaf in leaves])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_two_micro_batches_in_flight():
    """Forward twice, then backward twice: no call disturbs what another kept."""
    g = torch.Generator(device="cuda").manual_seed(1)
    w = _normal(g, 8, 64, scale=0.125, dtype=torch.float32).requires_grad_()
    bias = torch.zeros(8, device="cuda", requires_grad=True)

    def forward(x):
        routed = autograd.route(x, w, bias, 2)
        packed, batch = autograd.dispatch(x, routed.ids, 8, alignment=8)
        return autograd.combine(packed * 2, batch, routed.weights).float().square().sum() + routed.losses.sum()

    xs = [_normal(g, 50, 64), _normal(g, 30, 64)]
    apart = []
    for x in xs:
        apart.append(torch.autograd.grad(forward(x), (w, bias)))
    totals = [forward(x) for x in xs]
    together = [torch.autograd.grad(total, (w, bias)) for total in totals]
    for a, b in zip(apart, together):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_layer_with_expert_adapters():
    """Fine-tuning step: router and per-expert adapters train around frozen grouped weights."""
    g = torch.Generator(device="cuda").manual_seed(2)
    tokens, hidden, width, experts, topk, rank = 100, 64, 64, 4, 2, 8
    x = _normal(g, tokens, hidden).requires_grad_()
    router = _normal(g, experts, hidden, scale=hidden**-0.5, dtype=torch.float32).requires_grad_()
    bias = (torch.randn(experts, device="cuda", generator=g) * 0.1).requires_grad_()
    frozen = _normal(g, experts, width, hidden, scale=hidden**-0.5)
    down = _normal(g, experts, rank, hidden, scale=hidden**-0.5).requires_grad_()
    up = _normal(g, experts, rank, width, scale=rank**-0.5).requires_grad_()
    mask = torch.arange(tokens, device="cuda") < 90
    coefficients = torch.tensor([0.5, 0.1], device="cuda")

    class Frozen(torch.autograd.Function):
        @staticmethod
        def forward(ctx, packed, offsets):
            ctx.offsets = offsets
            out = torch.zeros(packed.shape[0], width, device="cuda", dtype=BF16)
            return grouped_linear(packed, frozen, offsets[1:], backend="hip", output=out, offsets=offsets)

        @staticmethod
        def backward(ctx, grad):
            back = frozen.transpose(1, 2).contiguous()
            out = torch.zeros(grad.shape[0], hidden, device="cuda", dtype=BF16)
            return grouped_linear(grad.contiguous(), back, ctx.offsets[1:], backend="hip", output=out,
                                  offsets=ctx.offsets), None

    routed = autograd.route(x, router, bias, topk, mask=mask)
    packed, batch = autograd.dispatch(x, routed.ids, experts, alignment=8)
    owner = torch.full((packed.shape[0],), -1, device="cuda", dtype=torch.int32)
    owner[batch.inverse.reshape(-1).long()] = routed.ids.reshape(-1)
    groups = AdapterGroups(packed.shape[0], experts)
    groups.assign(owner)
    y = autograd.low_rank_add(Frozen.apply(packed, batch.offsets), packed, down, up, groups)
    out = autograd.combine(y, batch, routed.weights)
    target = _normal(g, tokens, width) * mask.unsqueeze(1)
    total = (out.float() * target).sum() + (routed.losses * coefficients).sum()
    got = torch.autograd.grad(total, (x, router, bias, down, up))

    leaves = [t.detach().double().requires_grad_() for t in (x, router, bias, down, up)]
    x64, router64, bias64, down64, up64 = leaves
    v = x64 @ router64.t() + bias64
    ids = routed.ids.long()
    weights = torch.softmax(v.gather(1, ids), 1)
    # A padding token's routing weights pass no gradient on.
    weights = torch.where(mask.unsqueeze(1), weights, weights.detach())
    counts = torch.bincount(ids[mask].reshape(-1), minlength=experts).double()
    assert torch.equal(routed.counts.double(), counts)
    balance = experts * torch.dot(counts / counts.sum(), torch.softmax(v[mask], 1).mean(0))
    z = torch.logsumexp(v[mask], 1).square().mean()
    each = torch.stack([x64 @ frozen[e].double().t() + (x64 @ down64[e].t()) @ up64[e] for e in range(experts)])
    mixed = sum(weights[:, k:k + 1] * each[ids[:, k], torch.arange(tokens, device="cuda")] for k in range(topk))
    want = torch.autograd.grad((mixed * target.double()).sum()
                               + (torch.stack([balance, z]) * coefficients.double()).sum(), leaves)
    # In norm: at most six bf16 roundings lie on a path (grouped product, adapter, combine and
    # their gradients), each half an eps of values of the result's size.
    for a, b, name in zip(got, want, ("x", "router", "bias", "down", "up")):
        error = float((a.double() - b).norm() / b.norm())
        assert error <= 6 * _half(BF16) * 2, (name, error)


def test_refusals():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = _normal(g, 8, 64).requires_grad_()
    w, bias = torch.zeros(4, 64, device="cuda"), torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="at least one token"):
        autograd.route(x[:0], w, bias, 2)
    with pytest.raises(ValueError, match="topk"):
        autograd.route(x, w, bias, 5)
    groups = AdapterGroups(8, 2)
    groups.assign(torch.zeros(8, device="cuda", dtype=torch.int32))
    down, up = _normal(g, 2, 4, 64), _normal(g, 2, 4, 16)
    with pytest.raises(ValueError, match="scales"):
        autograd.low_rank_add(None, x, down, up, groups, scales=torch.ones(2, device="cuda", requires_grad=True))
    y = autograd.low_rank_add(None, x, down, up, groups)
    first, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        first.float().sum().backward()


def test_capture_is_refused(monkeypatch):
    g = torch.Generator(device="cuda").manual_seed(4)
    x = _normal(g, 8, 64).requires_grad_()
    w, bias = torch.zeros(4, 64, device="cuda"), torch.zeros(4, device="cuda")
    routed = autograd.route(x, w, bias, 2)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="eager"):
        autograd.route(x, w, bias, 2)
    with pytest.raises(RuntimeError, match="eager"):
        routed.losses.sum().backward()
