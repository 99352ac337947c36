"""Scored routing and its gradient, against 64-bit formulas.

Ids have to be the definition's, near ties among them. Weights: exp, its argument, a sum of up
to 16 terms a lane and 6 steps, divisions and the scale are under 40 roundings of a weight
(U = 2^-24); exp's argument adds one of its size, up to the logits' range R.
"""

import math

import pytest
import torch

from moe_dispatch import autograd, route_scored, route_scored_backward
from tests._helpers import gpu

pytestmark = gpu

U = 2.0**-24
INF = math.inf


def _reference(logits, topk, scoring="softmax", bias=None, groups=1, top_groups=1, group_best=2, renormalize=True,
               scale=1.0):
    """ids and weights of finite logits, or of ones with -inf (out), in 64 bits."""
    l = logits.double()
    tokens, experts = l.shape
    out = l == -INF
    if scoring == "sigmoid":
        s = 1 / (1 + torch.exp(-l))
    else:
        top = l.amax(-1, keepdim=True)
        e = torch.exp(l - torch.where(torch.isfinite(top), top, 0.0))
        total = e.sum(-1, keepdim=True)
        s = e / torch.where(total > 0, total, 1.0)
    keys = (s if bias is None else s + bias.double()).masked_fill(out, -INF)
    order = keys if bias is not None else l
    shut = torch.zeros_like(out)
    if groups > 1:
        inside = keys.view(tokens, groups, -1)
        best = torch.sort(inside, dim=-1, descending=True).values[..., :group_best]
        score = torch.where(best > -INF, best, 0.0).sum(-1)
        score = torch.where(best[..., 0] > -INF, score, -INF)
        kept = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :top_groups]
        is_open = torch.zeros_like(score, dtype=torch.bool).scatter_(1, kept, True)
        shut = ~is_open.repeat_interleave(experts // groups, dim=1)
    # Experts of other groups never; ones that are out last, in order.
    rank = torch.where(shut, 2, torch.where(out, 1, 0))
    first = torch.sort(torch.where(rank == 0, order, -INF), dim=-1, descending=True, stable=True).indices
    ids = first.gather(1, torch.sort(rank.gather(1, first), dim=-1, stable=True).indices)
    picks = ids[:, :topk].clone()
    weights = s.gather(1, picks)
    if renormalize:
        if scoring == "sigmoid":
            # In logarithms: a sum of scores that all underflow keeps its ratios.
            ls = torch.nn.functional.logsigmoid(l).gather(1, picks)
        else:
            ls = l.gather(1, picks)
        top = ls.amax(-1, keepdim=True)
        e = torch.exp(ls - torch.where(torch.isfinite(top), top, 0.0))
        total = e.sum(-1, keepdim=True)
        weights = e / torch.where(total > 0, total, 1.0)
    return picks.int(), weights * scale


def _weights_near(got, want, logits, what):
    finite = logits[torch.isfinite(logits)]
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    tol = want.abs() * (40 + 2 * spread) * U + 1e-37
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} off, by {float(((got.double() - want).abs() / want.abs()).nan_to_num().max()):.3g}"


def _logits(tokens, experts, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(tokens, experts, device="cuda", generator=g) * scale


# experts, topk, groups, top_groups: every number of lanes and experts a lane among them
CHOICES = [(1, 1, 1, 1), (2, 2, 1, 1), (3, 3, 1, 1), (8, 2, 1, 1), (13, 8, 1, 1), (33, 4, 1, 1), (64, 6, 8, 4), (64, 8, 16, 3),
           (60, 6, 12, 2), (100, 8, 20, 7), (127, 7, 1, 1), (160, 6, 8, 3), (192, 8, 6, 2), (256, 8, 8, 4),
           (289, 8, 17, 4), (300, 5, 3, 1), (495, 8, 15, 6), (510, 8, 2, 1), (512, 8, 1, 1), (512, 8, 64, 9), (64, 2, 64, 2),
           (128, 8, 64, 8), (257, 3, 1, 1), (9, 3, 3, 1), (510, 6, 34, 5)]


@pytest.mark.parametrize("experts,topk,groups,top_groups", CHOICES)
def test_routes_against_the_definition(experts, topk, groups, top_groups):
    for i, tokens in enumerate((1, 37, 700)):
        for scoring in ("softmax", "sigmoid"):
            for with_bias in (False, True):
                logits = _logits(tokens, experts, 10 * experts + i, scale=1.0 + i)
                bias = _logits(1, experts, 7)[0] * (0.1 if scoring == "sigmoid" else 0.3 / experts) if with_bias else None
                for best, renormalize, scale in ((2, True, 1.0), (1, False, 2.5)):
                    options = dict(scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=best,
                                   renormalize=renormalize, scale=scale)
                    ids, weights = route_scored(logits, topk, **options)
                    want_ids, want = _reference(logits, topk, **options)
                    assert torch.equal(ids, want_ids), (tokens, options)
                    _weights_near(weights, want, logits, (tokens, options))
    assert route_scored(logits[:0], topk, groups=groups, top_groups=top_groups)[0].shape == (0, topk)


def test_choices_that_fp32_cannot_tell_apart():
    """Scores one ulp of the logit apart round to one fp32 score; equal ones are ties."""
    g = torch.Generator(device="cuda").manual_seed(1)
    for experts, groups, top_groups in ((64, 1, 1), (64, 8, 4), (256, 8, 2), (12, 1, 1), (512, 16, 3)):
        for center, scoring in ((3.0, "sigmoid"), (9.0, "sigmoid"), (0.5, "softmax")):
            ulp = 2.0**-22 if center == 3.0 else 2.0**-20 if center == 9.0 else 2.0**-24
            steps = torch.randint(0, 40, (200, experts), device="cuda", generator=g)
            logits = (center + steps.double() * ulp).float()
            bias = torch.full((experts,), 0.125, device="cuda")
            # A group's best alone: sums of two such scores differ by less than 64 bits hold.
            options = dict(scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=1)
            ids, _ = route_scored(logits, min(8, experts), **options)
            assert torch.equal(ids, _reference(logits, min(8, experts), **options)[0]), (experts, groups, center)
    # Wholly equal: the lowest indexes, of the lowest groups.
    logits = torch.zeros(5, 64, device="cuda")
    for bias in (None, torch.zeros(64, device="cuda")):
        ids, weights = route_scored(logits, 4, scoring="sigmoid", bias=bias, groups=8, top_groups=2)
        assert ids.tolist() == [[0, 1, 2, 3]] * 5 and torch.equal(weights, torch.full_like(weights, 0.25))


@pytest.mark.parametrize("experts,topk,groups,top_groups", [(64, 8, 1, 1), (256, 8, 8, 4), (256, 6, 1, 1), (512, 8, 16, 4),
                                                            (160, 6, 8, 3), (510, 5, 2, 1)])
@pytest.mark.parametrize("scoring,with_bias", [("sigmoid", True), ("softmax", True), ("softmax", False), ("sigmoid", False)])
def test_clusters_of_near_and_equal_keys(experts, topk, groups, top_groups, scoring, with_bias):
    """Two to forty keys within an fp32 rounding or equal, above, across and below the last choice, spread over the
    experts or side by side."""
    g = torch.Generator(device="cuda").manual_seed(experts + topk)
    logits = torch.randn(600, experts, device="cuda", generator=g)
    for t in range(600):
        size, at = 2 + t % 39, t % 12
        row = logits[t]
        order = torch.argsort(row, descending=True)
        where = order[at:at + size] if t % 3 else (torch.arange(size, device="cuda") + t) % experts
        value = row[order[at]]
        step = torch.arange(size, device="cuda") * (0.0 if t % 2 else 1.2e-7) * value.abs()
        row[where] = value + step
    bias = torch.full((experts,), 0.25, device="cuda") if with_bias else None
    options = dict(scoring=scoring, bias=bias, groups=groups, top_groups=top_groups)
    ids, weights = route_scored(logits, topk, **options)
    want_ids, want = _reference(logits, topk, **options)
    assert torch.equal(ids, want_ids)
    _weights_near(weights, want, logits, options)


@pytest.mark.parametrize("experts,groups,top_groups", [(256, 8, 4), (160, 8, 3), (510, 34, 5), (512, 16, 4), (64, 4, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_groups_that_are_near_or_equal_at_the_cut(experts, groups, top_groups, scoring):
    """The last group in and the first one out hold the same logits, in another order, or one that is an ulp more."""
    g = torch.Generator(device="cuda").manual_seed(groups)
    size = experts // groups
    logits = torch.randn(300, experts, device="cuda", generator=g)
    for best in (1, 2):
        options = dict(scoring=scoring, bias=None, groups=groups, top_groups=top_groups, group_best=best)
        inside = logits.view(300, groups, size)
        order = torch.argsort(torch.sort(inside, -1, descending=True).values[..., :best].exp().sum(-1), -1, descending=True)
        tokens = torch.arange(300, device="cuda")
        last, out = order[:, top_groups - 1], order[:, top_groups]
        near = inside.clone()
        near[tokens, out] = inside[tokens, last].flip(-1)
        top = near[tokens, out].argmax(-1)
        more = near[tokens, out, top]
        near[tokens[::2], out[::2], top[::2]] = torch.nextafter(more, more + 1)[::2]
        near = near.view(300, experts)
        ids, weights = route_scored(near, 6, **options)
        want_ids, want = _reference(near, 6, **options)
        assert torch.equal(ids, want_ids), best
        _weights_near(weights, want, near, options)


def test_a_bias_that_drowns_scores():
    """Keys of a bias so large that fp32 keys would lose the scores' differences."""
    logits = _logits(400, 64, 2)
    for value in (1000.0, -1000.0, 1e6):
        for groups, top_groups in ((1, 1), (8, 4)):
            options = dict(scoring="sigmoid", bias=torch.full((64,), value, device="cuda"), groups=groups,
                           top_groups=top_groups)
            assert torch.equal(route_scored(logits, 6, **options)[0], _reference(logits, 6, **options)[0])


def test_groups_whose_sums_leave_fp32():
    bias = torch.tensor([3.3e38, 1e38, 2.5e38, 2.4e38], device="cuda")
    logits = _logits(70, 4, 12)
    for scoring in ("softmax", "sigmoid"):
        ids, _ = route_scored(logits, 2, scoring=scoring, bias=bias, groups=2, top_groups=1)
        assert ids.tolist() == [[2, 3]] * 70


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_experts_that_are_out(scoring, with_bias):
    """-inf logits: some, all but a few, whole groups, everything."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for experts, topk, groups, top_groups in ((16, 4, 1, 1), (64, 6, 8, 3), (60, 8, 12, 2), (512, 8, 16, 2), (5, 5, 1, 1)):
        logits = torch.randn(300, experts, device="cuda", generator=g)
        logits[torch.rand(300, experts, device="cuda", generator=g) < 0.5] = -INF
        logits[:40, topk - 1:] = -INF
        logits[40:60] = -INF
        logits[60:80, : experts // 2] = -INF
        bias = torch.randn(experts, device="cuda", generator=g) * 0.2 if with_bias else None
        for best, renormalize in ((2, True), (1, False)):
            options = dict(scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=best,
                           renormalize=renormalize)
            ids, weights = route_scored(logits, topk, **options)
            want_ids, want = _reference(logits, topk, **options)
            assert torch.equal(ids, want_ids), (experts, options)
            _weights_near(weights, want, logits, (experts, options))
            assert torch.equal(weights[40:60], torch.zeros_like(weights[40:60]))
            grad = route_scored_backward(torch.ones_like(weights), logits, ids, scoring=scoring, renormalize=renormalize)
            assert torch.isfinite(grad).all()


def test_values_that_are_no_numbers():
    """NaN logits: the token's weights are NaN, its ids different experts; other tokens are untouched."""
    logits = _logits(130, 64, 4)
    bias = _logits(1, 64, 5)[0] * 0.1
    for options in (dict(scoring="sigmoid", bias=bias, groups=8, top_groups=4), dict(scoring="softmax"),
                    dict(scoring="softmax", bias=bias, renormalize=False), dict(scoring="sigmoid", renormalize=False)):
        clean_ids, clean = route_scored(logits, 6, **options)
        bad = logits.clone()
        bad[3, 10] = float("nan")
        bad[70] = float("nan")
        bad[90, 5] = INF
        ids, weights = route_scored(bad, 6, **options)
        keep = [t for t in range(130) if t not in (3, 70, 90)]
        assert torch.equal(ids[keep], clean_ids[keep]) and torch.equal(weights[keep], clean[keep])
        assert torch.isnan(weights[3]).all() and torch.isnan(weights[70]).all()
        assert all(len(set(row)) == 6 and 0 <= min(row) and max(row) < 64 for row in ids.tolist())
        assert 10 not in ids[3].tolist()
        if options["scoring"] == "softmax":
            assert torch.isnan(weights[90]).any()
        else:
            assert torch.isfinite(weights[90]).all()


def test_extreme_logits_keep_their_ratios():
    """Scores that underflow fp32 are renormalised by their ratios."""
    for base in (-60.0, -200.0, -1000.0, 80.0):
        logits = _logits(50, 16, 6) + base
        for scoring in ("softmax", "sigmoid"):
            ids, weights = route_scored(logits, 4, scoring=scoring)
            want_ids, want = _reference(logits, 4, scoring=scoring)
            assert torch.equal(ids, want_ids)
            tol = want * (60 + 2 * abs(base)) * U
            assert bool(((weights.double() - want).abs() <= tol).all()), (base, scoring)


def _dense_gradient(logits, ids, grad, scoring, renormalize, scale):
    l = logits.double().requires_grad_()
    s = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, -1)
    w = s.gather(1, ids.long())
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    (w * scale * grad.double()).sum().backward()
    return l.grad


@pytest.mark.parametrize("experts,topk", [(1, 1), (3, 2), (8, 2), (17, 8), (64, 6), (100, 4), (256, 8), (300, 1), (512, 8)])
def test_gradient_against_the_formula(experts, topk):
    for tokens in (1, 65, 900):
        logits = _logits(tokens, experts, experts + tokens, scale=2.0)
        grad = _logits(tokens, topk, 8)
        for scoring in ("softmax", "sigmoid"):
            for renormalize in (True, False):
                ids, _ = route_scored(logits, topk, scoring=scoring, renormalize=renormalize)
                got = route_scored_backward(grad, logits, ids, scoring=scoring, renormalize=renormalize, scale=2.5)
                want = _dense_gradient(logits, ids, grad, scoring, renormalize, 2.5)
                s = torch.softmax(logits.double(), -1) if scoring == "softmax" else torch.sigmoid(logits.double())
                if renormalize:
                    chosen = torch.zeros_like(s).scatter_(1, ids.long(), s.gather(1, ids.long()))
                    s = chosen / chosen.sum(-1, keepdim=True)
                # Terms: each is a score times gradients of at most the row's largest and their weighted sum.
                size = 2.5 * s * 2 * grad.double().abs().amax(-1, keepdim=True)
                spread = float(logits.max() - logits.min())
                # The reference's own rounding: experts that were not chosen have a gradient of exactly 0
                # when renormalised, which autograd's chain of softmax, sum and division gives as a
                # difference of terms of at most this size, rounded in 64 bits a few times each.
                own = 2.5 * grad.double().abs().amax(-1, keepdim=True) * topk * 16 * 2.0**-52
                bad = ~((got.double() - want).abs() <= size * (60 + 2 * spread) * U + own)
                assert not bool(bad.any()), (tokens, scoring, renormalize, int(bad.sum()))
                if topk == 1 and renormalize:
                    assert torch.equal(got, torch.zeros_like(got))


def test_gradient_against_differences():
    """Central differences of the 64-bit definition with the ids held: h^2 / 6 of its third derivative
    is 1e-10 of the value."""
    logits = _logits(40, 24, 9)
    grad, v = _logits(40, 4, 10), _logits(40, 24, 11).double()
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            ids, _ = route_scored(logits, 4, scoring=scoring, renormalize=renormalize)

            def f(h):
                l = logits.double() + h * v
                s = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, -1)
                w = s.gather(1, ids.long())
                w = w / w.sum(-1, keepdim=True) if renormalize else w
                return float((w * grad.double()).sum())

            want = (f(1e-5) - f(-1e-5)) / 2e-5
            got = route_scored_backward(grad, logits, ids, scoring=scoring, renormalize=renormalize).double()
            size = float((got * v).abs().sum()) + float(grad.abs().sum())
            assert abs(float((got * v).sum()) - want) <= size * (100 * U + 1e-8)


def test_ids_that_are_out_of_range_or_repeated():
    logits = _logits(20, 16, 12)
    ids, _ = route_scored(logits, 4, renormalize=False)
    grad = _logits(20, 4, 13)
    odd = ids.clone()
    odd[:, 2] = -1
    odd[:, 3] = 99
    got = route_scored_backward(grad, logits, odd, renormalize=False)
    want = route_scored_backward(grad[:, :2].contiguous(), logits, ids[:, :2].contiguous(), renormalize=False)
    assert bool(((got - want).abs() <= 1e-6).all())
    twice = ids.clone()
    twice[:, 1] = twice[:, 0]
    got = route_scored_backward(grad, logits, twice, scoring="sigmoid", renormalize=False)
    want = _dense_gradient(logits, twice, grad, "sigmoid", False, 1.0)
    assert bool(((got.double() - want).abs() <= 1e-6).all())


def test_autograd_route_scored():
    logits = _logits(33, 64, 14).requires_grad_()
    bias = _logits(1, 64, 15)[0] * 0.1
    options = dict(scoring="sigmoid", bias=bias, groups=8, top_groups=3, scale=2.0)
    ids, weights = autograd.route_scored(logits, 6, **options)
    grad = _logits(33, 6, 16)
    weights.backward(grad)
    assert torch.equal(logits.grad, route_scored_backward(grad, logits.detach(), ids, scoring="sigmoid", scale=2.0))
    with pytest.raises(ValueError, match="bias"):
        autograd.route_scored(logits, 6, bias=bias.clone().requires_grad_())


def test_scored_routes_in_a_graph_beside_eager_work():
    logits, grad = _logits(300, 256, 17), _logits(300, 8, 18)
    bias = _logits(1, 256, 19)[0] * 0.1
    options = dict(scoring="sigmoid", bias=bias, groups=8, top_groups=4)

    def step():
        ids, weights = route_scored(logits, 8, **options)
        return ids, weights, route_scored_backward(grad, logits, ids, scoring="sigmoid")

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        logits.copy_(_logits(300, 256, 30 + seed))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_many_tokens():
    """The largest batch: its last tokens as in a small call."""
    tokens = 2**21
    logits = _logits(8, 512, 20).repeat(tokens // 8, 1)
    options = dict(scoring="sigmoid", bias=_logits(1, 512, 21)[0] * 0.1, groups=16, top_groups=4)
    ids, weights = route_scored(logits, 8, **options)
    want_ids, want = route_scored(logits[:8].clone(), 8, **options)
    assert torch.equal(ids[-8:], want_ids) and torch.equal(weights[-8:], want)
    grad = route_scored_backward(weights, logits, ids, scoring="sigmoid")
    assert torch.equal(grad[-8:], route_scored_backward(want, logits[:8].clone(), want_ids, scoring="sigmoid"))
