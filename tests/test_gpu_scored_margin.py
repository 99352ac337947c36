"""Scored routing where fp32 scores do not tell which groups or experts are ahead, against 64 bits."""

import pytest
import torch

from moe_dispatch import route_scored
from tests._helpers import gpu
from tests.test_gpu_scored import _reference

pytestmark = gpu


def _near_groups(tokens, experts, groups, best, shift, seed):
    """Logits around `shift` whose groups' best one or two sum to nearly the same: 1e-8 to 1e-5 apart, either way."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn(tokens, experts, device="cuda", generator=g) * 0.5).double()
    inside = logits.view(tokens, groups, -1)

    def size(group):
        s = torch.sigmoid(group + shift)
        return torch.topk(s, min(best, s.shape[-1]), -1).values.sum(-1)

    want = size(inside[:, 0])
    for j in range(1, groups):
        apart = 10 ** (-8 + 3 * torch.rand(tokens, device="cuda", generator=g, dtype=torch.float64))
        apart *= torch.randint(0, 2, (tokens,), device="cuda", generator=g) * 2 - 1
        for _ in range(3):  # of a sigmoid, by Newton's steps in the logits
            now = size(inside[:, j])
            s = torch.sigmoid(inside[:, j] + shift)
            slope = (1 - torch.topk(s, 1, -1).values[:, 0]).clamp(min=1e-3)
            inside[:, j] += ((torch.log(want / now) + apart) / slope).unsqueeze(-1)
    return (logits + shift).float()


SHAPES = [(256, 8, 4), (64, 4, 2), (64, 8, 4), (24, 2, 1), (12, 3, 2), (510, 34, 5), (512, 16, 4)]


@pytest.mark.parametrize("experts,groups,top_groups", SHAPES)
@pytest.mark.parametrize("shift", [4.0, 0.0, -4.0, -12.0, -16.0, -24.0, -30.0, -45.0, -60.0, -80.0, -87.0, -88.0, -95.0])
def test_near_groups_of_sigmoid_scores_at_any_size(experts, groups, top_groups, shift):
    for best in (1, 2):
        logits = _near_groups(1500, experts, groups, best, shift, groups + best)
        middle = float(torch.sigmoid(logits.double()).mean())
        for bias in (None, 0.0, -0.25, -0.5 * middle, -middle):
            b = None if bias is None else torch.full((experts,), bias, device="cuda")
            options = dict(scoring="sigmoid", bias=b, groups=groups, top_groups=top_groups, group_best=best)
            ids, _ = route_scored(logits, 4, **options)
            want, _ = _reference(logits, 4, **options)
            wrong = int((ids != want).any(-1).sum())
            assert wrong == 0, (best, bias, wrong)


@pytest.mark.parametrize("shift", [0.0, -5.0, -16.0, -45.0, -87.5, -100.0])
@pytest.mark.parametrize("experts", [8, 64, 256, 512])
def test_near_keys_under_a_bias_that_cancels_scores(experts, shift):
    """Keys s + b with b near -s, and zero: their order is that of scores whose roundings are those of s."""
    g = torch.Generator(device="cuda").manual_seed(experts)
    logits = shift + 1e-6 * abs(shift) * torch.randn(1000, experts, device="cuda", generator=g) + 1e-3 * torch.randn(
        1000, 1, device="cuda", generator=g)
    for scoring in ("sigmoid", "softmax"):
        s = torch.sigmoid(logits.double()) if scoring == "sigmoid" else torch.softmax(logits.double(), -1)
        for part in (0.0, -0.5, -1.0):
            bias = (part * s.mean(0)).float()
            options = dict(scoring=scoring, bias=bias)
            want, _ = _reference(logits, 6, **options)
            assert torch.equal(route_scored(logits, 6, **options)[0], want), (scoring, part)


@pytest.mark.parametrize("experts,groups,top_groups", [(64, 1, 1), (64, 8, 4), (12, 3, 2), (256, 8, 4), (510, 34, 5)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [True, False])
def test_values_that_are_no_numbers_leave_the_others_their_order(experts, groups, top_groups, scoring, with_bias):
    """NaN is out: the choice is that of the row with -inf in its place. +inf outweighs the rest: of the row with a
    logit so large that all others' scores are 0 beside it (sigmoid: 1)."""
    g = torch.Generator(device="cuda").manual_seed(experts)
    logits = torch.randn(60, experts, device="cuda", generator=g)
    bias = 0.01 * torch.randn(experts, device="cuda", generator=g) if with_bias else None
    for best in (1, 2):
        options = dict(scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=best)
        clean, _ = route_scored(logits, 4, **options)
        rows = torch.arange(60, device="cuda")
        for place in ("first", "chosen", "last", "several"):
            where = torch.zeros(60, experts, dtype=torch.bool, device="cuda")
            if place == "chosen":
                where[rows, clean[:, 1].long()] = True
            else:
                where[:, {"first": [0], "last": [experts - 1], "several": [0, 1, 2, experts // 2]}[place]] = True
            for value, stand_in in ((float("nan"), float("-inf")), (float("inf"), 2e4)):
                ids, weights = route_scored(logits.masked_fill(where, value), 4, **options)
                want, _ = _reference(logits.masked_fill(where, stand_in), 4, **options)
                assert torch.equal(ids, want), (best, place, value)
                if value != value:
                    assert torch.isnan(weights).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_logits_of_the_lowest_value(scoring):
    """fp32's lowest value masks as -inf does, but stays an expert: of score 0, ahead of those that are out."""
    g = torch.Generator(device="cuda").manual_seed(4)
    lowest = torch.finfo(torch.float32).min
    for experts, groups, top_groups in ((64, 1, 1), (256, 8, 4), (12, 3, 2), (510, 34, 5)):
        logits = torch.randn(200, experts, device="cuda", generator=g)
        for share in (0.5, 0.98, 1.0):
            logits[torch.rand(200, experts, device="cuda", generator=g) < share] = lowest
            logits[:50][torch.rand(50, experts, device="cuda", generator=g) < 0.5] = float("-inf")
            for bias in (None, 0.01 * torch.randn(experts, device="cuda", generator=g)):
                options = dict(scoring=scoring, bias=bias, groups=groups, top_groups=top_groups)
                ids, weights = route_scored(logits, 4, **options)
                want, _ = _reference(logits, 4, **options)
                assert torch.equal(ids, want) and not bool(torch.isnan(weights).any())
