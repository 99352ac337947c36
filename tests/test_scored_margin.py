"""The error bound by which scored routing trusts fp32 keys, replayed on the CPU.

choose_fast (cuda-moe-engine_amd/csrc/scored_route.hip) orders keys in fp32 and has those compared in 64 bits that are nearer
than a margin. The margin is right when no fp32 key is further than half of it from the exact key, and no fp32 group score
further than what its comparison allows. This replays the fp32 steps with exp2 and reciprocal up to one ulp off either way
(the hardware's bound), results below 2^-126 flushed, and compares with 64 bits. The constants are the kernel's.
"""

import numpy as np
import pytest

F = np.float32
LOG2E = F(1.4426950408889634)
U = 2.0**-24


def _ulp_off(exact, rng):
    """fp32 of an exact value, then one ulp down, none or one up; below the normal range 0."""
    with np.errstate(over="ignore"):
        near = exact.astype(F)
    off = rng.integers(-1, 2, near.shape)
    out = np.where(off > 0, np.nextafter(near, F(np.inf)), np.where(off < 0, np.nextafter(near, F(0)), near))
    return np.where(out < F(2.0**-126), F(0), out).astype(F)


def _exp(x, rng):
    return _ulp_off(np.exp2(np.minimum((x * LOG2E).astype(F).astype(np.float64), 1100)), rng)


def _reciprocal(x, rng):
    return _ulp_off(1 / x.astype(np.float64), rng)


def _sigmoid(l, rng):
    """Scores, the bound's reach of each token, and the exact scores."""
    s = _reciprocal((F(1) + _exp(-l, rng)).astype(F), rng)
    top = l.max(-1, keepdims=True)
    reach = _reciprocal((F(1) + _exp(-top, rng)).astype(F), rng) * (8 + 2 * np.clip(-top, 0, 128))
    return s, reach, 8.0, 1 / (1 + np.exp(-l.astype(np.float64)))


def _softmax(l, rng, lane):
    """`lane` experts a lane: its sum one by one, then lanes in pairs."""
    top = l.max(-1, keepdims=True)
    e = _exp((l - top).astype(F), rng)
    parts = e.reshape(len(l), -1, lane)
    total = np.zeros(parts.shape[:2], F)
    for i in range(lane):
        total = (total + parts[..., i]).astype(F)
    while total.shape[-1] > 1:
        total = (total[:, ::2] + total[:, 1::2]).astype(F)
    inverse = _reciprocal(total, rng)
    x = l.astype(np.float64)
    exact = np.exp(x - x.max(-1, keepdims=True))
    return (e * inverse).astype(F), inverse * F(lane + 24), lane + 24.0, exact / exact.sum(-1, keepdims=True)


def _best_two(keys):
    best = np.sort(keys, -1)
    return best[..., -1], best[..., -2]


def _excess(s, reach, weight, exact, bias, margin=None):
    """By how much fp32 keys and group sums leave what the margin allows, at most (in parts of it)."""
    keys = (s + bias).astype(F)
    want = exact + bias.astype(np.float64)
    near = 2.0**-23 * np.maximum(reach, weight * np.abs(bias).max()) + 2.0**-124 if margin is None else margin(keys, bias)
    near = near.astype(F).astype(np.float64)
    worst = float((np.abs(keys - want) / (near / 2)).max())
    (f1, f2), (w1, w2) = _best_two(keys.reshape(len(s), -1, 8)), _best_two(want.reshape(len(s), -1, 8))
    group = (f1 + f2).astype(F)
    off = np.abs(group - (w1 + w2)) + U * (np.abs(group) + 3 * near)  # and the rounding of group +- 2.3 near
    return worst, float((off / (1.15 * near)).max())


def _biases(exact, experts, rng):
    """None, zeros, near -s/2 and -s of the token's scores (where keys cancel), small and large ones."""
    size = exact.max(-1).mean()
    ones = np.ones(experts, F)
    yield F(0) * ones
    for part in (-0.25, -0.5, -1.0, -2.0, 0.5, 30.0):
        yield F(part * size) * ones
    yield (rng.standard_normal(experts) * size).astype(F)


SHIFTS = [20, 6, 2, 0, -1, -2, -3, -5, -8, -12, -16, -24, -30, -45, -60, -75, -84, -86, -87, -88, -90, -100, -110]


@pytest.mark.parametrize("shift", SHIFTS)
def test_sigmoid_keys_stay_within_the_margin(shift):
    rng = np.random.default_rng(abs(shift) + 7)
    for spread in (0.05, 1.0, 4.0):
        l = (rng.standard_normal((400, 64)) * spread + shift).astype(F)
        scores = _sigmoid(l, rng)
        for bias in _biases(scores[3], 64, rng):
            key, group = _excess(*scores, bias)
            assert key <= 1 and group <= 1, (shift, spread, float(bias[0]), key, group)


@pytest.mark.parametrize("experts,lane", [(8, 4), (64, 4), (256, 4), (256, 8), (512, 8), (512, 16)])
def test_softmax_keys_stay_within_the_margin(experts, lane):
    rng = np.random.default_rng(experts + lane)
    for spread in (0.0, 0.05, 1.0, 5.0, 30.0):
        l = (rng.standard_normal((200, experts)) * spread).astype(F)
        l[::2, rng.integers(experts)] += F(5)  # the others at the distance where their arguments weigh most in the sum
        scores = _softmax(l, rng, lane)
        for bias in _biases(scores[3], experts, rng):
            key, group = _excess(*scores, bias)
            assert key <= 1 and group <= 1, (spread, float(bias[0]), key, group)


@pytest.mark.parametrize("shift", [-16, -30, -45, -60])
def test_a_margin_without_the_argument_is_too_small(shift):
    """Eight roundings of the largest key, whatever the logits: the argument's rounding alone passes it."""
    rng = np.random.default_rng(-shift)
    l = (rng.standard_normal((4000, 64)) * 0.1 + shift).astype(F)

    def fixed(keys, bias):
        return 2.0**-20 * np.maximum(np.abs(keys), np.abs(bias)).max(-1, keepdims=True).astype(np.float64)

    key, group = _excess(*_sigmoid(l, rng), np.zeros(64, F), fixed)
    assert max(key, group) > 1, (key, group)
