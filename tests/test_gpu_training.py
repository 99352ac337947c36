"""The router's losses and gradients and the transport's gradients, against 64-bit formulas.

Tolerances count roundings: u = 2^-24 for an fp32 operation, half = eps / 2 for a result
rounded once to its type, and per element the sum S of the terms' magnitudes. exp, log,
the subtraction of the maximum and a division are taken as at most V + 8 roundings of
their value, V the range of the logits; a sum of n terms as at most n + 8 of S (its
chains are far shorter than n). MFMA sums count twice a rounding per product, for
hardware that truncates.
"""

import pytest
import torch

from moe_dispatch import (combine, combine_backward, dispatch, dispatch_backward, route_backward,
                          route_logits_backward, router_loss)
from moe_dispatch._extension import get_extension
from tests._helpers import gpu

pytestmark = gpu

U = 2.0**-24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _router_case(tokens, experts, topk, seed, masked=False, hidden=None, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    case = {"logits": normal(tokens, experts) * scale, "bias": normal(experts) * 0.5, "mask": None}
    case["ids"] = torch.topk(case["logits"] + case["bias"], topk, dim=-1).indices.int().contiguous()
    if masked:
        case["mask"] = torch.rand(tokens, device="cuda", generator=g) < 0.7
    case["grad_losses"] = torch.tensor([0.3, -0.02], device="cuda")
    case["grad_weights"] = normal(tokens, topk)
    if hidden:
        case["x"] = normal(tokens, hidden).bfloat16()
        case["w"] = normal(experts, hidden) / hidden**0.5
        case["grad_x"] = normal(tokens, hidden).bfloat16()
    return case


def _reference(case, with_losses=True, with_weights=True):
    """The formulas in 64 bits: losses, counts, dv, and the scale of dv's terms."""
    v = case["logits"].double() + (case["bias"].double() if case["bias"] is not None else 0)
    tokens, experts = v.shape
    ids = case["ids"].long()
    topk = ids.shape[1]
    valid = torch.ones(tokens, device="cuda", dtype=torch.bool) if case["mask"] is None else case["mask"]
    keep = valid.double().unsqueeze(1)
    n = int(valid.sum())
    top = v.max(dim=1, keepdim=True).values
    finite = torch.isfinite(top)
    e = torch.where(finite, torch.exp(v - torch.where(finite, top, 0.0)), 0.0)
    total = torch.where(finite, e.sum(1, keepdim=True), 1.0)
    p = e / total
    lse = torch.where(finite, top + torch.log(total), 0.0).squeeze(1)
    routed = (ids >= 0) & (ids < experts)
    hits = torch.zeros(tokens, experts, device="cuda", dtype=torch.float64)
    hits.scatter_add_(1, ids.clamp(0, experts - 1), routed.double())
    counts = (hits * keep).sum(0)
    balance = experts * torch.dot(counts, (p * keep).sum(0)) / (n * n * topk) if n else torch.zeros((), device="cuda")
    z = (lse * lse * valid).sum() / n if n else torch.zeros((), device="cuda")
    dv = torch.zeros_like(v)
    scale = torch.zeros_like(v)
    if with_losses and n:
        gb, gz = case["grad_losses"].double().tolist()
        cb = gb * experts / (n * n * topk)
        mean = (p * counts).sum(1, keepdim=True)
        dv += cb * p * (counts - mean) + gz * 2 / n * lse.unsqueeze(1) * p
        scale += abs(cb) * p * (counts + mean) + abs(gz) * 2 / n * lse.abs().unsqueeze(1) * p
    if with_weights:
        chosen = torch.where(routed, v.gather(1, ids.clamp(0, experts - 1)), -float("inf"))
        w = torch.nan_to_num(torch.softmax(chosen, dim=1))  # nothing routed: 0
        dw = case["grad_weights"].double()
        dot = (w * dw).sum(1, keepdim=True)
        dv.scatter_add_(1, ids.clamp(0, experts - 1), w * (dw - dot))
        scale.scatter_add_(1, ids.clamp(0, experts - 1), w * (dw.abs() + (w * dw.abs()).sum(1, keepdim=True)))
    return {"losses": torch.stack([balance, z]).double(), "counts": counts, "n": n, "lse": lse, "dv": dv * keep,
            "scale": scale * keep, "range": float(v[torch.isfinite(v)].abs().max()) * 2 if v.numel() else 0.0}


def _within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        i = int(torch.nonzero(bad.reshape(-1))[0])
        t = tol.reshape(-1)[i] if isinstance(tol, torch.Tensor) and tol.numel() > 1 else tol
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; [{i}] {got.reshape(-1)[i].item()!r} against "
                             f"{want.reshape(-1)[i].item()!r}, tolerance {float(t):.3g}")


def _check_losses(loss, ref, tokens):
    assert torch.equal(loss.counts.double(), ref["counts"]) and int(loss.stats[-1]) == ref["n"]
    # Positive terms throughout: a relative error; a thread's chain is at most T / 256 + 32 sums.
    roundings = ref["range"] + 40 + tokens / 256
    _within(loss.balance, ref["losses"][0], float(ref["losses"][0]) * roundings * U, "balance")
    lse = ref["lse"].abs()
    delta = (ref["range"] + 16) * U * (1 + lse)
    top = float((2 * lse * delta + delta**2).max()) if lse.numel() else 0.0
    _within(loss.z, ref["losses"][1], top + float(ref["losses"][1]) * (tokens / 256 + 40) * U, "z")


def _logits_tolerance(ref):
    return ref["scale"] * (2 * ref["range"] + 60) * U + 1e-37


SHAPES = [(1, 1, 1), (1, 8, 2), (5, 3, 3), (64, 2, 1), (127, 8, 2), (333, 12, 3), (513, 16, 8), (700, 33, 4),
          (1025, 64, 6), (4096, 8, 2), (8191, 64, 8)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("tokens,experts,topk", SHAPES)
def test_losses_and_logits_gradient(tokens, experts, topk, masked):
    case = _router_case(tokens, experts, topk, tokens + experts, masked)
    args = (case["logits"], case["ids"], case["bias"])
    loss = router_loss(*args, mask=case["mask"])
    _check_losses(loss, _reference(case), tokens)
    for losses, weights in ((True, True), (True, False), (False, True), (False, False)):
        got = route_logits_backward(*args, mask=case["mask"], loss=loss if losses else None,
                                    grad_losses=case["grad_losses"] if losses else None,
                                    grad_weights=case["grad_weights"] if weights else None)
        ref = _reference(case, losses, weights)
        _within(got, ref["dv"], _logits_tolerance(ref), f"dv losses={losses} weights={weights}")


def test_no_tokens_and_no_valid_tokens():
    empty = router_loss(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 2, device="cuda", dtype=torch.int32))
    assert empty.losses.tolist() == [0, 0] and empty.stats.tolist() == [0] * 9
    case = _router_case(300, 8, 2, 1, hidden=64)
    case["mask"] = torch.zeros(300, device="cuda", dtype=torch.bool)
    args = (case["logits"], case["ids"], case["bias"])
    loss = router_loss(*args, mask=case["mask"])
    assert loss.losses.tolist() == [0, 0] and loss.stats.tolist() == [0] * 9
    gx, gw, gb = route_backward(case["x"], case["w"], *args, mask=case["mask"], loss=loss,
                                grad_losses=case["grad_losses"], grad_weights=case["grad_weights"], grad_x=case["grad_x"])
    assert torch.equal(gx, case["grad_x"]) and not gw.any() and not gb.any()
    none = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16)
    gx, gw, gb = route_backward(none, case["w"], case["logits"][:0], case["ids"][:0])
    assert gx.shape == (0, 64) and not gw.any() and not gb.any()


def test_masked_tokens_are_not_read():
    case = _router_case(200, 16, 2, 3, masked=True, hidden=64)
    clean = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in case.items()}
    off = ~case["mask"]
    case["logits"][off] = float("nan")
    case["ids"][off] = 99
    case["grad_weights"][off] = float("inf")
    results = []
    for c in (case, clean):
        args = (c["logits"], c["ids"], c["bias"])
        loss = router_loss(*args, mask=c["mask"])
        results.append((loss.losses, loss.stats) + route_backward(
            c["x"], c["w"], *args, mask=c["mask"], loss=loss, grad_losses=c["grad_losses"],
            grad_weights=c["grad_weights"], grad_x=c["grad_x"]))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,experts", [(1, 4), (200, 16), (3000, 64)])
def test_masked_rows_of_x_reach_nothing(tokens, experts):
    """Padding tokens' activations may be anything: their gradients are 0, and 0 times NaN is not."""
    case = _router_case(tokens, experts, 2, 21, masked=True, hidden=136)
    if tokens == 1:
        case["mask"][0] = False
    args = (case["logits"], case["ids"], case["bias"])
    loss = router_loss(*args, mask=case["mask"])
    dirty = case["x"].clone()
    dirty[~case["mask"]] = float("nan")
    assert dirty.isnan().any()
    clean, got = (route_backward(x, case["w"], *args, mask=case["mask"], loss=loss, grad_losses=case["grad_losses"],
                                 grad_weights=case["grad_weights"], grad_x=case["grad_x"]) for x in (case["x"], dirty))
    for a, b in zip(got, clean):
        assert torch.equal(a, b)


def test_gradients_not_wanted():
    for tokens in (0, 100):
        case = _router_case(tokens, 8, 2, 22, hidden=64)
        args = (case["x"], case["w"], case["logits"], case["ids"], case["bias"])
        full = route_backward(*args, grad_weights=case["grad_weights"])
        for wanted in range(8):
            flags = tuple(bool(wanted >> i & 1) for i in range(3))
            got = route_backward(*args, grad_weights=case["grad_weights"], gradients=flags)
            for flag, a, b in zip(flags, got, full):
                assert torch.equal(a, b) if flag else a is None


def test_disabled_experts_and_empty_rows():
    """-inf logits (disabled experts; a token with none left) and ids that were not routed."""
    case = _router_case(150, 8, 3, 4)
    case["bias"][5] = -float("inf")
    case["logits"][7] = -float("inf")
    case["logits"][9, :6] = -float("inf")
    case["ids"] = torch.topk(case["logits"] + case["bias"], 3, dim=-1).indices.int().contiguous()
    case["ids"][11, 1] = -1
    case["ids"][12] = 8
    args = (case["logits"], case["ids"], case["bias"])
    loss = router_loss(*args)
    ref = _reference(case)
    _check_losses(loss, ref, 150)
    got = route_logits_backward(*args, loss=loss, grad_losses=case["grad_losses"], grad_weights=case["grad_weights"])
    _within(got, ref["dv"], _logits_tolerance(ref), "dv")


def test_the_lowest_value_masks_like_infinity():
    """Logits masked with the type's lowest value give what -inf gives, bit for bit."""
    results = []
    for value in (torch.finfo(torch.float32).min, -float("inf")):
        case = _router_case(200, 16, 2, 16)
        case["logits"][:, 3] = value
        case["logits"][5:50, 8:] = value
        case["bias"] = None
        case["ids"] = torch.topk(case["logits"], 2, dim=-1).indices.int().contiguous()
        loss = router_loss(case["logits"], case["ids"])
        results.append((loss.losses, loss.stats, route_logits_backward(
            case["logits"], case["ids"], loss=loss, grad_losses=case["grad_losses"], grad_weights=case["grad_weights"])))
    for a, b in zip(*results):
        assert torch.equal(a, b) and torch.isfinite(a).all()


def test_an_expert_chosen_twice():
    """Ids of a program's own router may name an expert twice: both terms count."""
    case = _router_case(300, 12, 4, 14)
    case["ids"] = torch.randint(0, 12, (300, 4), device="cuda", dtype=torch.int32)
    args = (case["logits"], case["ids"], case["bias"])
    loss = router_loss(*args)
    ref = _reference(case)
    _check_losses(loss, ref, 300)
    got = route_logits_backward(*args, loss=loss, grad_losses=case["grad_losses"], grad_weights=case["grad_weights"])
    _within(got, ref["dv"], _logits_tolerance(ref), "dv")


@pytest.mark.parametrize("tokens", [100, 3000])
def test_each_gradient_alone(tokens):
    """Through the C entry any gradient may be left out; the others stay the same."""
    case = _router_case(tokens, 16, 2, 15, hidden=64)
    args = (case["x"], case["w"], case["logits"], case["ids"], case["bias"])
    full = route_backward(*args, grad_weights=case["grad_weights"], grad_x=case["grad_x"])
    lib = get_extension().lib
    need = lib.moe_route_backward_scratch_bytes(tokens, 64, 16)
    scratch = torch.empty(need, device="cuda", dtype=torch.uint8)
    # The entry takes the bias before the ids.
    inputs = [case[name].data_ptr() for name in ("x", "w", "logits", "bias", "ids")]
    for wanted in range(3):
        out = torch.full_like(full[wanted], 7.0)
        outs = [None, None, None]
        outs[wanted] = out.data_ptr()
        lib.check(lib.moe_route_backward(
            *inputs, None, None, None, case["grad_weights"].data_ptr(), case["grad_x"].data_ptr(),
            *outs, scratch.data_ptr(), need, tokens, 64, 16, 2, torch.cuda.current_stream().cuda_stream), "route")
        assert torch.equal(out, full[wanted])


def test_nan_and_infinite_logits_show():
    case = _router_case(64, 8, 2, 5)
    for value in (float("nan"), float("inf")):
        logits = case["logits"].clone()
        logits[3, 1] = value
        assert not torch.isfinite(router_loss(logits, case["ids"], case["bias"]).losses).all()
        # Other tokens' routing-weight gradients are their own.
        got = route_logits_backward(logits, case["ids"], case["bias"], grad_weights=case["grad_weights"])
        want = route_logits_backward(case["logits"], case["ids"], case["bias"], grad_weights=case["grad_weights"])
        rows = torch.arange(64, device="cuda") != 3
        assert torch.equal(got[rows], want[rows])


def test_logits_gradient_against_differences():
    """Central differences of the 64-bit losses and weights in a few random directions."""
    case = _router_case(40, 8, 2, 6, masked=True)
    loss = router_loss(case["logits"], case["ids"], case["bias"], mask=case["mask"])
    got = route_logits_backward(case["logits"], case["ids"], case["bias"], mask=case["mask"], loss=loss,
                                grad_losses=case["grad_losses"], grad_weights=case["grad_weights"]).double()

    def total(logits):
        v = (logits + case["bias"].double())[case["mask"]]
        ids = case["ids"].long()[case["mask"]]
        counts = torch.bincount(ids.reshape(-1), minlength=8).double()
        balance = 8 * torch.dot(counts / ids.numel(), torch.softmax(v, 1).mean(0))
        z = torch.logsumexp(v, 1).square().mean()
        w = torch.softmax(v.gather(1, ids), 1)
        return (case["grad_losses"].double() * torch.stack([balance, z])).sum() + (
            w * case["grad_weights"].double()[case["mask"]]).sum()

    g = torch.Generator(device="cuda").manual_seed(0)
    ref = _reference(case)
    for _ in range(4):
        d = torch.randn(40, 8, device="cuda", generator=g, dtype=torch.float64)
        step = 1e-5
        slope = (total(case["logits"].double() + step * d) - total(case["logits"].double() - step * d)) / (2 * step)
        # Third derivatives are below 10 per token here; then the gradient's own tolerance.
        tol = float((_logits_tolerance(ref) * d.abs()).sum()) + 40 * 10 * 5**3 * step**2 + 1e-10 / step * 1e-3
        assert abs(float((got * d).sum() - slope)) <= tol


def _check_route_backward(case, tokens, experts, topk, hidden):
    args = (case["logits"], case["ids"], case["bias"])
    loss = router_loss(*args, mask=case["mask"])
    gx, gw, gb = route_backward(case["x"], case["w"], *args, mask=case["mask"], loss=loss,
                                grad_losses=case["grad_losses"], grad_weights=case["grad_weights"], grad_x=case["grad_x"])
    ref = _reference(case)
    dv, tol_dv = ref["dv"], _logits_tolerance(ref)
    w, x = case["w"].double(), case["x"].double()
    base = case["grad_x"].double() if case["grad_x"] is not None else torch.zeros_like(x)
    want = base + dv @ w
    # dv and W as two bf16 parts each: 2^-16 of each factor, and the product of the rests.
    size = dv.abs() @ w.abs()
    tol = _half(torch.bfloat16) * want.abs() + size * (3 * 2.0**-16 + 2 * (3 * experts + 8) * U) \
        + tol_dv @ w.abs() + base.abs() * U
    _within(gx, want, tol * 1.01, "grad_x")
    size = dv.abs().t() @ x.abs()
    tol = size * 2 * (min(tokens, 3 * 1024) + 40) * U + tol_dv.t() @ x.abs()
    _within(gw, dv.t() @ x, tol, "grad_router_weight")
    _within(gb, dv.sum(0), dv.abs().sum(0) * (tokens / 256 + 40) * U + tol_dv.sum(0), "grad_bias")
    return gx, gw, gb


@pytest.mark.parametrize("tokens,hidden,experts,topk", [
    (1, 8, 1, 1), (1, 4096, 8, 2), (3, 72, 5, 2), (63, 512, 8, 2), (64, 1000, 12, 3), (65, 136, 16, 4), (129, 256, 17, 2),
    (300, 2048, 32, 4), (777, 1000, 33, 3), (2049, 520, 64, 6), (5000, 128, 64, 8), (1100, 65536, 8, 2)])
def test_route_backward(tokens, hidden, experts, topk):
    case = _router_case(tokens, experts, topk, tokens * 7 + experts, masked=tokens > 100, hidden=hidden)
    first = _check_route_backward(case, tokens, experts, topk, hidden)
    case["grad_x"] = None
    case["bias"] = None if experts % 2 == 0 else case["bias"]
    case["ids"] = torch.topk(case["logits"] if case["bias"] is None else case["logits"] + case["bias"], topk,
                             dim=-1).indices.int().contiguous()
    _check_route_backward(case, tokens, experts, topk, hidden)
    assert first[0].dtype == torch.bfloat16


@pytest.mark.parametrize("experts", [8, 20, 64])
def test_route_backward_of_a_streamed_base(experts):
    """Past 24 M elements of x's gradient; every expert count's variant."""
    case = _router_case(3100, experts, 2, 31, masked=True, hidden=8192)
    _check_route_backward(case, 3100, experts, 2, 8192)


def test_route_backward_follows_the_framework_router():
    """The routing weights' gradient belongs to the weights that the fused router returns."""
    ext = get_extension()
    case = _router_case(96, 8, 2, 8, hidden=256)
    ids, ids64 = (torch.empty(96, 2, device="cuda", dtype=t) for t in (torch.int32, torch.int64))
    weights, logits = torch.empty(96, 2, device="cuda"), torch.empty(96, 8, device="cuda")
    ext.router_fused_out(case["x"], case["w"], case["bias"], ids, ids64, weights, logits=logits)
    chosen = (logits.double() + case["bias"].double()).gather(1, ids64)
    _within(weights, torch.softmax(chosen, 1), 40 * U, "weights")
    case["logits"], case["ids"] = logits, ids
    _check_route_backward(case, 96, 8, 2, 256)


def test_route_backward_into_its_own_base():
    case = _router_case(130, 8, 2, 9, hidden=128)
    args = (case["x"], case["w"], case["logits"], case["ids"], case["bias"])
    want, _, _ = route_backward(*args, grad_weights=case["grad_weights"], grad_x=case["grad_x"])
    ext = get_extension()
    need = ext.lib.moe_route_backward_scratch_bytes(130, 128, 8)
    scratch = torch.empty(need, device="cuda", dtype=torch.uint8)
    gx = case["grad_x"].clone()
    ext.lib.check(ext.lib.moe_route_backward(
        case["x"].data_ptr(), case["w"].data_ptr(), case["logits"].data_ptr(), case["bias"].data_ptr(),
        case["ids"].data_ptr(), None, None, None, case["grad_weights"].data_ptr(), gx.data_ptr(), gx.data_ptr(), None,
        None, scratch.data_ptr(), need, 130, 128, 8, 2, torch.cuda.current_stream().cuda_stream), "route_backward")
    assert torch.equal(gx, want)


# -- transport ----------------------------------------------------------------
def _transport(tokens, hidden, experts, topk, dtype, alignment, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).to(dtype)
    ids = torch.randint(0, experts, (tokens, topk), device="cuda", generator=g, dtype=torch.int32)
    weights = torch.softmax(torch.randn(tokens, topk, device="cuda", generator=g), 1).contiguous()
    batch = dispatch(x, ids, experts, alignment=alignment)
    y = torch.randn(batch.packed.shape, device="cuda", generator=g).to(dtype)
    dout = torch.randn(tokens, hidden, device="cuda", generator=g).to(dtype)
    return x, ids, weights, batch, y, dout


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,hidden,experts,topk,alignment", [
    (0, 16, 4, 2, 1), (1, 1, 1, 1, 1), (1, 4096, 8, 2, 8), (7, 3, 5, 2, 1), (65, 31, 8, 3, 16), (130, 512, 16, 4, 1),
    (257, 1023, 64, 8, 8), (300, 1000, 12, 5, 128)])
def test_transport_gradients(tokens, hidden, experts, topk, alignment, dtype):
    x, ids, weights, batch, y, dout = _transport(tokens, hidden, experts, topk, dtype, alignment, tokens + hidden)
    gy, gw = combine_backward(dout, y, batch, weights)
    inverse = batch.inverse.long()
    want = torch.zeros(y.shape, device="cuda", dtype=torch.float64)
    want[inverse.reshape(-1)] = (weights.double().unsqueeze(-1) * dout.double().unsqueeze(1)).reshape(-1, hidden)
    # fp32 product, then the rounding to the type (subnormal halves: half of their spacing).
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    _within(gy, want, want.abs() * (_half(dtype) + U) * 1.01 + tiny, "grad_expert_output")
    rows = y.double()[inverse.reshape(-1)].view(tokens, topk, hidden)
    terms = rows * dout.double().unsqueeze(1)
    _within(gw, terms.sum(-1), terms.abs().sum(-1) * (hidden / 64 + 16) * U, "grad_weights")
    back = torch.randn(batch.packed.shape, device="cuda").to(dtype)
    gx = dispatch_backward(back, batch)
    parts = back.double()[inverse.reshape(-1)].view(tokens, topk, hidden)
    want = parts.sum(1)
    _within(gx, want, want.abs() * _half(dtype) + parts.abs().sum(1) * (topk + 1) * U + tiny, "grad_x")


@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 1000), (torch.float32, 1023), (torch.float16, 7)])
def test_padding_rows_are_zero(dtype, hidden):
    """64 experts of spans rounded up to 128 rows: most packed rows hold no assignment."""
    g = torch.Generator(device="cuda").manual_seed(23)
    tokens, experts = 500, 64
    x = torch.randn(tokens, hidden, device="cuda", generator=g).to(dtype)
    ids = torch.randint(0, experts, (tokens, 1), device="cuda", generator=g, dtype=torch.int32)
    batch = dispatch(x, ids, experts, alignment=128)
    y = torch.full(batch.packed.shape, float("nan"), device="cuda", dtype=dtype)
    held = torch.zeros(batch.packed.shape[0], device="cuda", dtype=torch.bool)
    held[batch.inverse.long().reshape(-1)] = True
    y[held] = 1.0
    dy, dw = combine_backward(x, y, batch, torch.ones(tokens, 1, device="cuda"))
    assert int(held.sum()) == tokens and not dy[~held].any()
    assert torch.equal(dy[batch.inverse.long().reshape(-1)], x) and dw.isfinite().all()


def test_combine_gradient_against_differences():
    """combine in 64 bits is linear in its rows and weights: a difference is exact there."""
    x, ids, weights, batch, y, dout = _transport(20, 24, 4, 2, torch.float32, 8, 3)
    gy, gw = combine_backward(dout, y, batch, weights)
    inverse = batch.inverse.long()

    def total(rows, w):
        out = (rows[inverse.reshape(-1)].view(20, 2, 24) * w.unsqueeze(-1)).sum(1)
        return (out * dout.double()).sum()

    d = torch.randn(y.shape, device="cuda", dtype=torch.float64)
    e = torch.randn(weights.shape, device="cuda", dtype=torch.float64)
    y64, w64 = y.double(), weights.double()
    slope = (total(y64 + d, w64) - total(y64 - d, w64)) / 2 + (total(y64, w64 + e) - total(y64, w64 - e)) / 2
    got = (gy.double() * d).sum() + (gw.double() * e).sum()
    size = (gy.double().abs() * d.abs()).sum() + (gw.double().abs() * e.abs()).sum()
    assert abs(float(got - slope)) <= float(size) * 64 * U


def test_gradients_are_the_same_every_time_and_under_replay():
    """Repeated calls, a side stream and graph replays give the same bits."""
    case = _router_case(777, 16, 2, 11, masked=True, hidden=520)
    _, _, weights, batch, y, dout = _transport(777, 520, 16, 2, torch.bfloat16, 8, 12)

    def run():
        args = (case["logits"], case["ids"], case["bias"])
        loss = router_loss(*args, mask=case["mask"])
        out = (loss.losses, loss.stats) + route_backward(
            case["x"], case["w"], *args, mask=case["mask"], loss=loss, grad_losses=case["grad_losses"],
            grad_weights=case["grad_weights"], grad_x=case["grad_x"])
        return out + combine_backward(dout, y, batch, weights) + (dispatch_backward(y, batch),)

    want = [t.clone() for t in run()]
    for a, b in zip(run(), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        results = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(results, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for round_ in range(3):
        for t in captured:
            t.zero_()
        case["grad_weights"].mul_(2 if round_ == 1 else 1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want if round_ == 0 else run()):
            assert torch.equal(a, b), round_


def test_autograd_inputs_are_refused():
    case = _router_case(8, 4, 1, 1)
    with pytest.raises(ValueError, match="autograd"):
        router_loss(case["logits"].requires_grad_(), case["ids"])
    with torch.no_grad():
        router_loss(case["logits"], case["ids"])


def test_training_step_through_the_transport():
    """Router, losses, dispatch, a program's own experts, combine, and every gradient back,
    against the same step in 64-bit autograd."""
    tokens, hidden, experts, topk = 160, 64, 8, 2
    ext = get_extension()
    case = _router_case(tokens, experts, topk, 21, hidden=hidden)
    ids, ids64 = (torch.empty(tokens, topk, device="cuda", dtype=t) for t in (torch.int32, torch.int64))
    weights, logits = torch.empty(tokens, topk, device="cuda"), torch.empty(tokens, experts, device="cuda")
    ext.router_fused_out(case["x"], case["w"], case["bias"], ids, ids64, weights, logits=logits)
    loss = router_loss(logits, ids, case["bias"])
    batch = dispatch(case["x"], ids, experts)
    expert_w = (torch.randn(experts, hidden, hidden, device="cuda") / hidden**0.5).bfloat16()
    ends = batch.offsets.tolist()
    y = torch.empty_like(batch.packed)
    for e in range(experts):
        y[ends[e]:ends[e + 1]] = batch.packed[ends[e]:ends[e + 1]] @ expert_w[e]
    combine(y, batch, weights)
    dout = torch.randn(tokens, hidden, device="cuda").bfloat16()
    gy, gw = combine_backward(dout, y, batch, weights)
    gp = torch.empty_like(gy)
    for e in range(experts):
        gp[ends[e]:ends[e + 1]] = gy[ends[e]:ends[e + 1]] @ expert_w[e].t().contiguous()
    gx = dispatch_backward(gp, batch)
    gx, g_router, g_bias = route_backward(case["x"], case["w"], logits, ids, case["bias"], loss=loss,
                                          grad_losses=case["grad_losses"], grad_weights=gw, grad_x=gx)

    x, w, bias = (t.double().requires_grad_() for t in (case["x"], case["w"], case["bias"]))
    v = x @ w.t() + bias
    p = torch.softmax(v, 1)
    counts = torch.bincount(ids64.reshape(-1), minlength=experts).double()
    balance = experts * torch.dot(counts / (tokens * topk), p.mean(0))
    z = torch.logsumexp(v, 1).square().mean()
    route = torch.softmax(v.gather(1, ids64), 1)
    each = torch.stack([x @ expert_w[e].double() for e in range(experts)])
    out = sum(route[:, k:k + 1] * each[ids64[:, k], torch.arange(tokens, device="cuda")] for k in range(topk))
    total = (case["grad_losses"].double() * torch.stack([balance, z])).sum() + (out * dout.double()).sum()
    want = torch.autograd.grad(total, (x, w, bias))
    # Four bf16 roundings lie between (y, gy, gp and the sum), each of values around the
    # result's own size: relative in norm, with room for their growth through the weights.
    for got, ref, name in zip((gx, g_router, g_bias), want, ("x", "router", "bias")):
        error = float((got.double() - ref).norm() / ref.norm())
        assert error <= 4 * _half(torch.bfloat16) * 2, (name, error)
