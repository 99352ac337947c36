"""Low-rank adapters, forward and backward, against 64-bit formulas.

Tolerances count roundings as in test_gpu_training: u = 2^-24 an fp32 rounding (MFMA sums
count two per product), half = eps / 2 the one rounding to bf16. h enters the second
product as two bf16 parts: 2^-16 of its value.
"""

import pytest
import torch

from moe_dispatch import AdapterGroups, CudaWorkspace, low_rank_add, low_rank_backward
from moe_dispatch.experts import grouped_linear
from tests._helpers import gpu
from tests.test_gpu_training import U, _half, _within

pytestmark = gpu

HALF = _half(torch.bfloat16)


def _ids(pattern, tokens, adapters, g):
    if pattern == "none":
        return torch.full((tokens,), -1, device="cuda", dtype=torch.int32)
    if pattern == "one":
        return torch.full((tokens,), adapters - 1, device="cuda", dtype=torch.int32)
    ids = torch.randint(-1, adapters, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    if pattern == "runs":  # neighbouring rows of a request
        return ids.sort().values.flip(0).contiguous()
    if pattern == "outside" and tokens >= 4:
        ids[1], ids[2], ids[3] = adapters, -2**31, 2**31 - 1
    return ids


def _case(tokens, hidden, width, rank, adapters, pattern="mixed", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + tokens * 3 + rank)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).bfloat16()

    case = {"x": normal(tokens, hidden), "base": normal(tokens, width),
            "down": normal(adapters, rank, hidden, scale=hidden**-0.5), "up": normal(adapters, rank, width),
            "scales": torch.rand(adapters, device="cuda", generator=g) + 0.5, "grad": normal(tokens, width),
            "grad_x": normal(tokens, hidden), "ids": _ids(pattern, tokens, adapters, g)}
    case["groups"] = AdapterGroups(tokens, adapters)
    case["groups"].assign(case["ids"])
    return case


def _check_groups(case):
    tokens, adapters = case["groups"].tokens, case["groups"].adapters
    ids = case["ids"].long()
    key = torch.where((ids >= 0) & (ids < adapters), ids, adapters)
    order = case["groups"].order.long()
    assert torch.equal(order, torch.sort(key, stable=True).indices), "order"
    return key


def _reference(case, scaled=True):
    """64-bit results and tolerances, adapter by adapter."""
    x, base, down, up, dy, gx = (case[n].double() for n in ("x", "base", "down", "up", "grad", "grad_x"))
    scales = case["scales"].double() if scaled else torch.ones_like(case["scales"]).double()
    ids = case["ids"].long()
    hidden, width, rank = x.shape[1], up.shape[2], up.shape[1]
    y, ty = base.clone(), torch.zeros_like(base)
    dx, tx = gx.clone(), torch.zeros_like(gx)
    gd, td = torch.zeros_like(down), torch.zeros_like(down)
    gu, tu = torch.zeros_like(up), torch.zeros_like(up)
    for a in range(down.shape[0]):
        rows = torch.nonzero(ids == a).squeeze(1)
        if rows.numel() == 0:
            continue
        s = float(scales[a])

        def contract(v, w):
            h = v @ w.t()
            n = v.shape[1] / 4 + 100  # a wave's share of the products, then the waves and slices
            return h, (v.abs() @ w.abs().t()) * 2 * n * U

        def spread(h, th, w):
            size = h.abs() @ w.abs()
            return s * (h @ w), s * (th @ w.abs() + size * (2.0**-16 + 2 * (2 * rank + 16) * U))

        def outer(h, th, v):
            n = 3 * min(rows.numel(), 1024) + rows.numel() / 128 + 20
            size = h.abs().t() @ v.abs()
            return s * (h.t() @ v), s * (th.t() @ v.abs() + size * 2 * n * U)

        h, th = contract(x[rows], down[a])
        dh, tdh = contract(dy[rows], up[a])
        part, tol = spread(h, th, up[a])
        y[rows] += part
        ty[rows] = tol
        part, tol = spread(dh, tdh, down[a])
        dx[rows] += part
        tx[rows] = tol
        gd[a], td[a] = outer(dh, tdh, x[rows])
        gu[a], tu[a] = outer(h, th, dy[rows])
    ty += (y.abs() + base.abs()) * 2 * U
    tx += (dx.abs() + gx.abs()) * 2 * U
    return {"y": (y, ty), "dx": (dx, tx), "gd": (gd, td), "gu": (gu, tu)}


def _check(got, ref, what, half=HALF):
    want, tol = ref
    _within(got, want, tol * (1 + half) + want.abs() * half, what)


SHAPES = [
    # tokens, hidden, width, rank, adapters, ids
    (1, 8, 8, 1, 1, "one"), (1, 4096, 4096, 16, 8, "one"), (2, 64, 72, 4, 3, "mixed"), (5, 1000, 2744, 12, 4, "outside"),
    (48, 2048, 1408, 16, 64, "mixed"), (63, 256, 512, 8, 1, "one"), (64, 264, 520, 17, 2, "runs"),
    (65, 256, 136, 32, 3, "mixed"), (129, 512, 1024, 33, 2, "runs"), (200, 520, 264, 64, 5, "mixed"),
    (300, 128, 640, 65, 3, "runs"), (333, 1000, 2744, 128, 4, "mixed"), (777, 1000, 2744, 12, 12, "runs"),
    (130, 64, 64, 16, 4096, "mixed"), (90, 64, 64, 8, 3, "none"), (4096, 64, 128, 16, 7, "mixed"),
    (4097, 64, 128, 16, 7, "runs"), (5000, 72, 64, 24, 300, "outside"), (20000, 64, 64, 8, 3, "mixed"),
    (300, 8, 16384, 16, 2, "mixed"), (40, 14336, 8, 16, 2, "mixed")]


@pytest.mark.parametrize("tokens,hidden,width,rank,adapters,pattern", SHAPES)
def test_forward_and_gradients(tokens, hidden, width, rank, adapters, pattern):
    case = _case(tokens, hidden, width, rank, adapters, pattern)
    _check_groups(case)
    ref = _reference(case)
    operands = (case["x"], case["down"], case["up"], case["groups"])
    y, kept = low_rank_add(case["base"], *operands, scales=case["scales"], return_hidden=True)
    _check(y, ref["y"], "y")
    dx, gd, gu = low_rank_backward(case["grad"], *operands, scales=case["scales"], hidden=kept, grad_x=case["grad_x"])
    _check(dx, ref["dx"], "grad_x")
    _check(gd, ref["gd"], "grad_down", U)
    _check(gu, ref["gu"], "grad_up", U)
    dx16, gd16, gu16 = low_rank_backward(case["grad"], *operands, scales=case["scales"], hidden=kept,
                                         grad_x=case["grad_x"], grad_dtype=torch.bfloat16)
    assert torch.equal(dx16, dx) and torch.equal(gd16, gd.bfloat16()) and torch.equal(gu16, gu.bfloat16())
    for wanted in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        some = low_rank_backward(case["grad"], *operands, scales=case["scales"], hidden=kept, grad_x=case["grad_x"],
                                 gradients=wanted)
        for got, full, want in zip(some, (dx, gd, gu), wanted):
            assert (got is None) if not want else torch.equal(got, full)
    plain = (case["ids"] < 0) | (case["ids"] >= adapters)
    assert torch.equal(y[plain], case["base"][plain]) and torch.equal(dx[plain], case["grad_x"][plain])


@pytest.mark.parametrize("rank", [7, 32, 33, 128])
def test_batches_whose_base_is_streamed(rank):
    """Past 24 M elements of base; every rank's variant of spread."""
    test_forward_and_gradients(3100, 4104, 8192, rank, 3, "runs")


@pytest.mark.parametrize("tokens,adapters,pattern", [
    (1000, 4096, "mixed"), (4096, 4096, "outside"), (4096, 1535, "mixed"), (4096, 1536, "runs"), (4095, 1, "mixed"),
    (4097, 4096, "mixed"), (8192, 1536, "outside"), (8193, 2, "one"), (12289, 1535, "runs"), (70000, 4096, "mixed"),
    (70000, 1, "none")])
def test_many_adapters_and_rows(tokens, adapters, pattern):
    """Both sides of where a batch is sorted in chunks, and by four waves instead of sixteen."""
    case = _case(tokens, 8, 8, 2, adapters, pattern)
    key = _check_groups(case)
    groups = case["groups"]
    y, kept = low_rank_add(case["base"], case["x"], case["down"], case["up"], groups, return_hidden=True)
    got = low_rank_backward(case["grad"], case["x"], case["down"], case["up"], groups, hidden=kept)
    # Every row of one adapter at a time would take a launch each; here each row's own factors.
    safe = key.clamp(max=adapters - 1)
    on = (key < adapters).double().unsqueeze(1)
    x, dy = case["x"].double(), case["grad"].double()
    down, up = case["down"].double()[safe], case["up"].double()[safe]
    middle = 2 * (8 / 4 + 100) * U  # of the first product, as in _reference

    def through(base, v, first, second):
        h = (first * v.unsqueeze(1)).sum(2) * on
        th = (first.abs() * v.abs().unsqueeze(1)).sum(2) * on * middle
        want = base + (second * h.unsqueeze(2)).sum(1)
        size = (second.abs() * h.abs().unsqueeze(2)).sum(1)
        tol = (second.abs() * th.unsqueeze(2)).sum(1) + size * (2.0**-16 + 2 * (2 * 2 + 16) * U)
        return h, th, (want, tol + (want.abs() + base.abs()) * 2 * U)

    h, th, ref = through(case["base"].double(), x, down, up)
    _check(y, ref, "output")
    dh, tdh, ref = through(torch.zeros_like(x), dy, up, down)
    _check(got[0], ref, "grad_x")
    for g, a, ta, b in ((got[1], dh, tdh, x), (got[2], h, th, dy)):
        want, size, tol = (torch.zeros(adapters + 1, 2, 8, device="cuda", dtype=torch.float64).index_add_(
            0, key, m.unsqueeze(2) * v.unsqueeze(1)) for m, v in ((a, b), (a.abs(), b.abs()), (ta, b.abs())))
        rows = torch.bincount(key, minlength=adapters + 1)[:-1].reshape(-1, 1, 1)
        n = 3 * rows.clamp(max=1024) + rows / 128 + 20
        _check(g, (want[:-1], tol[:-1] + size[:-1] * 2 * n * U), "adapter gradient", half=0.0)


def test_without_base_and_scales_and_in_place():
    case = _case(150, 136, 264, 16, 3)
    ref = _reference(case, scaled=False)
    operands = (case["x"], case["down"], case["up"], case["groups"])
    y = low_rank_add(case["base"], *operands)
    _check(y, ref["y"], "y")
    buffer = case["base"].clone()
    assert low_rank_add(buffer, *operands, output=buffer) is buffer and torch.equal(buffer, y)
    zero = torch.zeros_like(case["base"])
    want = low_rank_add(zero, *operands)
    out = torch.full_like(zero, float("nan"))
    assert torch.equal(low_rank_add(None, *operands, output=out), want)
    _, kept = low_rank_add(None, *operands, return_hidden=True)
    dx, _, _ = low_rank_backward(case["grad"], *operands, hidden=kept)
    ref["dx"] = (ref["dx"][0] - case["grad_x"].double(), ref["dx"][1])
    _check(dx, ref["dx"], "grad_x")


def test_no_rows():
    case = _case(0, 64, 128, 8, 3, "none")
    y, kept = low_rank_add(case["base"], case["x"], case["down"], case["up"], case["groups"], return_hidden=True)
    assert y.shape == (0, 128)
    dx, gd, gu = low_rank_backward(case["grad"], case["x"], case["down"], case["up"], case["groups"], hidden=kept)
    assert dx.shape == (0, 64) and not gd.any() and not gu.any()


def test_each_row_and_adapter_stands_alone():
    """NaN in one row, and in one adapter, reaches only the results that depend on it."""
    case = _case(100, 128, 256, 16, 4, "mixed")
    operands = (case["down"], case["up"], case["groups"])
    clean = low_rank_add(case["base"], case["x"], *operands, scales=case["scales"])
    x = case["x"].clone()
    x[17] = float("nan")
    got = low_rank_add(case["base"], x, *operands, scales=case["scales"])
    rows = torch.arange(100, device="cuda") != 17
    assert torch.equal(got[rows], clean[rows])
    down = case["down"].clone()
    down[2] = float("nan")
    got = low_rank_add(case["base"], case["x"], down, *operands[1:], scales=case["scales"])
    rows = case["ids"] != 2
    assert torch.equal(got[rows], clean[rows]) and got[~rows].isnan().all()
    # The rank's last row only reaches through its own ranks: a finite adapter beside a NaN one.
    up = case["up"].clone()
    up[0] = float("inf")
    got = low_rank_add(case["base"], case["x"], case["down"], up, case["groups"], scales=case["scales"])
    rows = case["ids"] != 0
    assert torch.equal(got[rows], clean[rows])
    y, kept = low_rank_add(case["base"], x, *operands, scales=case["scales"], return_hidden=True)
    grad = case["grad"]
    want = low_rank_backward(grad, case["x"], *operands, scales=case["scales"],
                             hidden=low_rank_add(case["base"], case["x"], *operands, return_hidden=True)[1])
    got = low_rank_backward(grad, x, *operands, scales=case["scales"], hidden=kept)
    own = int(case["ids"][17])
    others = [a for a in range(4) if a != own]
    assert torch.equal(got[0], want[0])
    assert torch.equal(got[1][others], want[1][others]) and torch.equal(got[2][others], want[2][others])


def test_rows_behind_a_batch_stay_as_they_were():
    """A batch's rows are the head of a larger buffer: nothing behind them is written."""
    case = _case(77, 64, 520, 16, 3)
    store = torch.full((77 * 520 + 4096,), 7.0, device="cuda", dtype=torch.bfloat16)
    out = store[:77 * 520].view(77, 520)
    low_rank_add(case["base"], case["x"], case["down"], case["up"], case["groups"], output=out)
    assert bool((store[77 * 520:] == 7.0).all())


def test_groups_serve_several_projections_and_new_batches():
    case = _case(200, 128, 256, 16, 4)
    wide = _case(200, 256, 64, 8, 4)
    groups = case["groups"]
    first = low_rank_add(wide["base"], wide["x"], wide["down"], wide["up"], groups)
    own = AdapterGroups(200, 4)
    own.assign(case["ids"])
    assert torch.equal(first, low_rank_add(wide["base"], wide["x"], wide["down"], wide["up"], own))
    _, kept = low_rank_add(case["base"], case["x"], case["down"], case["up"], groups, return_hidden=True)
    groups.assign(wide["ids"])
    with pytest.raises(RuntimeError, match="another assignment"):
        low_rank_backward(case["grad"], case["x"], case["down"], case["up"], groups, hidden=kept)
    own.assign(wide["ids"])
    assert torch.equal(low_rank_add(case["base"], case["x"], case["down"], case["up"], groups),
                       low_rank_add(case["base"], case["x"], case["down"], case["up"], own))


@pytest.mark.parametrize("tokens,adapters", [(333, 5), (5000, 5)])
def test_same_every_time_on_streams_and_under_replay(tokens, adapters):
    case = _case(tokens, 256, 520, 24, adapters, "mixed")
    groups = case["groups"]

    def run():
        groups.assign(case["ids"])
        operands = (case["x"], case["down"], case["up"], groups)
        y, kept = low_rank_add(case["base"], *operands, scales=case["scales"], return_hidden=True)
        return (y, kept.values) + low_rank_backward(case["grad"], *operands, scales=case["scales"], hidden=kept,
                                                    grad_x=case["grad_x"])

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
        if round_ == 1:
            case["ids"].copy_(case["ids"].flip(0).contiguous())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want if round_ == 0 else run()):
            assert torch.equal(a, b), round_


def test_two_streams_share_the_groups():
    """Calls that only read the groups may run at once: their sums are their own."""
    case = _case(2000, 512, 1024, 16, 5)
    operands = (case["x"], case["down"], case["up"], case["groups"])
    want, kept = low_rank_add(case["base"], *operands, return_hidden=True)
    grads = low_rank_backward(case["grad"], *operands, hidden=kept)
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                y, h = low_rank_add(case["base"], *operands, return_hidden=True)
                results.append((y,) + low_rank_backward(case["grad"], *operands, hidden=h))
    for stream in streams:
        torch.cuda.current_stream().wait_stream(stream)
    for result in results:
        for a, b in zip(result, (want,) + grads):
            assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,hidden,width,rank", [(40, 4096, 1000, 16), (40, 2056, 1000, 32), (300, 2048, 2048, 32),
                                                      (16, 4104, 256, 16), (600, 64, 64, 33)])
def test_where_one_launch_ends(tokens, hidden, width, rank):
    """Sizes on either side of the rule that fuses the two products."""
    case = _case(tokens, hidden, width, rank, 3, "runs")
    ref = _reference(case)
    operands = (case["x"], case["down"], case["up"], case["groups"])
    y, kept = low_rank_add(case["base"], *operands, scales=case["scales"], return_hidden=True)
    _check(y, ref["y"], "y")
    dx, gd, gu = low_rank_backward(case["grad"], *operands, scales=case["scales"], hidden=kept, grad_x=case["grad_x"])
    _check(dx, ref["dx"], "grad_x")
    _check(gd, ref["gd"], "grad_down", U)
    _check(gu, ref["gu"], "grad_up", U)


def test_gradients_against_differences():
    """The 64-bit forward in random directions of x, down and up."""
    case = _case(60, 64, 72, 8, 3)
    operands = (case["x"], case["down"], case["up"], case["groups"])
    _, kept = low_rank_add(case["base"], *operands, scales=case["scales"], return_hidden=True)
    grads = low_rank_backward(case["grad"], *operands, scales=case["scales"], hidden=kept)
    ref = _reference(case)
    tols = [ref["dx"][1] + HALF * (ref["dx"][0] - case["grad_x"].double()).abs(), ref["gd"][1], ref["gu"][1]]
    ids = case["ids"].long()

    def total(x, down, up):
        out = torch.zeros((), device="cuda", dtype=torch.float64)
        for a in range(3):
            rows = ids == a
            out = out + float(case["scales"][a]) * ((x[rows] @ down[a].t()) @ up[a] * case["grad"][rows].double()).sum()
        return out

    point = [case[n].double() for n in ("x", "down", "up")]
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(3):
        d = torch.randn(point[i].shape, device="cuda", generator=g, dtype=torch.float64)
        plus, minus = list(point), list(point)
        plus[i], minus[i] = point[i] + d, point[i] - d  # linear in each: exact up to 64 bits
        slope = float(total(*plus) - total(*minus)) / 2
        got = float((grads[i].double() * d).sum())
        assert abs(got - slope) <= float((tols[i] * d.abs()).sum()) + 1e-9 * abs(slope)


def test_rows_past_two_to_the_31_elements():
    """Row offsets past 2^31 elements: 70000 rows of 32768 columns."""
    tokens, width, hidden, rank = 70000, 32768, 8, 4
    g = torch.Generator(device="cuda").manual_seed(5)
    base = torch.empty(tokens, width, device="cuda", dtype=torch.bfloat16)
    base.fill_(0.5)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16()
    down = torch.randn(2, rank, hidden, device="cuda", generator=g).bfloat16()
    up = torch.randn(2, rank, width, device="cuda", generator=g).bfloat16()
    ids = torch.randint(0, 2, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    groups = AdapterGroups(tokens, 2)
    groups.assign(ids)
    y, kept = low_rank_add(base, x, down, up, groups, return_hidden=True)
    for row in (0, 65535, 65536, tokens - 1):
        a = int(ids[row])
        h = x[row].double() @ down[a].double().t()
        want = 0.5 + h @ up[a].double()
        size = (x[row].double().abs() @ down[a].double().abs().t()) @ up[a].double().abs()
        _within(y[row], want, HALF * want.abs() + size * (2.0**-16 + 400 * U), f"row {row}")
    # The wide rows read back: dh from base's buffer, and the outer product over them.
    dx, gd, gu = low_rank_backward(y, x, down, up, groups, hidden=kept)
    row = tokens - 1
    a = int(ids[row])
    dh = y[row].double() @ up[a].double().t()
    want = dh @ down[a].double()
    size = (y[row].double().abs() @ up[a].double().abs().t()) @ down[a].double().abs()
    _within(dx[row], want, HALF * want.abs() + size * (2.0**-16 + 2 * (width / 4 + 100) * U), "grad_x")


def test_expert_adapters_beside_the_grouped_projection():
    """Rows packed by expert: frozen grouped weights (grouped_linear) with an adapter per
    expert, one step forward and backward against 64 bits."""
    tokens, hidden, width, experts, topk, rank = 120, 128, 256, 6, 2, 8
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16()
    ids = torch.randint(0, experts, (tokens, topk), device="cuda", generator=g, dtype=torch.int32)
    ws = CudaWorkspace(tokens, hidden, experts, topk, torch.bfloat16, alignment=8)
    ws.packed.zero_()
    ws.dispatch(x, ids)
    rows = ws.capacity_rows
    owner = torch.full((rows,), -1, device="cuda", dtype=torch.int32)
    owner[ws.inverse.reshape(-1).long()] = ids.reshape(-1)
    weight = (torch.randn(experts, width, hidden, device="cuda", generator=g) * hidden**-0.5).bfloat16()
    case = _case(rows, hidden, width, rank, experts, seed=2)
    case["x"], case["ids"] = ws.packed, owner
    case["base"] = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    grouped_linear(ws.packed, weight, ws.offsets[1:], backend="hip", output=case["base"], offsets=ws.offsets)
    case["groups"].assign(owner)
    ref = _reference(case)
    operands = (case["x"], case["down"], case["up"], case["groups"])
    y, kept = low_rank_add(case["base"], *operands, scales=case["scales"], return_hidden=True)
    _check(y, ref["y"], "y")
    dx, gd, gu = low_rank_backward(case["grad"], *operands, scales=case["scales"], hidden=kept, grad_x=case["grad_x"])
    for got, name, half in ((dx, "dx", HALF), (gd, "gd", U), (gu, "gu", U)):
        _check(got, ref[name], name, half)
