"""Performance cases of the training and adapter operators, over their real range of sizes.

A case is a dict of plain values. ``prepare`` builds what a program holds before the
call, ``run`` makes one pass through an operator and returns its whole outputs: with
``own`` true through the public entry points, otherwise in elementary torch operations
in 32 bits. ``exact`` evaluates the same inputs in 64 bits from the definitions.

Kinds:

* ``loss``: the router's auxiliary losses (balance and z), per-expert counts and the
  gradient of the logits, for a program whose logits come from elsewhere.
* ``route``: one training pass of the router behind its forward: the losses, then the
  gradients of logits, x, router weight and bias from the losses and the routing weights.
* ``combine``: the gradients of the weighted combine (expert rows and routing weights)
  and of the dispatch (x).
* ``adapter``: low-rank adapters of many requests beside a shared projection, forward.
* ``adapter_train``: one training pass of them, forward and all gradients.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PACKAGE = str(Path.cwd() / "cuda-moe-engine_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# A request in this many asks for the base model: its rows take no adapter (id -1).
_PLAIN_REQUESTS = 8


def _loss(name, tokens, experts, topk, padded):
    return {"name": name, "kind": "loss", "tokens": tokens, "experts": experts, "topk": topk, "padded": padded}


def _route(name, tokens, hidden, experts, topk, padded):
    return {"name": name, "kind": "route", "tokens": tokens, "hidden": hidden, "experts": experts, "topk": topk,
            "padded": padded}


def _combine(name, tokens, hidden, experts, topk, dtype):
    return {"name": name, "kind": "combine", "tokens": tokens, "hidden": hidden, "experts": experts, "topk": topk,
            "dtype": dtype}


def _adapter(name, tokens, hidden, width, rank, adapters, requests, assign=False, train=False):
    return {"name": name, "kind": "adapter_train" if train else "adapter", "tokens": tokens, "hidden": hidden,
            "width": width, "rank": rank, "adapters": adapters, "requests": requests, "assign": assign}


def listed():
    return [
        # The losses and their gradient for a small batch (latency), and for a
        # fine-grained layer's training batch whose last rows are padding.
        _loss("loss_128", 128, 8, 2, False),
        _loss("loss_fine_8192", 8192, 64, 6, True),
        # A training step of the router: eight large experts, and 64 small ones with a
        # padded batch.
        _route("route_4096", 4096, 4096, 8, 2, False),
        _route("route_fine_8192", 8192, 2048, 64, 6, True),
        # Gradients through the transport around a program's own experts: bf16 rows of
        # a training batch, and float32 rows of an odd width.
        _combine("combine_4096", 4096, 2048, 8, 2, "bf16"),
        _combine("combine_odd_2048", 2048, 1023, 16, 2, "fp32"),
        # Decoding: one request, and 48 requests over a bank of 64 adapters beside a
        # wide projection. The step's grouping of rows is in hand (each of a model's
        # projections uses it).
        _adapter("adapter_decode_1", 1, 4096, 4096, 16, 8, 1),
        _adapter("adapter_decode_48", 48, 4096, 14336, 16, 64, 48),
        # Prefill: a batch of prompts with adapters of a large rank; and short prompts,
        # an odd batch, widths that are multiples of 8 only, a rank that fills no tile,
        # with the rows grouped in the pass.
        _adapter("adapter_prefill_4096", 4096, 4096, 4096, 64, 8, 6),
        _adapter("adapter_ragged_777", 777, 1000, 2744, 12, 12, 30, assign=True),
        # Fine-tuning: several tenants' adapters in one batch, and an odd small batch
        # with the rows grouped in the pass.
        _adapter("adapter_train_4096", 4096, 4096, 4096, 16, 4, 8, train=True),
        _adapter("adapter_train_ragged_333", 333, 1000, 2744, 12, 5, 11, assign=True, train=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {unit: max(work(case)[unit] for case in listed()) for unit in ("bytes", "flops")}
    kind = rng.choice(("loss", "route", "combine", "adapter", "adapter", "adapter_train"))
    experts = rng.choice((4, 6, 8, 8, 12, 16, 24, 32, 48, 64))
    topk = min(rng.choice((1, 2, 2, 3, 4, 6, 8)), experts)
    unit = rng.choice((128, 64, 8))
    hidden = max(_log_int(rng, 256, 8192) // unit, 1) * unit
    tokens = _log_int(rng, 1, 16384)
    if kind == "loss":
        case = _loss("", tokens, experts, topk, rng.random() < 0.5)
    elif kind == "route":
        case = _route("", tokens, hidden, experts, topk, rng.random() < 0.5)
    elif kind == "combine":
        if rng.random() < 0.25:
            hidden = _log_int(rng, 64, 4096)
        case = _combine("", tokens, hidden, experts, topk, rng.choice(("bf16", "bf16", "fp16", "fp32")))
    else:
        width = max(_log_int(rng, 256, 14336) // unit, 1) * unit
        rank = rng.choice((4, 8, 8, 16, 16, 24, 32, 64, 128))
        train = kind == "adapter_train"
        # Decoding: a request a row. Otherwise prompts, or a training batch of few tenants.
        decode = not train and rng.random() < 0.5
        adapters = _log_int(rng, 1, 8 if train else 128)
        tokens = _log_int(rng, 1, 256) if decode else tokens
        requests = tokens if decode else min(_log_int(rng, 1, 64), tokens)
        case = _adapter("", tokens, hidden, width, rank, adapters, requests, rng.random() < 0.3, train)
    while case["tokens"] > 1 and any(work(case)[unit] > most[unit] for unit in most):
        case["tokens"] = max(case["tokens"] * 3 // 4, 1)
        if "requests" in case:
            case["requests"] = min(case["requests"], case["tokens"])
    del case["name"]
    return case


# -- inputs ------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g).mul_(scale).to(dtype)


def _router_inputs(case, seed):
    g = _generator(seed)
    t, e, k = case["tokens"], case["experts"], case["topk"]
    data = {"logits": _normal(g, (t, e)), "bias": _normal(g, (e,), 0.5)}
    data["ids"] = torch.topk(data["logits"] + data["bias"], k, dim=-1).indices.to(torch.int32).contiguous()
    # What the two losses weigh in the training loss.
    data["grad_losses"] = torch.tensor([1e-2, 1e-3], device="cuda")
    data["mask"] = None
    if case["padded"]:
        # The last rows are padding: up to an eighth of the batch, by the seed.
        valid = t - int(torch.randint(0, t // 8 + 1, (1,), device="cuda", generator=g))
        data["mask"] = torch.arange(t, device="cuda") < valid
    if case["kind"] == "route":
        h = case["hidden"]
        data["x"] = _normal(g, (t, h), 1.0, torch.bfloat16)
        data["router_weight"] = _normal(g, (e, h), 1 / math.sqrt(h))
        data["grad_weights"] = _normal(g, (t, k), 1e-3)
        # x's gradient along its other paths (the experts).
        data["grad_x"] = _normal(g, (t, h), 1e-3, torch.bfloat16)
    return data


def _combine_inputs(case, seed):
    g = _generator(seed)
    t, h, e, k = case["tokens"], case["hidden"], case["experts"], case["topk"]
    dtype = _DTYPES[case["dtype"]]
    values, ids = torch.topk(_normal(g, (t, e)), k, dim=-1)
    return {"x": _normal(g, (t, h), 1.0, dtype), "ids": ids.to(torch.int32).contiguous(),
            "weights": torch.softmax(values, dim=-1).contiguous(), "expert_output": _normal(g, (t * k, h), 1.0, dtype),
            "grad_output": _normal(g, (t, h), 1e-2, dtype), "grad_packed": _normal(g, (t * k, h), 1e-2, dtype)}


def _request_rows(case, seed):
    """(first row, rows, adapter) of each request: contiguous rows, adapter -1 for the base model."""
    g = torch.Generator().manual_seed(seed)
    n, t = case["requests"], case["tokens"]
    share = torch.rand(n, generator=g, dtype=torch.float64) + 0.1
    ends = [min(max(int(round(c)), i + 1), t - (n - 1 - i))
            for i, c in enumerate((share.cumsum(0) / share.sum() * t).tolist())]
    ends[-1] = t
    adapters = torch.randint(0, case["adapters"], (n,), generator=g).tolist()
    plain = torch.randint(0, _PLAIN_REQUESTS, (n,), generator=g).tolist()
    if n == 1:
        plain = [1]
    out, start = [], 0
    for end, adapter, choice in zip(ends, adapters, plain):
        if end > start:
            out.append((start, end - start, -1 if choice == 0 else adapter))
        start = max(start, end)
    return out


def _adapter_inputs(case, seed):
    g = _generator(seed)
    t, h, o, r, n = (case[name] for name in ("tokens", "hidden", "width", "rank", "adapters"))
    bf16 = torch.bfloat16
    requests = _request_rows(case, seed)
    ids = torch.empty(t, dtype=torch.int32)
    for start, rows, adapter in requests:
        ids[start:start + rows] = adapter
    data = {"requests": requests, "ids": ids.cuda(), "x": _normal(g, (t, h), 1.0, bf16),
            "base": _normal(g, (t, o), 1.0, bf16), "down": _normal(g, (n, r, h), 1 / math.sqrt(h), bf16),
            "up": _normal(g, (n, r, o), 1 / math.sqrt(r), bf16),
            "scales": torch.rand(n, device="cuda", generator=g) + 0.5}
    if case["kind"] == "adapter_train":
        data["grad_output"] = _normal(g, (t, o), 1e-2, bf16)
        # x's gradient through the shared projection.
        data["grad_x"] = _normal(g, (t, h), 1e-2, bf16)
    return data


def prepare(case, seed):
    kind = case["kind"]
    state = {"kind": kind, "case": case}
    if kind in ("loss", "route"):
        state.update(_router_inputs(case, seed))
        return state
    if kind == "combine":
        state.update(_combine_inputs(case, seed))
        if own:
            from moe_dispatch import dispatch

            state["batch"] = dispatch(state["x"], state["ids"], case["experts"])
        else:
            # Row of each assignment: experts in order, each one's assignments in flat order.
            flat = state["ids"].reshape(-1).long()
            inverse = torch.empty_like(flat)
            inverse[torch.argsort(flat, stable=True)] = torch.arange(flat.numel(), device="cuda")
            state["inverse"] = inverse.view(state["ids"].shape)
        return state
    state.update(_adapter_inputs(case, seed))
    if own:
        from moe_dispatch import AdapterGroups

        state["groups"] = AdapterGroups(case["tokens"], case["adapters"], device=state["x"].device)
        state["groups"].assign(state["ids"])
    return state


# -- plain forms -------------------------------------------------------------
def _softmax_parts(logits, bias):
    v = logits + bias
    top = v.max(dim=-1, keepdim=True).values
    e = torch.exp(v - top)
    total = e.sum(dim=-1, keepdim=True)
    return v, e / total, (top + torch.log(total)).squeeze(-1)


def _plain_loss(s):
    t, e = s["logits"].shape
    k = s["ids"].shape[1]
    v, p, lse = _softmax_parts(s["logits"], s["bias"])
    hits = (s["ids"].unsqueeze(-1) == torch.arange(e, device="cuda", dtype=torch.int32)).sum(dim=1)
    tokens = torch.tensor(float(t), device="cuda")
    if s["mask"] is not None:
        valid = s["mask"].float()
        tokens = valid.sum()
        p, lse, hits = p * valid.unsqueeze(-1), lse * valid, hits * s["mask"].unsqueeze(-1)
    counts = hits.sum(dim=0)
    some = torch.clamp(tokens, min=1.0)
    c = counts.float()
    balance = e * ((c / (some * k)) * (p.sum(dim=0) / some)).sum()
    z = (lse * lse).sum() / some
    grad = p * (c - (p * c).sum(dim=-1, keepdim=True)) * (s["grad_losses"][0] * e / (some * some * k))
    grad = grad + p * lse.unsqueeze(-1) * (s["grad_losses"][1] * 2 / some)
    if "grad_weights" in s:
        ids = s["ids"].long()
        chosen = v.gather(1, ids)
        w = torch.exp(chosen - chosen.max(dim=-1, keepdim=True).values)
        w = w / w.sum(dim=-1, keepdim=True)
        dw = s["grad_weights"]
        grad.scatter_add_(1, ids, w * (dw - (w * dw).sum(dim=-1, keepdim=True)))
        if s["mask"] is not None:
            grad = grad * valid.unsqueeze(-1)
    return {"losses": torch.stack([balance, z]), "counts": counts.to(torch.int32), "grad_logits": grad}


def _plain_route(s):
    out = _plain_loss(s)
    grad = out.pop("grad_logits")
    out["grad_x"] = (s["grad_x"].float() + grad @ s["router_weight"]).to(torch.bfloat16)
    out["grad_router_weight"] = grad.t() @ s["x"].float()
    out["grad_bias"] = grad.sum(dim=0)
    return out


def _plain_combine(s):
    dtype = s["grad_output"].dtype
    t, k = s["ids"].shape
    dout = s["grad_output"].float().unsqueeze(1)
    rows = s["expert_output"][s["inverse"].reshape(-1)].float().view(t, k, -1)
    grad_expert = torch.empty_like(s["expert_output"])
    grad_expert[s["inverse"].reshape(-1)] = (dout * s["weights"].unsqueeze(-1)).to(dtype).view(t * k, -1)
    back = s["grad_packed"][s["inverse"].reshape(-1)].float().view(t, k, -1)
    return {"grad_expert": grad_expert, "grad_weights": (dout * rows).sum(dim=-1), "grad_x": back.sum(dim=1).to(dtype)}


def _plain_adapter(s):
    case = s["case"]
    x, base = s["x"].float(), s["base"].float()
    if case["requests"] == case["tokens"]:
        # A request a row: every row's own adapter, gathered.
        some = s["ids"].clamp(min=0).long()
        scale = torch.where(s["ids"] >= 0, s["scales"][some], 0.0)
        h = (s["down"][some].float() * x.unsqueeze(1)).sum(dim=-1)
        return {"y": (base + (h.unsqueeze(-1) * s["up"][some].float()).sum(dim=1) * scale.unsqueeze(-1)
                      ).to(torch.bfloat16)}
    y = base
    for start, rows, a in s["requests"]:
        if a >= 0:
            part = slice(start, start + rows)
            h = x[part] @ s["down"][a].float().t()
            y[part] += (h @ s["up"][a].float()) * s["scales"][a]
    return {"y": y.to(torch.bfloat16)}


def _plain_adapter_train(s):
    x, y, dx, dy = s["x"].float(), s["base"].float(), s["grad_x"].float(), s["grad_output"].float()
    grad_down = torch.zeros(s["down"].shape, device="cuda")
    grad_up = torch.zeros(s["up"].shape, device="cuda")
    for start, rows, a in s["requests"]:
        if a >= 0:
            part = slice(start, start + rows)
            down, up = s["down"][a].float(), s["up"][a].float()
            h = (x[part] @ down.t()) * s["scales"][a]
            y[part] += h @ up
            dh = (dy[part] @ up.t()) * s["scales"][a]
            dx[part] += dh @ down
            grad_down[a] += dh.t() @ x[part]
            grad_up[a] += h.t() @ dy[part]
    return {"y": y.to(torch.bfloat16), "grad_x": dx.to(torch.bfloat16), "grad_down": grad_down, "grad_up": grad_up}


_PLAIN = {"loss": _plain_loss, "route": _plain_route, "combine": _plain_combine, "adapter": _plain_adapter,
          "adapter_train": _plain_adapter_train}


# -- the framework's operators -----------------------------------------------
def _own_loss(s):
    from moe_dispatch import route_logits_backward, router_loss

    loss = router_loss(s["logits"], s["ids"], s["bias"], mask=s["mask"])
    grad_logits = route_logits_backward(s["logits"], s["ids"], s["bias"], mask=s["mask"], loss=loss,
                                        grad_losses=s["grad_losses"])
    return {"losses": loss.losses, "counts": loss.counts, "grad_logits": grad_logits}


def _own_route(s):
    from moe_dispatch import route_backward, router_loss

    loss = router_loss(s["logits"], s["ids"], s["bias"], mask=s["mask"])
    grad_x, grad_router_weight, grad_bias = route_backward(
        s["x"], s["router_weight"], s["logits"], s["ids"], s["bias"], mask=s["mask"], loss=loss,
        grad_losses=s["grad_losses"], grad_weights=s["grad_weights"], grad_x=s["grad_x"])
    return {"losses": loss.losses, "counts": loss.counts, "grad_x": grad_x, "grad_router_weight": grad_router_weight,
            "grad_bias": grad_bias}


def _own_combine(s):
    from moe_dispatch import combine_backward, dispatch_backward

    grad_expert, grad_weights = combine_backward(s["grad_output"], s["expert_output"], s["batch"], s["weights"])
    return {"grad_expert": grad_expert, "grad_weights": grad_weights,
            "grad_x": dispatch_backward(s["grad_packed"], s["batch"])}


def _own_adapter(s):
    from moe_dispatch import low_rank_add

    if s["case"]["assign"]:
        s["groups"].assign(s["ids"])
    return {"y": low_rank_add(s["base"], s["x"], s["down"], s["up"], s["groups"], scales=s["scales"])}


def _own_adapter_train(s):
    from moe_dispatch import low_rank_add, low_rank_backward

    if s["case"]["assign"]:
        s["groups"].assign(s["ids"])
    y, hidden = low_rank_add(s["base"], s["x"], s["down"], s["up"], s["groups"], scales=s["scales"],
                             return_hidden=True)
    grad_x, grad_down, grad_up = low_rank_backward(s["grad_output"], s["x"], s["down"], s["up"], s["groups"],
                                                   scales=s["scales"], hidden=hidden, grad_x=s["grad_x"])
    return {"y": y, "grad_x": grad_x, "grad_down": grad_down, "grad_up": grad_up}


_OWN = {"loss": _own_loss, "route": _own_route, "combine": _own_combine, "adapter": _own_adapter,
        "adapter_train": _own_adapter_train}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# -- work --------------------------------------------------------------------
def work(case):
    t = case["tokens"]
    if case["kind"] in ("loss", "route"):
        e, k = case["experts"], case["topk"]
        size = {"bytes": 4 * t * e + 4 * t * k + 8 * e + (t if case["padded"] else 0), "flops": 12 * t * e}
        if case["kind"] == "loss":
            size["bytes"] += 4 * t * e
        else:
            h = case["hidden"]
            # x, the gradient it joins and its own; the router weight and its gradient.
            size["bytes"] += 3 * 2 * t * h + 2 * 4 * e * h + 4 * t * k
            size["flops"] += 4 * t * e * h
        return size
    if case["kind"] == "combine":
        h, k = case["hidden"], case["topk"]
        row = h * torch.finfo(_DTYPES[case["dtype"]]).bits // 8
        # grad_output, grad_x; expert rows, their gradients and the packed rows' gradients.
        return {"bytes": 2 * t * row + 3 * t * k * row + 12 * t * k, "flops": 4 * t * k * h}
    h, o, r, n = (case[name] for name in ("hidden", "width", "rank", "adapters"))
    requests = case["requests"] * (1 - 1 / _PLAIN_REQUESTS) if case["requests"] > 1 else 1
    active = n * (1 - (1 - 1 / n) ** requests)
    size = {"bytes": 2 * t * (h + 2 * o) + 2 * active * r * (h + o) + 4 * t, "flops": 2 * t * r * (h + o)}
    if case["kind"] == "adapter_train":
        # The output's gradient, the gradient that x's joins and x's own; the adapters' gradients.
        size["bytes"] += 2 * t * (2 * h + o) + 4 * n * r * (h + o)
        size["flops"] *= 3
    return size


# -- exact -------------------------------------------------------------------
def _exact_router(case, seed):
    d = _router_inputs(case, seed)
    t, e, k = case["tokens"], case["experts"], case["topk"]
    ids = d["ids"].long()
    rows = torch.arange(t, device="cuda") if d["mask"] is None else torch.nonzero(d["mask"]).squeeze(1)
    n = rows.numel()
    counts = torch.bincount(ids[rows].reshape(-1), minlength=e)
    leaf = (d["logits"].double() + d["bias"].double()).requires_grad_()
    v = leaf[rows]
    if n:
        balance = e * torch.dot(counts.double() / (n * k), torch.softmax(v, dim=-1).mean(dim=0))
        z = torch.logsumexp(v, dim=-1).square().mean()
    else:
        balance = z = v.sum()
    out = {"losses": torch.stack([balance, z]).detach(), "counts": counts.to(torch.int32)}
    total = (d["grad_losses"].double() * torch.stack([balance, z])).sum()
    if case["kind"] == "loss":
        out["grad_logits"], = torch.autograd.grad(total, leaf)
        return out
    weights = torch.softmax(v.gather(1, ids[rows]), dim=-1)
    total = total + (weights * d["grad_weights"][rows].double()).sum()
    grad, = torch.autograd.grad(total, leaf)
    out["grad_x"] = d["grad_x"].double() + grad @ d["router_weight"].double()
    out["grad_router_weight"] = grad.t() @ d["x"].double()
    out["grad_bias"] = grad.sum(dim=0)
    return out


def _exact_combine(case, seed):
    d = _combine_inputs(case, seed)
    t, k = d["ids"].shape
    flat = d["ids"].reshape(-1)
    order = torch.sort(flat.long() * flat.numel() + torch.arange(flat.numel(), device="cuda")).indices
    token = order // k  # packed row -> token
    dout = d["grad_output"].double()
    grad_weights = torch.empty(t * k, device="cuda", dtype=torch.float64)
    grad_weights[order] = (dout[token] * d["expert_output"].double()).sum(dim=-1)
    grad_x = torch.zeros_like(dout).index_add_(0, token, d["grad_packed"].double())
    return {"grad_expert": dout[token] * d["weights"].double().reshape(-1)[order].unsqueeze(-1),
            "grad_weights": grad_weights.view(t, k), "grad_x": grad_x}


def _exact_adapter(case, seed):
    d = _adapter_inputs(case, seed)
    train = case["kind"] == "adapter_train"
    x, down, up = (d[name].double().requires_grad_(train) for name in ("x", "down", "up"))
    y = d["base"].double()
    parts = []
    for a in sorted(set(d["ids"].tolist()) - {-1}):
        rows = torch.nonzero(d["ids"] == a).squeeze(1)
        part = (x[rows] @ down[a].t()) @ up[a] * d["scales"][a].double()
        y = y.index_add(0, rows, part.detach())
        parts.append((part, rows))
    out = {"y": y}
    if train:
        grads = [torch.zeros_like(leaf) for leaf in (x, down, up)]
        if parts:
            dy = d["grad_output"].double()
            grads = torch.autograd.grad([part for part, _ in parts], [x, down, up], [dy[rows] for _, rows in parts])
        out.update(grad_x=d["grad_x"].double() + grads[0], grad_down=grads[1], grad_up=grads[2])
    return out


def exact(case, seed):
    if case["kind"] in ("loss", "route"):
        return _exact_router(case, seed)
    if case["kind"] == "combine":
        return _exact_combine(case, seed)
    return _exact_adapter(case, seed)
