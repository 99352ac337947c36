"""Refusals and argument structs of norm, scored routing, dense products and clipping, where no kernel can launch."""

import re
import struct

import pytest
import torch

from moe_dispatch import (QuantizedRows, _lib, clip_gradients, linear, quantize_rows, rms_norm, rms_norm_backward,
                          route_scored, route_scored_backward)
from tests.test_abi import HEADER, stand_in_addresses

BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn


def test_argument_structs_are_the_headers():
    """Each packer has its struct's fields, in order and kind, and writes the struct's size first."""
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for name, packer in (("rms_norm", _lib.RMS_NORM_ARGS), ("route_scored", _lib.ROUTE_SCORED_ARGS),
                         ("route_scored_backward", _lib.ROUTE_SCORED_BACKWARD_ARGS), ("linear", _lib.LINEAR_ARGS),
                         ("clip", _lib.CLIP_ARGS)):
        body = re.search(r"typedef struct moe_%s_args \{(.*?)\}" % name, text, flags=re.S).group(1)
        kinds = ["P" if "*" in d else "d" if "double" in d else "q" for d in body.split(";") if d.strip()]
        layout = struct.Struct("@" + "".join(kinds))
        packed = packer(*range(1, len(kinds)))
        assert len(packed) == layout.size == 8 * len(kinds)
        assert layout.unpack(packed) == (layout.size, *range(1, len(kinds))), name


def test_rms_norm_refuses_bad_tensors():
    x, w = torch.zeros(4, 64, dtype=BF16), torch.ones(64, dtype=BF16)
    with pytest.raises(TypeError, match="x must be"):
        rms_norm(x.double(), w)
    with pytest.raises(ValueError, match="contiguous"):
        rms_norm(torch.zeros(64, 4, dtype=BF16).t(), w)
    with pytest.raises(ValueError, match="2 dimensions"):
        rms_norm(torch.zeros(2, 4, 64, dtype=BF16), w)
    with pytest.raises(ValueError, match="weight"):
        rms_norm(x, w[:63])
    with pytest.raises(TypeError, match="weight"):
        rms_norm(x, w.half())
    with pytest.raises(TypeError, match="residual"):
        rms_norm(x, w, residual=x.float())
    with pytest.raises(ValueError, match="residual"):
        rms_norm(x, w, residual=x[:3])
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            rms_norm(x, w, eps=eps)
    with pytest.raises(ValueError, match="16384"):
        rms_norm(torch.zeros(1, 16385, dtype=BF16))
    for hidden in (0, 32769):
        with pytest.raises(ValueError, match="32768"):
            quantize_rows(torch.zeros(1, hidden, dtype=BF16))
    with pytest.raises(ValueError, match="2\\^21"):
        rms_norm(torch.zeros(2**21 + 1, 1, dtype=BF16))
    rstd = torch.ones(4)
    with pytest.raises(ValueError, match="rstd"):
        rms_norm_backward(x, x, w, rstd[:3])
    with pytest.raises(TypeError, match="grad_output"):
        rms_norm_backward(x.float(), x, w, rstd)
    with pytest.raises(ValueError, match="grad_x"):
        rms_norm_backward(x, x, w, rstd, grad_x=x[:2])


def test_route_scored_refuses_bad_arguments():
    logits = torch.zeros(4, 16)
    for arguments, match in ((dict(topk=0), "topk"), (dict(topk=9), "topk"), (dict(topk=2.0), "topk"),
                             (dict(topk=2, scoring="tanh"), "scoring"), (dict(topk=2, groups=3), "groups"),
                             (dict(topk=2, groups=0), "groups"), (dict(topk=2, groups=4, top_groups=5), "top_groups"),
                             (dict(topk=2, groups=4, top_groups=0), "top_groups"),
                             (dict(topk=5, groups=4, top_groups=1), "topk exceeds"),
                             (dict(topk=2, groups=4, group_best=3), "group_best"),
                             (dict(topk=2, bias=torch.zeros(15)), "bias")):
        with pytest.raises(ValueError, match=match):
            route_scored(logits, **arguments)
    with pytest.raises(TypeError, match="bias"):
        route_scored(logits, 2, bias=torch.zeros(16, dtype=BF16))
    with pytest.raises(TypeError, match="logits"):
        route_scored(logits.to(BF16), 2)
    with pytest.raises(ValueError, match="1..512"):
        route_scored(torch.zeros(1, 513), 2)
    with pytest.raises(ValueError, match="topk exceeds"):
        route_scored(torch.zeros(1, 2), 3)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="grad_weights"):
        route_scored_backward(torch.zeros(4, 3), logits, ids)
    with pytest.raises(TypeError, match="ids"):
        route_scored_backward(torch.zeros(4, 2), logits, ids.long())
    with pytest.raises(ValueError, match="ids"):
        route_scored_backward(torch.zeros(3, 2), logits, ids[:3])


def _eight(rows, k):
    return QuantizedRows(torch.zeros(rows, k, dtype=E4M3), torch.ones(rows))


def test_linear_refuses_bad_tensors():
    x, w = torch.zeros(4, 64, dtype=BF16), torch.zeros(32, 64, dtype=BF16)
    with pytest.raises(TypeError, match="x must be"):
        linear(x.float(), w)
    with pytest.raises(TypeError, match="weight must be"):
        linear(x, w.float())
    with pytest.raises(TypeError, match="both"):
        linear(x, _eight(32, 64))
    with pytest.raises(TypeError, match="both"):
        linear(_eight(4, 64), w)
    with pytest.raises(ValueError, match="rows of 64"):
        linear(x, w[:, :32].contiguous())
    with pytest.raises(ValueError, match="padding"):
        linear(x, torch.zeros(64, 32, dtype=BF16).t())
    with pytest.raises(ValueError, match="multiples of 8"):
        linear(x, torch.zeros(32, 68, dtype=BF16)[:, :64])
    with pytest.raises(ValueError, match="padding"):
        linear(x, torch.zeros(64, dtype=BF16).expand(32, 64))
    with pytest.raises(ValueError, match="multiples of 8"):
        linear(x[:, :12].contiguous(), w[:, :12].contiguous())
    with pytest.raises(ValueError, match="multiples of 16"):
        linear(_eight(4, 24), _eight(32, 24))
    with pytest.raises(ValueError, match="width"):
        linear(x, w[:12])
    with pytest.raises(ValueError, match="even"):
        linear(x, w[:31], activation="swiglu")
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="bias"):
        linear(x, w, torch.zeros(31))
    with pytest.raises(TypeError, match="bias"):
        linear(x, w, torch.zeros(32, dtype=torch.float16))
    with pytest.raises(ValueError, match="bias"):
        linear(x, w, torch.zeros(16), activation="swiglu")
    with pytest.raises(ValueError, match="residual"):
        linear(x, w, residual=torch.zeros(4, 31, dtype=BF16))
    with pytest.raises(TypeError, match="residual"):
        linear(x, w, residual=torch.zeros(4, 32))
    with pytest.raises(ValueError, match="scales"):
        linear(_eight(4, 64)._replace(scales=torch.ones(3)), _eight(32, 64))
    with pytest.raises(TypeError, match="x must be"):
        linear(QuantizedRows(x, torch.ones(4)), _eight(32, 64))
    with pytest.raises(ValueError, match="overlap"):
        linear(x, w, output=w.view(-1)[:128].view(4, 32))
    both = torch.zeros(8, 32, dtype=BF16)
    with pytest.raises(ValueError, match="overlap"):
        linear(x, w, residual=both[:4], output=both[2:6])


def test_clip_gradients_refuses_bad_lists():
    g = torch.zeros(8)
    with pytest.raises(ValueError, match="at least one"):
        clip_gradients([], 1.0)
    for most in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_gradients([g], most)
    with pytest.raises(TypeError, match=r"grads\[1\]"):
        clip_gradients([g, torch.zeros(4, dtype=torch.int32)], 1.0)
    with pytest.raises(TypeError, match=r"grads\[0\]"):
        clip_gradients([None], 1.0)
    with pytest.raises(ValueError, match="contiguous"):
        clip_gradients([torch.zeros(4, 4).t()], 1.0)
    # One gradient twice would be scaled twice, in an order that nobody knows.
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([g, g], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([g[:5], g[4:]], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([g[:4], g[4:]], 1.0, outputs=[torch.zeros(4), g[:4]])
    with pytest.raises(ValueError, match="for each"):
        clip_gradients([g], 1.0, outputs=[])
    with pytest.raises(ValueError, match="sizes and types"):
        clip_gradients([g], 1.0, outputs=[torch.zeros(9)])
    with pytest.raises(ValueError, match="sizes and types"):
        clip_gradients([g], 1.0, outputs=[torch.zeros(8, dtype=BF16)])


def test_operators_that_record_no_graph_say_so():
    if torch.cuda.is_available():
        pytest.skip("checks come before the GPU's presence here")
    x = torch.zeros(8, 64, dtype=BF16, requires_grad=True)
    for call in (lambda: rms_norm(x), lambda: linear(x, x), lambda: clip_gradients([x], 1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@stand_in_addresses
def test_entry_points_check_their_arguments_without_launching():
    lib = _lib.load_library()
    A = 1 << 20  # stand-in addresses, never dereferenced
    ok, invalid, unsupported, capacity, workspace = 0, 1, 2, 3, 4

    def norm(x=A, residual=0, weight=A, total=0, output=A, scales=0, rstd=0, tokens=4, hidden=64, dtype=2,
             weight_dtype=2, eps=1e-6):
        return lib.moe_rms_norm(_lib.RMS_NORM_ARGS(x, residual, weight, total, output, scales, rstd, tokens, hidden, dtype,
                                                   weight_dtype, eps), None)

    assert lib.moe_rms_norm(None, None) == invalid and lib.moe_rms_norm(struct.pack("q", 8), None) == invalid
    assert norm(tokens=0) == ok and norm(x=0) == invalid and norm(residual=A) == invalid and norm(x=A + 1) == invalid
    assert norm(dtype=3) == invalid and norm(weight_dtype=1) == invalid and norm(eps=-1.0) == invalid
    assert norm(eps=float("nan")) == invalid and norm(hidden=0) == unsupported and norm(hidden=16385) == unsupported
    assert norm(tokens=2**21 + 1) == capacity and norm(tokens=-1) == invalid and norm(scales=A + 2) == invalid
    assert lib.moe_quantize_rows(A, 2, A, None, 4, 64, None) == invalid
    assert lib.moe_quantize_rows(A, 2, A, A, 0, 64, None) == ok

    need = lib.moe_rms_norm_backward_scratch_bytes(100, 64, 2)
    assert need >= 64 * 4 and lib.moe_rms_norm_backward_scratch_bytes(100, 0, 2) == -1
    assert lib.moe_rms_norm_backward_scratch_bytes(100, 64, 3) == -1

    def grad(g=A, rstd=A, out=A, grad_weight=A, scratch=A, nbytes=need, tokens=100):
        return lib.moe_rms_norm_backward(g, A, 2, A, 2, rstd, None, out, grad_weight, scratch, nbytes, tokens, 64, None)

    assert grad(nbytes=need - 1) == workspace and grad(scratch=None) == workspace and grad(rstd=None) == invalid
    assert grad(tokens=0) == invalid and grad(g=None) == invalid and grad(out=A + 1) == invalid
    assert grad(out=None, grad_weight=None) == ok

    def route(logits=A, bias=0, ids=A, weights=A, tokens=4, experts=64, topk=6, groups=8, top_groups=4, best=2):
        return lib.moe_route_scored(_lib.ROUTE_SCORED_ARGS(logits, bias, ids, weights, tokens, experts, topk, groups,
                                                           top_groups, best, 1, 1, 1.0), None)

    assert route(tokens=0) == ok and route(ids=0) == invalid and route(weights=A + 2) == invalid
    assert route(experts=513) == unsupported and route(experts=0) == unsupported and route(topk=9) == unsupported
    assert route(groups=7) == unsupported and route(groups=0) == unsupported and route(groups=65, experts=65) == unsupported
    assert route(top_groups=9) == invalid and route(top_groups=0) == invalid and route(best=0) == invalid
    assert route(experts=16, top_groups=2) == invalid  # two groups of two hold four
    back = _lib.ROUTE_SCORED_BACKWARD_ARGS
    assert lib.moe_route_scored_backward(back(A, A, 0, A, 4, 64, 6, 1, 1, 1.0), None) == invalid
    assert lib.moe_route_scored_backward(back(A, A, A, A, 4, 64, 0, 1, 1, 1.0), None) == unsupported
    assert lib.moe_route_scored_backward(back(0, 0, 0, 0, 0, 64, 6, 1, 1, 1.0), None) == ok

    def dense(x=A, weight=A, xs=0, ws=0, bias=0, residual=0, output=A, scratch=A, nbytes=1 << 40, tokens=4, hidden=64,
              width=64, stride=64, bias_dtype=0, activation=0):
        return lib.moe_linear(_lib.LINEAR_ARGS(x, weight, xs, ws, bias, residual, output, scratch, nbytes, tokens, hidden,
                                               width, stride, bias_dtype, activation), None)

    assert dense(tokens=0) == ok and dense(x=A + 8) == invalid and dense(output=0) == invalid
    assert dense(xs=A) == invalid and dense(ws=A) == invalid  # both scales or neither
    assert dense(hidden=60, stride=64) == unsupported and dense(width=60) == unsupported
    assert dense(xs=A, ws=A, hidden=72, stride=72) == unsupported  # 8 bits: multiples of 16
    assert dense(stride=56) == unsupported and dense(stride=68) == unsupported and dense(activation=6) == unsupported
    assert dense(width=1 << 20, hidden=1 << 12, stride=1 << 12) == capacity
    assert dense(tokens=2**21 + 1) == unsupported and dense(bias_dtype=1) == invalid and dense(residual=A + 8) == invalid
    assert lib.moe_linear_scratch_bytes(4, 64, 64, 0, 0) >= 0 and lib.moe_linear_scratch_bytes(4, 60, 64, 0, 0) == -1

    def clip(grads=A, tensors=0, norm=A, scratch=A, nbytes=lib.moe_clip_scratch_bytes(), most=1.0):
        return lib.moe_clip_gradients(_lib.CLIP_ARGS(grads, grads, grads, grads, tensors, norm, scratch, nbytes, most),
                                      None)

    assert clip(norm=0) == invalid and clip(most=0.0) == invalid and clip(most=float("nan")) == invalid
    assert clip(nbytes=8) == workspace and clip(tensors=-1) == capacity and clip(tensors=2**16 + 1) == capacity
    assert clip(grads=0, tensors=1) == invalid


def test_overlap_check_takes_no_null_pointers():
    lib = _lib.load_library()
    assert lib.moe_clip_overlap(None, None, None, None, None, 0) == 0
    assert lib.moe_clip_overlap(None, None, None, None, None, 2) == 1  # MOE_ERR_INVALID_ARGUMENT


def test_operands_that_are_no_tensors():
    x = torch.zeros(2, 16, dtype=BF16)
    for call in (lambda: rms_norm([1.0]), lambda: rms_norm(x, [1.0] * 16), lambda: rms_norm(x, residual=[0.0]),
                 lambda: linear(x, [[0.0] * 16]), lambda: linear(x, x.new_zeros(8, 16), [0.0] * 8),
                 lambda: linear(x, x.new_zeros(8, 16), residual=0), lambda: quantize_rows(3), lambda: route_scored([1.0], 1),
                 lambda: clip_gradients([x, None], 1.0)):
        with pytest.raises(TypeError, match="tensor"):
            call()
