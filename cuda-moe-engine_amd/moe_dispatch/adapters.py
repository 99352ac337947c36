"""Low-rank adapters of many requests at once, beside a shared or grouped projection.

A batch's rows belong to requests with adapters of their own: row t with adapter a gets

    output[t] = base[t] + scales[a] * up[a]^T (down[a] x[t]),

``base`` the shared projection's output (``experts.grouped_linear``, or any other product);
rows without an adapter keep it. ``down`` is [N, r, H] and ``up`` [N, r, O], both
rank-major, so that the forward and the gradients are the same kernels; an adapter stored
as [O, r] is transposed once when it is loaded, one of a lower rank padded with zero rows.

``AdapterGroups`` sorts a batch's rows by adapter once a step; every projection of every
layer of that step then takes the same groups. ``low_rank_add`` serves prefill batches
and single tokens alike; ``low_rank_backward`` gives x's and the adapters' gradients. Rows
packed by expert (``ops.dispatch``) are grouped the same way, with each packed row's
expert, or expert and adapter, as its id. No counterpart in the reference.

Checks, streams and errors are those of ``moe_dispatch.training``.
"""

from typing import NamedTuple

import torch

from ._extension import DTYPE_CODES, current_stream_handle, get_extension
from .training import _ptr, on_device, refuse_autograd, require_tensor, shape_of

MAX_ADAPTERS = 4096
MAX_RANK = 128
MAX_ROWS = 2**21
MAX_WIDTH = 2**20


class AdapterGroups:
    """The rows of one batch sorted by adapter, on the device.

    ``assign(ids)`` groups the rows by their int32 adapter ids [T]; an id outside
    [0, adapters) means no adapter. The groups hold until the next ``assign``. One object
    serves one sequential stream of calls; a graph that captured its calls needs it kept.

    The first ``assign`` must run, not be captured (``RuntimeError``): a captured one writes
    nothing before its graph is replayed, and calls before that would read row numbers that
    nobody wrote. A replayed ``assign`` changes the groups without a host call:
    ``low_rank_backward`` cannot tell that a ``hidden`` is older than it.
    """

    def __init__(self, tokens, adapters, *, device="cuda", extension=None):
        if not isinstance(tokens, int) or not 0 <= tokens <= MAX_ROWS:
            raise ValueError("tokens must be an integer in 0..2^21")
        if not isinstance(adapters, int) or not 1 <= adapters <= MAX_ADAPTERS:
            raise ValueError("adapters must be an integer in 1..4096")
        device = torch.device(device)
        if device.type != "cuda" or not torch.cuda.is_available():
            raise RuntimeError("AdapterGroups requires an AMD GPU")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.tokens, self.adapters, self.device = tokens, adapters, device
        self.extension = extension if extension is not None else get_extension()
        self.assignment = 0  # how many times assign ran: what a kept hidden belongs to
        nbytes = self.extension.lib.moe_adapter_table_bytes(tokens, adapters)
        self.table = torch.empty(nbytes // 4, dtype=torch.int32, device=device)
        self.table_bytes = nbytes
        self._sizes = {}  # shapes of x, down and up that fit -> _Sizes

    def assign(self, ids):
        require_tensor(ids, "ids", (self.tokens,), torch.int32, self.device)
        if self.assignment == 0 and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("assign the groups once before capturing: until the graph's first replay they would "
                               "hold no rows' numbers")
        lib = self.extension.lib
        with on_device(self.device):
            lib.check(lib.moe_adapter_group(ids.data_ptr(), self.table.data_ptr(), self.table_bytes, self.tokens,
                                            self.adapters, current_stream_handle(self.device.index)), "assign")
        self.assignment += 1

    @property
    def order(self):
        """The rows in sorted order, int32 [T] (a view): by adapter, each one's rows in
        batch order, rows of no adapter last."""
        return self.table[4:4 + self.tokens]


class LowRankHidden(NamedTuple):
    """``down[a] x`` of one ``low_rank_add``, fp32 [T, r] in the groups' row order, for its
    ``low_rank_backward`` on the same assignment."""

    values: torch.Tensor
    groups: AdapterGroups
    assignment: int


def _check_width(n, name):
    if n < 8 or n % 8 or n > MAX_WIDTH:
        raise ValueError(f"{name} must be a multiple of 8 up to 2^20")


class _Sizes(NamedTuple):
    hidden: int
    width: int
    rank: int
    forward_bytes: int
    backward_bytes: dict  # by which gradients are wanted


def _check_sizes(x, down, up, groups):
    """Sizes and scratch of operands whose shapes fit each other and the groups."""
    tokens, adapters = groups.tokens, groups.adapters
    hidden = shape_of(x, "x", 2)[1]
    rank = shape_of(down, "down", 3)[1]
    width = shape_of(up, "up", 3)[2]
    for t, name, shape in ((x, "x", (tokens, hidden)), (down, "down", (adapters, rank, hidden)),
                           (up, "up", (adapters, rank, width))):
        if t.shape != shape:
            raise ValueError(f"{name}: expected shape {list(shape)}, got {list(t.shape)}")
    _check_width(hidden, "hidden")
    _check_width(width, "width")
    if not 1 <= rank <= MAX_RANK:
        raise ValueError("rank must be in 1..128")
    need = groups.extension.lib.moe_low_rank_scratch_bytes
    sizes = _Sizes(hidden, width, rank, need(tokens, hidden, width, rank, adapters, 0), {})
    groups._sizes[(x.shape, down.shape, up.shape)] = sizes
    return sizes


def _check_operands(x, down, up, groups, scales):
    if not isinstance(groups, AdapterGroups):
        raise TypeError("groups must be AdapterGroups")
    if groups.assignment == 0:
        raise RuntimeError("AdapterGroups.assign has not grouped any rows yet")
    device = groups.device
    for t, name in ((x, "x"), (down, "down"), (up, "up")):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.bfloat16 or t.device != device or not t.is_contiguous():
            require_tensor(t, name, getattr(t, "shape", ()), torch.bfloat16, device)
    sizes = groups._sizes.get((x.shape, down.shape, up.shape))
    if sizes is None:
        sizes = _check_sizes(x, down, up, groups)
    if scales is not None:
        require_tensor(scales, "scales", (groups.adapters,), torch.float32, device)
    return sizes


def _overlaps(a, b):
    return a.numel() > 0 and b.numel() > 0 and a.data_ptr() < b.data_ptr() + b.numel() * b.element_size() and (
        b.data_ptr() < a.data_ptr() + a.numel() * a.element_size())


def low_rank_add(base, x, down, up, groups, *, scales=None, output=None, return_hidden=False):
    """``base`` plus each row's adapter: bf16 [T, O], rounded once from fp32.

    ``base`` bf16 [T, O] (None: 0), x bf16 [T, H], ``scales`` fp32 [N] (None: 1). H and O are
    multiples of 8, r is 1..128. ``output``: where the result goes, ``base`` itself included
    (in place); a new tensor when None. With ``return_hidden`` the result is
    ``(output, hidden)``, ``hidden`` for ``low_rank_backward``.
    """
    hidden, width, rank, need, _ = _check_operands(x, down, up, groups, scales)
    tokens, device = groups.tokens, groups.device
    if base is not None:
        require_tensor(base, "base", (tokens, width), torch.bfloat16, device)
    if output is not None:
        require_tensor(output, "output", (tokens, width), torch.bfloat16, device)
        if any(_overlaps(output, t) for t in (x, down, up)) or (
                base is not None and output.data_ptr() != base.data_ptr() and _overlaps(output, base)):
            raise ValueError("output may be base itself, but must not overlap another operand")
    refuse_autograd(base, x, down, up, scales, output)
    lib = groups.extension.lib
    with on_device(device):
        if output is None:
            output = torch.empty_like(base) if base is not None else x.new_empty((tokens, width))
        kept = x.new_empty((tokens, rank), dtype=torch.float32) if return_hidden else None
        scratch = x.new_empty(need // 2) if need else None
        lib.check(lib.moe_low_rank_add(
            x.data_ptr(), down.data_ptr(), up.data_ptr(), _ptr(scales), groups.table.data_ptr(),
            groups.table_bytes, _ptr(base), output.data_ptr(), _ptr(kept), _ptr(scratch), need, tokens,
            hidden, width, rank, groups.adapters, current_stream_handle(device.index)), "low_rank_add")
    return (output, LowRankHidden(kept, groups, groups.assignment)) if return_hidden else output


def low_rank_backward(grad_output, x, down, up, groups, *, scales=None, hidden, grad_x=None,
                      grad_dtype=torch.float32, gradients=(True, True, True)):
    """Gradients of ``low_rank_add``: ``(grad_x, grad_down, grad_up)``; base's is ``grad_output``.

    ``hidden`` is what the forward returned with ``return_hidden``, on the groups' current
    assignment. ``grad_x`` bf16 [T, H] is x's gradient along its other paths (the shared
    projection): the result is the sum, rounded once. grad_down and grad_up are
    ``grad_dtype`` (fp32, or bf16 rounded once), zero for adapters without rows. scales get
    no gradient. ``gradients``: which of the three are wanted; the others are None, are not
    computed and take no memory.
    """
    h, width, rank, _, scratch_bytes = _check_operands(x, down, up, groups, scales)
    tokens, device = groups.tokens, groups.device
    require_tensor(grad_output, "grad_output", (tokens, width), torch.bfloat16, device)
    if not isinstance(hidden, LowRankHidden):
        raise TypeError("hidden must be what low_rank_add returned with return_hidden")
    if hidden.groups is not groups or hidden.assignment != groups.assignment:
        raise RuntimeError("hidden belongs to another assignment of these groups")
    require_tensor(hidden.values, "hidden", (tokens, rank), torch.float32, device)
    if grad_x is not None:
        require_tensor(grad_x, "grad_x", (tokens, h), torch.bfloat16, device)
    if grad_dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("grad_dtype must be float32 or bfloat16")
    refuse_autograd(grad_output, x, down, up, scales, grad_x)
    lib = groups.extension.lib
    with on_device(device):
        want_x, want_down, want_up = gradients
        without = (0 if want_x else 2) + (0 if want_down else 4) + (0 if want_up else 8)  # MOE_WITHOUT_GRAD_*
        need = scratch_bytes.get(without)
        if need is None:
            need = scratch_bytes[without] = lib.moe_low_rank_scratch_bytes(tokens, h, width, rank, groups.adapters,
                                                                           1 + without)
        out_x = torch.empty_like(x) if want_x else None
        grad_down = torch.empty_like(down, dtype=grad_dtype) if want_down else None
        grad_up = torch.empty_like(up, dtype=grad_dtype) if want_up else None
        scratch = x.new_empty(need // 2) if need else None
        lib.check(lib.moe_low_rank_backward(
            grad_output.data_ptr(), x.data_ptr(), down.data_ptr(), up.data_ptr(), _ptr(scales),
            groups.table.data_ptr(), groups.table_bytes, hidden.values.data_ptr(), _ptr(grad_x),
            _ptr(out_x), _ptr(grad_down), _ptr(grad_up), DTYPE_CODES[grad_dtype], _ptr(scratch),
            need, tokens, h, width, rank, groups.adapters, current_stream_handle(device.index)),
            "low_rank_backward")
    return out_x, grad_down, grad_up
