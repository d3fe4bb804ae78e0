"""What the emulated ranks exchange inside a transformer block, on torch tensors.

``EmulatedGroup`` offers these as methods; this module holds their argument checks, the calls into the HIP library
(``include/sar.h``, block operators) and their gradients.  A block's tokens are the rows of one tensor, sharded over
the ranks by rows; experts are owned by the ranks in equal consecutive parts.

Every call runs on torch's current stream of the group's device, waits for nothing and takes its outputs and
workspaces from torch's allocator, so it may be captured into a graph (each graph then has workspaces of its own).
The differentiable calls refuse to RECORD gradients while a stream is being captured: a captured training step calls
them under ``torch.no_grad()`` together with the ``*_backward`` calls, which need no autograd graph.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import capi

DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_EXPERTS, MAX_TOPK, MAX_NORM_DIM = 1024, 64, 16384
_GATE_NONE, _GATE_CHANNEL, _GATE_TOKEN, _GATE_FULL = range(4)


class Routing:
    """Where every (token, choice) slot goes, as ``EmulatedGroup.route`` found it.  ``row_of_slot`` [tokens, topk]: the
    slot's row among the rows sorted by expert, -1 = dropped.  ``slot_of_row`` [tokens * topk]: the slot (token * topk
    + choice) of each row, -1 behind the last.  ``offsets`` [num_experts + 1]: first row of each expert, then the
    number of rows; ``rank_offsets`` [ranks + 1]: the same for the ranks that own the experts.  All int32 on the GPU."""

    __slots__ = ("row_of_slot", "slot_of_row", "offsets", "num_experts", "ranks")

    def __init__(self, row_of_slot, slot_of_row, offsets, num_experts: int, ranks: int):
        self.row_of_slot, self.slot_of_row, self.offsets = row_of_slot, slot_of_row, offsets
        self.num_experts, self.ranks = num_experts, ranks

    @property
    def tokens(self) -> int:
        return self.row_of_slot.shape[0]

    @property
    def topk(self) -> int:
        return self.row_of_slot.shape[1]

    @property
    def rank_offsets(self):
        return self.offsets[::self.num_experts // self.ranks]


class ReduceNormSaved(NamedTuple):
    """What ``reduce_norm_backward`` needs of a forward call."""
    sources: int
    copies: int
    partial_shape: tuple
    total: torch.Tensor
    stats: torch.Tensor
    residual: torch.Tensor
    pre_weight: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]
    residual_scale: float
    eps: float


class ReduceNormGrads(NamedTuple):
    """Gradients of ``reduce_norm``; ``partials`` has the shape the partials were given in ([ranks, tokens, dim] for a
    sequence of tensors), and what was not asked for is None."""
    partials: Optional[torch.Tensor]
    residual: Optional[torch.Tensor]
    pre_weight: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]


def _tensor(name, t, shape=None, dtypes=None):
    """Type, shape and layout of an argument; the device comes last so that everything else can be said without one."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, need %s" % (name, tuple(t.shape), tuple(shape)))
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError("%s has dtype %s, need %s" % (name, t.dtype, " or ".join(str(d) for d in dtypes)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)


def _on_device(group, **tensors):
    for name, t in tensors.items():
        if t is not None and (not t.is_cuda or t.device.index != group.device):
            raise ValueError("%s must be a CUDA tensor on device %d" % (name, group.device))


def _stream(group) -> int:
    return torch.cuda.current_stream(group.device).cuda_stream


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _recording(*tensors) -> bool:
    """Whether autograd has to record the call."""
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors):
        return False
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("gradients cannot be recorded while a stream is being captured: call this under torch.no_grad() "
                           "and the *_backward call in the same capture")
    return True


def _refuse_captured_backward():
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the backward pass of a call recorded by autograd cannot be captured: capture the *_backward call")


# ---- route ---------------------------------------------------------------------------------------------------

def route(group, experts, num_experts: int) -> Routing:
    if not isinstance(experts, torch.Tensor) or experts.dim() != 2:
        raise ValueError("experts must be a tensor [tokens, topk]")
    tokens, topk = experts.shape
    _tensor("experts", experts, dtypes=(torch.int64, torch.int32))
    if not 1 <= topk <= MAX_TOPK:
        raise ValueError("topk must be 1 to %d, got %d" % (MAX_TOPK, topk))
    if not 1 <= num_experts <= MAX_EXPERTS or num_experts % group.n:
        raise ValueError("num_experts must be a multiple of the %d ranks, at most %d: got %d" % (group.n, MAX_EXPERTS, num_experts))
    if tokens * topk >= 1 << 31:
        raise ValueError("tokens * topk must stay below 2^31")
    _on_device(group, experts=experts)
    lib = group._lib
    slots = tokens * topk
    # one allocation: row_of_slot, slot_of_row, offsets
    out = torch.empty(2 * slots + num_experts + 1, dtype=torch.int32, device=experts.device)
    need = lib.lib.sar_route_workspace(tokens, topk, num_experts)
    work = torch.empty(need // 4, dtype=torch.int32, device=experts.device) if need else None
    base = out.data_ptr()
    lib.check(lib.lib.sar_route(group.device, _stream(group), experts.data_ptr(), experts.element_size(), tokens, topk, num_experts,
                                base, base + 4 * slots, base + 8 * slots, _ptr(work), need))
    return Routing(out[:slots].view(tokens, topk), out[slots:2 * slots], out[2 * slots:], num_experts, group.n)


# ---- dispatch, combine -----------------------------------------------------------------------------------------

def _dispatch(group, rows, routing, weights=None):
    dim = rows.shape[1]
    out = torch.empty(routing.tokens * routing.topk, dim, dtype=rows.dtype, device=rows.device)
    lib = group._lib
    lib.check(lib.lib.sar_dispatch(group.device, _stream(group), DTYPE_CODES[rows.dtype], rows.data_ptr(), routing.tokens, routing.topk, dim,
                                   routing.row_of_slot.data_ptr(), routing.offsets.data_ptr(), routing.num_experts,
                                   _ptr(weights), DTYPE_CODES[weights.dtype] if weights is not None else 0, out.data_ptr()))
    return out


def _combine(group, rows, routing, weights=None):
    dim = rows.shape[1]
    out = torch.empty(routing.tokens, dim, dtype=rows.dtype, device=rows.device)
    lib = group._lib
    lib.check(lib.lib.sar_combine(group.device, _stream(group), DTYPE_CODES[rows.dtype], rows.data_ptr(), routing.tokens, routing.topk, dim,
                                  routing.row_of_slot.data_ptr(), _ptr(weights), DTYPE_CODES[weights.dtype] if weights is not None else 0, out.data_ptr()))
    return out


def _combine_backward(group, grad, rows, routing, weights, want_rows, want_weights):
    if not want_weights:
        return (_dispatch(group, grad, routing, weights) if want_rows else None), None
    grad_rows = torch.empty_like(rows) if want_rows else None
    grad_weights = torch.empty_like(weights)
    lib = group._lib
    lib.check(lib.lib.sar_combine_backward(group.device, _stream(group), DTYPE_CODES[rows.dtype], grad.data_ptr(), rows.data_ptr(), routing.tokens,
                                           routing.topk, rows.shape[1], routing.row_of_slot.data_ptr(), routing.offsets.data_ptr(),
                                           routing.num_experts, weights.data_ptr(), DTYPE_CODES[weights.dtype], _ptr(grad_rows), grad_weights.data_ptr()))
    return grad_rows, grad_weights


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, group, routing):
        ctx.group, ctx.routing = group, routing
        return _dispatch(group, rows, routing)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _refuse_captured_backward()
        return _combine(ctx.group, grad.contiguous(), ctx.routing), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, group, routing):
        ctx.group, ctx.routing = group, routing
        ctx.save_for_backward(rows, weights)
        return _combine(group, rows, routing, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _refuse_captured_backward()
        rows, weights = ctx.saved_tensors
        grads = _combine_backward(ctx.group, grad.contiguous(), rows, ctx.routing, weights, ctx.needs_input_grad[0],
                                  weights is not None and ctx.needs_input_grad[1])
        return grads[0], grads[1], None, None


def _check_rows(name, t, rows):
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.shape[0] != rows:
        raise ValueError("%s must be a tensor [%d, dim], got %s" % (name, rows, tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__))
    _tensor(name, t, dtypes=tuple(DTYPE_CODES))
    if not 1 <= t.shape[1] <= 1 << 24:
        raise ValueError("%s needs 1 to 2^24 columns" % name)


def _check_weights(routing, weights, dtype):
    if weights is not None:
        _tensor("weights", weights, (routing.tokens, routing.topk), (dtype,) if dtype == torch.float32 else (torch.float32, dtype))


def dispatch(group, tokens, routing):
    if not isinstance(routing, Routing):
        raise TypeError("routing must come from EmulatedGroup.route")
    _check_rows("tokens", tokens, routing.tokens)
    _on_device(group, tokens=tokens, routing=routing.offsets)
    if _recording(tokens):
        return _Dispatch.apply(tokens, group, routing)
    return _dispatch(group, tokens, routing)


def combine(group, rows, routing, weights=None):
    if not isinstance(routing, Routing):
        raise TypeError("routing must come from EmulatedGroup.route")
    _check_rows("rows", rows, routing.tokens * routing.topk)
    _check_weights(routing, weights, rows.dtype)
    _on_device(group, rows=rows, weights=weights, routing=routing.offsets)
    if _recording(rows, weights):
        return _Combine.apply(rows, weights, group, routing)
    return _combine(group, rows, routing, weights)


def dispatch_backward(group, grad, routing):
    if not isinstance(routing, Routing):
        raise TypeError("routing must come from EmulatedGroup.route")
    _check_rows("grad", grad, routing.tokens * routing.topk)
    _on_device(group, grad=grad, routing=routing.offsets)
    return _combine(group, grad, routing)


def combine_backward(group, grad, rows, routing, weights=None):
    if not isinstance(routing, Routing):
        raise TypeError("routing must come from EmulatedGroup.route")
    _check_rows("rows", rows, routing.tokens * routing.topk)
    _tensor("grad", grad, (routing.tokens, rows.shape[1]), (rows.dtype,))
    _check_weights(routing, weights, rows.dtype)
    _on_device(group, grad=grad, rows=rows, weights=weights, routing=routing.offsets)
    return _combine_backward(group, grad, rows, routing, weights, True, weights is not None)


# ---- sum over the ranks, norms, gate, residual -------------------------------------------------------------------

def _reduce_norm(group, partials, residual, pre_weight, post_weight, gate, residual_scale, eps, gather, save):
    """`partials`: list of tensors [tokens, dim].  Returns hidden, normed (or None), total and stats (or None)."""
    tokens, dim = residual.shape
    copies = group.n if gather else 1
    hidden = torch.empty_like(residual)
    normed = None
    if pre_weight is not None:
        normed = torch.empty((copies, tokens, dim) if gather else (tokens, dim), dtype=residual.dtype, device=residual.device)
    total = stats = None
    if save:
        total = partials[0] if len(partials) == 1 else torch.empty(tokens, dim, dtype=torch.float32, device=residual.device)
        stats = torch.empty(2, tokens, dtype=torch.float32, device=residual.device)
    args = _norm_args(len(partials), copies, residual, pre_weight, post_weight, gate, residual_scale, eps, stats)
    args.partials = (ctypes.c_void_p * len(partials))(*[p.data_ptr() for p in partials])
    args.hidden, args.normed = hidden.data_ptr(), _ptr(normed)
    args.total = total.data_ptr() if save and len(partials) > 1 else None
    lib = group._lib
    lib.check(lib.lib.sar_reduce_norm(group.device, _stream(group), ctypes.byref(args)))
    return hidden, normed, total, stats


def _norm_args(sources, copies, residual, pre_weight, post_weight, gate, residual_scale, eps, stats):
    tokens, dim = residual.shape
    code = DTYPE_CODES[residual.dtype]
    args = capi.ReduceNormArgs(dtype=code, pre_dtype=code, post_dtype=code, gate_dtype=code, sources=sources, copies=copies,
                               tokens=tokens, dim=dim, eps=eps, residual_scale=residual_scale, residual=residual.data_ptr())
    if pre_weight is not None:
        args.pre_dtype, args.pre_weight = DTYPE_CODES[pre_weight.dtype], pre_weight.data_ptr()
    if post_weight is not None:
        args.post_dtype, args.post_weight = DTYPE_CODES[post_weight.dtype], post_weight.data_ptr()
    if gate is not None:
        args.gate_dtype, args.gate = DTYPE_CODES[gate.dtype], gate.data_ptr()
        args.gate_kind = _GATE_CHANNEL if gate.dim() == 1 else _GATE_TOKEN if gate.shape[1] == 1 and dim > 1 else _GATE_FULL
    if stats is not None:
        args.stats = stats.data_ptr()
    return args


def _reduce_norm_backward(group, saved: ReduceNormSaved, grad_hidden, grad_normed, want) -> ReduceNormGrads:
    """`want`: truth values for partials, residual, pre_weight, post_weight, gate."""
    s = saved
    tokens, dim = s.residual.shape
    dev = s.residual.device
    args = _norm_args(s.sources, s.copies, s.residual, s.pre_weight, s.post_weight, s.gate, s.residual_scale, s.eps, s.stats)
    if grad_normed is None or s.pre_weight is None:
        grad_normed = None
    out = ReduceNormGrads(
        torch.empty(s.partial_shape, dtype=s.residual.dtype, device=dev) if want[0] else None,
        torch.empty_like(s.residual) if want[1] else None,
        torch.empty_like(s.pre_weight) if want[2] and s.pre_weight is not None else None,
        torch.empty_like(s.post_weight) if want[3] and s.post_weight is not None else None,
        torch.empty_like(s.gate) if want[4] and s.gate is not None else None)
    lib = group._lib
    need = lib.lib.sar_reduce_norm_workspace(tokens, dim, args.dtype)
    work = torch.empty(need // 4, dtype=torch.float32, device=dev)
    grads = capi.ReduceNormGrads(total=s.total.data_ptr(), total_dtype=DTYPE_CODES[s.total.dtype], grad_hidden=_ptr(grad_hidden),
                                 grad_normed=_ptr(grad_normed), grad_partials=_ptr(out.partials), grad_residual=_ptr(out.residual),
                                 grad_pre_weight=_ptr(out.pre_weight), grad_post_weight=_ptr(out.post_weight), grad_gate=_ptr(out.gate),
                                 workspace=work.data_ptr(), workspace_bytes=need)
    lib.check(lib.lib.sar_reduce_norm_backward(group.device, _stream(group), ctypes.byref(args), ctypes.byref(grads)))
    return out


class _ReduceNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, group, shape, residual_scale, eps, gather, residual, pre_weight, post_weight, gate, *partials):
        rows = partials if len(shape) == 2 or len(partials) > 1 else partials[0].unbind(0)
        hidden, normed, total, stats = _reduce_norm(group, rows, residual, pre_weight, post_weight, gate, residual_scale, eps, gather, True)
        ctx.group, ctx.shape, ctx.sources, ctx.inputs = group, shape, len(rows), len(partials)
        ctx.options = (residual_scale, eps, gather)
        ctx.save_for_backward(total, stats, residual, pre_weight, post_weight, gate)
        ctx.set_materialize_grads(False)
        return hidden, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_hidden, grad_normed):
        _refuse_captured_backward()
        total, stats, residual, pre_weight, post_weight, gate = ctx.saved_tensors
        scale, eps, gather = ctx.options
        saved = ReduceNormSaved(ctx.sources, ctx.group.n if gather else 1, ctx.shape, total, stats, residual, pre_weight, post_weight, gate, scale, eps)
        need = ctx.needs_input_grad
        g = _reduce_norm_backward(ctx.group, saved, grad_hidden.contiguous() if grad_hidden is not None else None,
                                  grad_normed.contiguous() if grad_normed is not None else None, (any(need[9:]),) + tuple(need[5:9]))
        if g.partials is None:
            partials = (None,) * ctx.inputs
        elif ctx.inputs == 1:
            partials = (g.partials,)
        else:
            partials = g.partials.unbind(0)
        return (None,) * 5 + (g.residual, g.pre_weight, g.post_weight, g.gate) + tuple(partials)


def reduce_norm(group, partials: Union[torch.Tensor, Sequence[torch.Tensor]], residual, pre_weight=None, post_weight=None, gate=None,
                residual_scale: float = 1.0, eps: float = 1e-6, gather: bool = True, save: bool = False):
    if not isinstance(residual, torch.Tensor) or residual.dim() != 2:
        raise ValueError("residual must be a tensor [tokens, dim]")
    _tensor("residual", residual, dtypes=tuple(DTYPE_CODES))
    tokens, dim = residual.shape
    dtype = residual.dtype
    if not 1 <= dim <= MAX_NORM_DIM:
        raise ValueError("dim must be 1 to %d, got %d" % (MAX_NORM_DIM, dim))
    if isinstance(partials, torch.Tensor):
        inputs = (partials,)
        if partials.dim() not in (2, 3) or partials.shape[-2:] != residual.shape or (partials.dim() == 3 and partials.shape[0] != group.n):
            raise ValueError("partials must be [%d ranks, tokens, dim] or, as a finished output, [tokens, dim]: got %s with residual %s"
                             % (group.n, tuple(partials.shape), tuple(residual.shape)))
        _tensor("partials", partials, dtypes=(dtype,))
        shape = tuple(partials.shape)
    else:
        inputs = tuple(partials)
        if len(inputs) != group.n:
            raise ValueError("need one partial output per emulated rank: %d, got %d" % (group.n, len(inputs)))
        for p in inputs:
            _tensor("a partial output", p, (tokens, dim), (dtype,))
        shape = (group.n, tokens, dim)
    kinds = (dtype,) if dtype == torch.float32 else (torch.float32, dtype)
    if pre_weight is not None:
        _tensor("pre_weight", pre_weight, (dim,), kinds)
    if post_weight is not None:
        _tensor("post_weight", post_weight, (dim,), kinds)
    if gate is not None:
        _tensor("gate", gate, dtypes=kinds)
        if tuple(gate.shape) not in ((dim,), (tokens, 1), (tokens, dim)):
            raise ValueError("gate must be [dim], [tokens, 1] or [tokens, dim]: got %s" % (tuple(gate.shape),))
    if not eps >= 0 or eps == float("inf"):
        raise ValueError("eps must be a finite number, zero or more")
    _on_device(group, residual=residual, pre_weight=pre_weight, post_weight=post_weight, gate=gate)
    for p in inputs:
        _on_device(group, partials=p)
    if _recording(residual, pre_weight, post_weight, gate, *inputs):
        if save:
            raise ValueError("save=True is for calls under torch.no_grad(): autograd keeps what it needs by itself")
        return _ReduceNorm.apply(group, shape, float(residual_scale), float(eps), bool(gather), residual, pre_weight, post_weight, gate, *inputs)
    rows = inputs if len(shape) == 2 or len(inputs) > 1 else inputs[0].unbind(0)
    hidden, normed, total, stats = _reduce_norm(group, rows, residual, pre_weight, post_weight, gate, residual_scale, eps, gather, save)
    if not save:
        return hidden, normed
    return hidden, normed, ReduceNormSaved(len(rows), group.n if gather else 1, shape, total, stats, residual, pre_weight, post_weight, gate,
                                           float(residual_scale), float(eps))


def reduce_norm_backward(group, saved: ReduceNormSaved, grad_hidden=None, grad_normed=None) -> ReduceNormGrads:
    if not isinstance(saved, ReduceNormSaved):
        raise TypeError("saved must come from reduce_norm(..., save=True)")
    tokens, dim = saved.residual.shape
    if grad_hidden is not None:
        _tensor("grad_hidden", grad_hidden, (tokens, dim), (saved.residual.dtype,))
    if grad_normed is not None:
        if saved.pre_weight is None:
            raise ValueError("grad_normed without a pre_weight in the forward call")
        ok = [(saved.copies, tokens, dim)] + ([(tokens, dim)] if saved.copies == 1 else [])
        if tuple(grad_normed.shape) not in ok:
            raise ValueError("grad_normed has shape %s, need %s" % (tuple(grad_normed.shape), ok[-1]))
        _tensor("grad_normed", grad_normed, dtypes=(saved.residual.dtype,))
    _on_device(group, grad_hidden=grad_hidden, grad_normed=grad_normed, residual=saved.residual)
    return _reduce_norm_backward(group, saved, grad_hidden, grad_normed, (True,) * 5)
