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
import functools
from typing import NamedTuple, Optional, Sequence, Union

import torch
from torch.autograd import forward_ad

from . import capi

DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_EXPERTS, MAX_TOPK, MAX_NORM_DIM = 1024, 64, 16384
_GATE_NONE, _GATE_CHANNEL, _GATE_TOKEN, _GATE_FULL = range(4)


class Routing:
    """Where every (token, choice) slot goes, as ``EmulatedGroup.route`` found it.  ``row_of_slot`` [tokens, topk]: the
    slot's row among the rows sorted by expert, -1 = dropped.  ``slot_of_row`` [tokens * topk]: the slot (token * topk
    + choice) of each row, -1 behind the last.  ``offsets`` [num_experts + 1]: first row of each expert, then the
    number of rows; ``rank_offsets`` [ranks + 1]: the same for the ranks that own the experts.  All int32 on the GPU.  The tensors
    stay as they are until the backward pass of every call that took them has run; autograd raises if they did not.
    A routing put together by hand is checked here, once, so its parts cannot be exchanged afterwards; row numbers outside
    the rows count as dropped, and rows below ``offsets[-1]`` that no slot names are left unwritten by ``dispatch``."""

    __slots__ = ("row_of_slot", "slot_of_row", "offsets", "num_experts", "ranks")

    def __init__(self, row_of_slot, slot_of_row, offsets, num_experts: int, ranks: int):
        if ranks < 1 or num_experts < 1 or row_of_slot.dim() != 2 or slot_of_row.numel() != row_of_slot.numel() or offsets.numel() != num_experts + 1 or num_experts % ranks:
            raise ValueError("row_of_slot [tokens, topk], slot_of_row [tokens * topk] and offsets [num_experts + 1] do not fit each other")
        for t in (row_of_slot, slot_of_row, offsets):
            if t.dtype is not torch.int32 or not t.is_contiguous() or t.device != offsets.device:
                raise ValueError("a routing is made of contiguous int32 tensors on one device")
        _fill(self, row_of_slot, slot_of_row, offsets, num_experts, ranks)

    def __setattr__(self, name, value):
        raise AttributeError("the parts of a routing are checked when it is made: make another Routing")

    def __reduce__(self):
        return type(self), (self.row_of_slot, self.slot_of_row, self.offsets, self.num_experts, self.ranks)

    @property
    def tokens(self) -> int:
        return self.row_of_slot.shape[0]

    @property
    def topk(self) -> int:
        return self.row_of_slot.shape[1]

    @property
    def rank_offsets(self):
        return self.offsets[::self.num_experts // self.ranks]


_PARTS = tuple(getattr(Routing, name).__set__ for name in Routing.__slots__)


def _fill(routing: Routing, *parts) -> Routing:
    for put, part in zip(_PARTS, parts):
        put(routing, part)
    return routing


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
    """Says what is wrong with an argument; the device comes last so that everything else can be said without one."""
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
        if t is not None and t.get_device() != group.device:
            raise ValueError("%s must be a CUDA tensor on device %d" % (name, group.device))


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _ptr(t):
    return t.data_ptr() if t is not None else None


_tracing, _modes, _function_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._is_torch_function_mode_enabled
_transforms = torch._C._functorch.peek_interpreter_stack


def _refuse_tracers():
    """The kernels run behind torch's dispatcher: whoever records its operations, or runs them on tensors without
    memory, gets the allocation of the outputs and nothing that fills them.  A dispatch mode that only watches
    (counts, logs, decides what to keep) is none of torch's own recorders and stays allowed."""
    if _modes() or _function_modes() or _tracing() or _transforms() is not None:
        _refuse_recorders()


def _refuse_recorders():
    if (_tracing() or any(m.is_infra_mode() for m in torch.utils._python_dispatch._get_current_dispatch_mode_stack())
            or torch._C._dispatch_tls_is_dispatch_key_included(torch._C.DispatchKey.PreDispatch)
            or any(i.key() == torch._C._functorch.TransformType.Functionalize for i in torch._C._functorch.get_interpreter_stack() or ())):
        raise RuntimeError("the block operators cannot be traced: their kernels are no torch operations")


def _refuse_tangents(*tensors):
    """There are no forward-mode derivatives: a tangent would be lost, which reads as a derivative of zero."""
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the block operators have no forward-mode derivatives")


def _capturing(device: int) -> bool:
    """Whether the current stream of `device`, which need not be the current device, is being captured."""
    if device < 0 or device == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _recording(*tensors) -> bool:
    """Whether autograd has to record the call."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(*tensors)
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            break
    else:
        return False
    if _capturing(t.get_device()):
        raise RuntimeError("gradients cannot be recorded while a stream is being captured: call this under torch.no_grad() "
                           "and the *_backward call in the same capture")
    return True


class _Node(torch.autograd.Function):
    """What the recorded calls share: `gradients(ctx, *grads)` is the backward pass.  It is not differentiable itself;
    the wrapper that says so when somebody tries is only paid for where a graph of the backward pass is asked for."""

    @staticmethod
    def gradients(ctx, *grads):
        raise NotImplementedError

    @classmethod
    def _backward(cls, ctx, *grads):
        _refuse_tracers()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the backward pass of a call recorded by autograd cannot be captured: capture the *_backward call")
        if torch.is_grad_enabled():
            return torch.autograd.function.once_differentiable(cls.gradients)(ctx, *grads)
        return cls.gradients(ctx, *grads)


# ---- route ---------------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=4096)
def _route_workspace(tokens, topk, num_experts):
    return capi.load_library().lib.sar_route_workspace(tokens, topk, num_experts)


def route(group, experts, num_experts: int) -> Routing:
    _refuse_tracers()
    if not isinstance(experts, torch.Tensor) or experts.dim() != 2:
        raise ValueError("experts must be a tensor [tokens, topk]")
    tokens, topk = experts.shape
    _tensor("experts", experts, dtypes=(torch.int64, torch.int32))
    if not 1 <= topk <= MAX_TOPK:
        raise ValueError("topk must be 1 to %d, got %d" % (MAX_TOPK, topk))
    if not 1 <= num_experts <= MAX_EXPERTS or num_experts % group.n:
        raise ValueError("num_experts must be a multiple of the %d ranks, at most %d: got %d" % (group.n, MAX_EXPERTS, num_experts))
    slots = tokens * topk
    if slots >= 1 << 31:
        raise ValueError("tokens * topk must stay below 2^31")
    _on_device(group, experts=experts)
    lib, device = group._lib, experts.device
    row_of_slot = torch.empty((tokens, topk), dtype=torch.int32, device=device)
    slot_of_row = torch.empty(slots, dtype=torch.int32, device=device)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    need = _route_workspace(tokens, topk, num_experts)
    work = torch.empty(need // 4, dtype=torch.int32, device=device) if need else None
    lib.check(lib.lib.sar_route(group.device, _raw_stream(group.device), experts.data_ptr(), experts.element_size(), tokens, topk, num_experts,
                                row_of_slot.data_ptr(), slot_of_row.data_ptr(), offsets.data_ptr(), _ptr(work), need))
    return _fill(object.__new__(Routing), row_of_slot, slot_of_row, offsets, num_experts, group.n)


# ---- dispatch, combine -----------------------------------------------------------------------------------------

def _dispatch(group, rows, row_of_slot, offsets, weights=None):
    tokens, topk = row_of_slot.shape
    dim = rows.shape[1]
    out = rows.new_empty((tokens * topk, dim))
    code, lib = DTYPE_CODES[rows.dtype], group._lib
    lib.check(lib.lib.sar_dispatch(group.device, _raw_stream(group.device), code, rows.data_ptr(), tokens, topk, dim,
                                   row_of_slot.data_ptr(), offsets.data_ptr(), offsets.numel() - 1,
                                   _ptr(weights), DTYPE_CODES[weights.dtype] if weights is not None else 0, out.data_ptr()))
    return out


def _combine(group, rows, row_of_slot, weights=None):
    tokens, topk = row_of_slot.shape
    dim = rows.shape[1]
    out = rows.new_empty((tokens, dim))
    code, lib = DTYPE_CODES[rows.dtype], group._lib
    lib.check(lib.lib.sar_combine(group.device, _raw_stream(group.device), code, rows.data_ptr(), tokens, topk, dim,
                                  row_of_slot.data_ptr(), _ptr(weights), DTYPE_CODES[weights.dtype] if weights is not None else 0, out.data_ptr()))
    return out


def _combine_backward(group, grad, rows, row_of_slot, offsets, weights, want_rows, want_weights):
    if not want_weights:
        return (_dispatch(group, grad, row_of_slot, offsets, weights) if want_rows else None), None
    tokens, topk = row_of_slot.shape
    grad_rows = torch.empty_like(rows) if want_rows else None
    grad_weights = torch.empty_like(weights)
    lib = group._lib
    lib.check(lib.lib.sar_combine_backward(group.device, _raw_stream(group.device), DTYPE_CODES[rows.dtype], grad.data_ptr(), rows.data_ptr(),
                                           tokens, topk, rows.shape[1], row_of_slot.data_ptr(), offsets.data_ptr(), offsets.numel() - 1,
                                           weights.data_ptr(), DTYPE_CODES[weights.dtype], _ptr(grad_rows), grad_weights.data_ptr()))
    return grad_rows, grad_weights


def _savable(t):
    """A routing's tensor for save_for_backward, whose version autograd then holds against the one it finds in the
    backward pass.  What route() made under inference_mode has no version and is refused there: a copy has one."""
    return t.clone() if t.is_inference() else t


_HOOKED = "a saved-tensor hook gave back a tensor of another type, size, order or device than it was given"
_hooks = torch._C._autograd._top_saved_tensors_default_hooks      # those in force, or None: asked when tensors are saved


def _given_back(group, t, dtype, shape):
    """A saved tensor as autograd gives it back.  Saved-tensor hooks come in between: what they return in another type,
    size, order or place would be read as what it was."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != group.device or not t.is_contiguous():
        raise RuntimeError(_HOOKED)


class _Dispatch(_Node):
    @staticmethod
    def forward(ctx, rows, plain):
        group, routing = plain
        ctx.plain = (group, routing.row_of_slot.shape, _hooks(True) is not None)
        ctx.save_for_backward(_savable(routing.row_of_slot))
        return _dispatch(group, rows, routing.row_of_slot, routing.offsets)

    @staticmethod
    def gradients(ctx, grad):
        (group, size, hooked), (row_of_slot,) = ctx.plain, ctx.saved_tensors
        if hooked:
            _given_back(group, row_of_slot, torch.int32, size)
        return _combine(group, grad.contiguous(), row_of_slot), None

    @staticmethod
    def backward(ctx, grad):
        return _Dispatch._backward(ctx, grad)


class _Combine(_Node):
    @staticmethod
    def forward(ctx, rows, weights, plain):
        group, routing = plain
        hooked = _hooks(True) and (routing.row_of_slot.shape, routing.offsets.shape, weights.dtype if weights is not None else None)
        ctx.plain = (group, hooked)
        # the rows, tokens * topk of them, are read by the weights' gradient alone
        kept = rows if weights is not None and ctx.needs_input_grad[1] else None
        ctx.save_for_backward(kept, weights, _savable(routing.row_of_slot), _savable(routing.offsets))
        return _combine(group, rows, routing.row_of_slot, weights)

    @staticmethod
    def gradients(ctx, grad):
        rows, weights, row_of_slot, offsets = ctx.saved_tensors
        (group, hooked), need = ctx.plain, ctx.needs_input_grad
        if hooked:
            size, ends, weight_dtype = hooked
            _given_back(group, row_of_slot, torch.int32, size)
            _given_back(group, offsets, torch.int32, ends)
            if rows is not None:
                _given_back(group, rows, grad.dtype, (size[0] * size[1], grad.shape[1]))
            if weights is not None:
                _given_back(group, weights, weight_dtype, size)
        a, b = _combine_backward(group, grad.contiguous(), rows, row_of_slot, offsets, weights, need[0], weights is not None and need[1])
        return a, b, None

    @staticmethod
    def backward(ctx, grad):
        return _Combine._backward(ctx, grad)


def _routing_rows(group, name, t, routing, sorted_rows):
    """The checks of a tensor of rows against a routing."""
    if not isinstance(routing, Routing):
        raise TypeError("routing must come from EmulatedGroup.route")
    tokens, topk = routing.row_of_slot.shape
    rows = tokens * topk if sorted_rows else tokens
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.shape[0] != rows:
        raise ValueError("%s must be a tensor [%d, dim], got %s" % (name, rows, tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__))
    _tensor(name, t, dtypes=DTYPE_CODES)
    if not 1 <= t.shape[1] <= 1 << 24:
        raise ValueError("%s needs 1 to 2^24 columns" % name)


def _fits_rows(group, t, routing, sorted_rows):
    """Whether the checks above and of the device pass, in as little time as they take."""
    if not isinstance(t, torch.Tensor) or not isinstance(routing, Routing):
        return False
    size = t.shape
    if len(size) != 2:
        return False
    tokens, topk = routing.row_of_slot.shape
    return (size[0] == (tokens * topk if sorted_rows else tokens) and t.dtype in DTYPE_CODES and t.is_contiguous()
            and t.get_device() == group.device and routing.offsets.get_device() == group.device and 1 <= size[1] <= 1 << 24)


def _check_weights(routing, weights, dtype):
    if weights is not None:
        _tensor("weights", weights, routing.row_of_slot.shape, (torch.float32, dtype))


def dispatch(group, tokens, routing):
    _refuse_tracers()
    if not _fits_rows(group, tokens, routing, False):
        _routing_rows(group, "tokens", tokens, routing, False)
        _on_device(group, tokens=tokens, routing=routing.offsets)
    if _recording(tokens):
        return _Dispatch.apply(tokens, (group, routing))
    return _dispatch(group, tokens, routing.row_of_slot, routing.offsets)


def combine(group, rows, routing, weights=None):
    _refuse_tracers()
    if not _fits_rows(group, rows, routing, True):
        _routing_rows(group, "rows", rows, routing, True)
        _check_weights(routing, weights, rows.dtype)
        _on_device(group, rows=rows, weights=weights, routing=routing.offsets)
    if weights is not None:
        _check_weights(routing, weights, rows.dtype)
        if weights.get_device() != group.device:
            _on_device(group, weights=weights)
    if _recording(rows, weights):
        return _Combine.apply(rows, weights, (group, routing))
    return _combine(group, rows, routing.row_of_slot, weights)


def dispatch_backward(group, grad, routing):
    _refuse_tracers()
    if not _fits_rows(group, grad, routing, True):
        _routing_rows(group, "grad", grad, routing, True)
        _on_device(group, grad=grad, routing=routing.offsets)
    _refuse_tangents(grad)
    return _combine(group, grad, routing.row_of_slot)


def combine_backward(group, grad, rows, routing, weights=None):
    _refuse_tracers()
    _routing_rows(group, "rows", rows, routing, True)
    _tensor("grad", grad, (routing.tokens, rows.shape[1]), (rows.dtype,))
    _check_weights(routing, weights, rows.dtype)
    _on_device(group, grad=grad, rows=rows, weights=weights, routing=routing.offsets)
    _refuse_tangents(grad, rows, weights)
    return _combine_backward(group, grad, rows, routing.row_of_slot, routing.offsets, weights, True, weights is not None)


# ---- sum over the ranks, norms, gate, residual -------------------------------------------------------------------

@functools.lru_cache(maxsize=4096)
def _norm_workspace(tokens, dim, code):
    return capi.load_library().lib.sar_reduce_norm_workspace(tokens, dim, code)


def _norm_args(sources, copies, residual, pre_weight, post_weight, gate, residual_scale, eps, partials=None, hidden=None, normed=None,
               total=None, stats=None):
    """sar_reduce_norm_args, by position: dtype, pre_dtype, post_dtype, gate_dtype, gate_kind, sources, copies, reserved, tokens, dim, eps,
    residual_scale, partials, residual, pre_weight, post_weight, gate, hidden, normed, total, stats."""
    tokens, dim = residual.shape
    code = DTYPE_CODES[residual.dtype]
    pre_code = post_code = gate_code = code
    kind, pre, post, gate_ptr = _GATE_NONE, None, None, None
    if pre_weight is not None:
        pre_code, pre = DTYPE_CODES[pre_weight.dtype], pre_weight.data_ptr()
    if post_weight is not None:
        post_code, post = DTYPE_CODES[post_weight.dtype], post_weight.data_ptr()
    if gate is not None:
        gate_code, gate_ptr = DTYPE_CODES[gate.dtype], gate.data_ptr()
        kind = _GATE_CHANNEL if gate.dim() == 1 else _GATE_TOKEN if gate.shape[1] == 1 and dim > 1 else _GATE_FULL
    return capi.ReduceNormArgs(code, pre_code, post_code, gate_code, kind, sources, copies, 0, tokens, dim, eps, residual_scale, partials,
                               residual.data_ptr(), pre, post, gate_ptr, hidden, normed, total, stats)


@functools.lru_cache(maxsize=None)
def _pointers(n):
    return ctypes.c_void_p * n


def _reduce_norm(group, partials, addresses, residual, pre_weight, post_weight, gate, residual_scale, eps, gather, save):
    """`addresses`: of the partials' rows.  Returns hidden, normed (or None), total and stats (or None); one partial is
    its own total."""
    tokens, dim = residual.shape
    sources = len(addresses)
    hidden = torch.empty_like(residual)
    normed = total = stats = None
    if pre_weight is not None:
        normed = residual.new_empty((group.n, tokens, dim) if gather else (tokens, dim))
    if save:
        total = partials if sources == 1 else torch.empty((tokens, dim), dtype=torch.float32, device=residual.device)
        stats = torch.empty((2, tokens), dtype=torch.float32, device=residual.device)
    args = _norm_args(sources, group.n if gather else 1, residual, pre_weight, post_weight, gate, residual_scale, eps,
                      _pointers(sources)(*addresses), hidden.data_ptr(), _ptr(normed),
                      total.data_ptr() if save and sources > 1 else None, _ptr(stats))
    lib = group._lib
    lib.check(lib.lib.sar_reduce_norm(group.device, _raw_stream(group.device), ctypes.byref(args)))
    return hidden, normed, total, stats


def _reduce_norm_backward(group, s: ReduceNormSaved, grad_hidden, grad_normed, want) -> ReduceNormGrads:
    """`want`: truth values for partials, residual, pre_weight, post_weight, gate."""
    residual, pre_weight, post_weight, gate, total = s.residual, s.pre_weight, s.post_weight, s.gate, s.total
    tokens, dim = residual.shape
    args = _norm_args(s.sources, s.copies, residual, pre_weight, post_weight, gate, s.residual_scale, s.eps, stats=s.stats.data_ptr())
    out = ReduceNormGrads(
        residual.new_empty(s.partial_shape) if want[0] else None,
        torch.empty_like(residual) if want[1] else None,
        torch.empty_like(pre_weight) if want[2] and pre_weight is not None else None,
        torch.empty_like(post_weight) if want[3] and post_weight is not None else None,
        torch.empty_like(gate) if want[4] and gate is not None else None)
    lib = group._lib
    need = _norm_workspace(tokens, dim, args.dtype)
    work = torch.empty(need // 4, dtype=torch.float32, device=residual.device) if need else None
    # total, total_dtype, reserved, then the gradients that come in, those that go out, and the workspace
    grads = capi.ReduceNormGrads(total.data_ptr(), DTYPE_CODES[total.dtype], 0, _ptr(grad_hidden), _ptr(grad_normed), _ptr(out[0]), _ptr(out[1]),
                                 _ptr(out[2]), _ptr(out[3]), _ptr(out[4]), _ptr(work), need)
    lib.check(lib.lib.sar_reduce_norm_backward(group.device, _raw_stream(group.device), ctypes.byref(args), ctypes.byref(grads)))
    return out


class _ReduceNorm(_Node):
    @staticmethod
    def forward(ctx, plain, residual, pre_weight, post_weight, gate, *partials):
        group, shape, addresses, residual_scale, eps, gather = plain
        hidden, normed, total, stats = _reduce_norm(group, partials[0], addresses, residual, pre_weight, post_weight, gate, residual_scale, eps,
                                                    gather, True)
        ctx.plain, ctx.hooked = plain, _hooks(True) and residual.dtype
        ctx.save_for_backward(total, stats, residual, pre_weight, post_weight, gate)
        ctx.set_materialize_grads(False)
        return hidden, normed

    @staticmethod
    def gradients(ctx, grad_hidden, grad_normed):
        group, shape, addresses, residual_scale, eps, gather = ctx.plain
        total, stats, residual, pre_weight, post_weight, gate = ctx.saved_tensors
        saved = ReduceNormSaved(len(addresses), group.n if gather else 1, shape, total, stats, residual, pre_weight,
                                post_weight, gate, residual_scale, eps)
        if ctx.hooked and (residual.dtype is not ctx.hooked or residual.shape != shape[-2:] or not _fits_saved(group, saved)):
            raise RuntimeError(_HOOKED)
        need = ctx.needs_input_grad
        g = _reduce_norm_backward(group, saved, grad_hidden.contiguous() if grad_hidden is not None else None,
                                  grad_normed.contiguous() if grad_normed is not None else None, (True in need[5:], need[1], need[2], need[3], need[4]))
        inputs = len(need) - 5
        if inputs == 1:
            return None, g[1], g[2], g[3], g[4], g[0]
        return (None, g[1], g[2], g[3], g[4], *(g[0].unbind(0) if g[0] is not None else (None,) * inputs))

    @staticmethod
    def backward(ctx, grad_hidden, grad_normed):
        return _ReduceNorm._backward(ctx, grad_hidden, grad_normed)


def _check_reduce_norm(group, partials, inputs, residual, pre_weight, post_weight, gate, eps):
    """Says what is wrong with the arguments of reduce_norm."""
    if not isinstance(residual, torch.Tensor) or residual.dim() != 2:
        raise ValueError("residual must be a tensor [tokens, dim]")
    _tensor("residual", residual, dtypes=DTYPE_CODES)
    (tokens, dim), dtype = residual.shape, residual.dtype
    if not 1 <= dim <= MAX_NORM_DIM:
        raise ValueError("dim must be 1 to %d, got %d" % (MAX_NORM_DIM, dim))
    if isinstance(partials, torch.Tensor):
        if partials.dim() not in (2, 3) or partials.shape[-2:] != residual.shape or (partials.dim() == 3 and partials.shape[0] != group.n):
            raise ValueError("partials must be [%d ranks, tokens, dim] or, as a finished output, [tokens, dim]: got %s with residual %s"
                             % (group.n, tuple(partials.shape), tuple(residual.shape)))
        _tensor("partials", partials, dtypes=(dtype,))
    else:
        if len(inputs) != group.n:
            raise ValueError("need one partial output per emulated rank: %d, got %d" % (group.n, len(inputs)))
        for p in inputs:
            _tensor("a partial output", p, residual.shape, (dtype,))
    kinds = (torch.float32, dtype)
    if pre_weight is not None:
        _tensor("pre_weight", pre_weight, (dim,), kinds)
    if post_weight is not None:
        _tensor("post_weight", post_weight, (dim,), kinds)
    if gate is not None:
        _tensor("gate", gate, dtypes=kinds)
        if tuple(gate.shape) not in ((dim,), (tokens, 1), (tokens, dim)):
            raise ValueError("gate must be [dim], [tokens, 1] or [tokens, dim]: got %s" % (tuple(gate.shape),))
    if not 0 <= eps < float("inf"):
        raise ValueError("eps must be a finite number, zero or more")
    for t in (residual, pre_weight, post_weight, gate, *inputs):
        if t is not None and t.get_device() != group.device:
            raise ValueError("every tensor must be a CUDA tensor on device %d" % group.device)


def _fits_reduce_norm(group, partials, inputs, residual, pre_weight, post_weight, gate, eps):
    """The checks above in as little time as they take: the addresses of the partials' rows, or None."""
    if not isinstance(residual, torch.Tensor) or residual.dim() != 2:
        return None
    size, dtype, device = residual.shape, residual.dtype, group.device
    tokens, dim = size
    if dtype not in DTYPE_CODES or not 1 <= dim <= MAX_NORM_DIM or not residual.is_contiguous() or residual.get_device() != device or not 0 <= eps < float("inf"):
        return None
    whole = partials is inputs[0] and partials.dim() == 3
    if whole:
        size = (group.n, tokens, dim)
    elif partials is not inputs[0] and len(inputs) != group.n:
        return None
    addresses = []
    for p in inputs:
        if not isinstance(p, torch.Tensor) or p.dtype is not dtype or p.shape != size or not p.is_contiguous() or p.get_device() != device:
            return None
        addresses.append(p.data_ptr())
    if whole:
        addresses = [addresses[0] + r * tokens * dim * residual.element_size() for r in range(group.n)]
    for w in (pre_weight, post_weight):
        if w is not None and (not isinstance(w, torch.Tensor) or w.dim() != 1 or w.shape[0] != dim or not w.is_contiguous() or w.get_device() != device
                              or (w.dtype is not dtype and w.dtype is not torch.float32)):
            return None
    if gate is not None and not (isinstance(gate, torch.Tensor) and gate.is_contiguous() and gate.get_device() == device
                                 and (gate.dtype is dtype or gate.dtype is torch.float32) and tuple(gate.shape) in ((dim,), (tokens, 1), (tokens, dim))):
        return None
    return addresses


def reduce_norm(group, partials: Union[torch.Tensor, Sequence[torch.Tensor]], residual, pre_weight=None, post_weight=None, gate=None,
                residual_scale: float = 1.0, eps: float = 1e-6, gather: bool = True, save: bool = False):
    _refuse_tracers()
    if isinstance(residual_scale, torch.Tensor) or isinstance(eps, torch.Tensor):
        raise TypeError("residual_scale and eps are numbers: a tensor's value would be waited for, and get no gradient")
    inputs = (partials,) if isinstance(partials, torch.Tensor) else tuple(partials)
    addresses = _fits_reduce_norm(group, partials, inputs, residual, pre_weight, post_weight, gate, eps) if inputs else None
    if addresses is None:
        _check_reduce_norm(group, partials, inputs, residual, pre_weight, post_weight, gate, eps)
        raise ValueError("the arguments do not fit each other")
    shape = tuple(partials.shape) if inputs[0] is partials else (group.n, *residual.shape)
    if _recording(residual, pre_weight, post_weight, gate, *inputs):
        if save:
            raise ValueError("save=True is for calls under torch.no_grad(): autograd keeps what it needs by itself")
        return _ReduceNorm.apply((group, shape, addresses, residual_scale, eps, gather), residual, pre_weight, post_weight, gate, *inputs)
    hidden, normed, total, stats = _reduce_norm(group, inputs[0], addresses, residual, pre_weight, post_weight, gate, residual_scale, eps, gather, save)
    if not save:
        return hidden, normed
    return hidden, normed, ReduceNormSaved(len(addresses), group.n if gather else 1, shape, total, stats, residual, pre_weight, post_weight, gate,
                                           residual_scale, eps)


def _fits_parameter(t, kinds, dim, device):
    return t is None or (isinstance(t, torch.Tensor) and t.dtype in kinds and t.shape == (dim,) and t.get_device() == device and t.is_contiguous())


def _fits_saved(group, s: ReduceNormSaved):
    """The checks below and of the devices in as little time as they take."""
    residual, total, stats, gate = s.residual, s.total, s.stats, s.gate
    if not isinstance(residual, torch.Tensor) or not isinstance(total, torch.Tensor) or not isinstance(stats, torch.Tensor):
        return False
    size, dtype, device = residual.shape, residual.dtype, group.device
    if len(size) != 2 or dtype not in DTYPE_CODES:
        return False
    tokens, dim = size
    kinds, shape = (torch.float32, dtype), tuple(s.partial_shape)
    return ((shape == (s.sources, tokens, dim) or (s.sources == 1 and shape == size)) and residual.get_device() == device and residual.is_contiguous()
            and total.shape == size and total.dtype in kinds and total.get_device() == device and total.is_contiguous()
            and stats.shape == (2, tokens) and stats.dtype is torch.float32 and stats.get_device() == device and stats.is_contiguous()
            and _fits_parameter(s.pre_weight, kinds, dim, device) and _fits_parameter(s.post_weight, kinds, dim, device)
            and (gate is None or (isinstance(gate, torch.Tensor) and gate.dtype in kinds and tuple(gate.shape) in ((dim,), (tokens, 1), (tokens, dim))
                                  and gate.get_device() == device and gate.is_contiguous())))


def _check_saved(s: ReduceNormSaved):
    """Says what is wrong with a saved call: the kernels take its sizes from its residual."""
    residual = s.residual
    if not isinstance(residual, torch.Tensor) or residual.dim() != 2:
        raise ValueError("saved.residual must be a tensor [tokens, dim]")
    _tensor("saved.residual", residual, dtypes=DTYPE_CODES)
    (tokens, dim), dtype = residual.shape, residual.dtype
    kinds = (torch.float32, dtype)
    _tensor("saved.total", s.total, (tokens, dim), kinds)
    _tensor("saved.stats", s.stats, (2, tokens), (torch.float32,))
    shape = tuple(s.partial_shape)
    if shape != (s.sources, tokens, dim) and not (s.sources == 1 and shape == (tokens, dim)):
        raise ValueError("saved.partial_shape is %s with %s sources of %s" % (shape, s.sources, (tokens, dim)))
    if s.pre_weight is not None:
        _tensor("saved.pre_weight", s.pre_weight, (dim,), kinds)
    if s.post_weight is not None:
        _tensor("saved.post_weight", s.post_weight, (dim,), kinds)
    if s.gate is not None:
        _tensor("saved.gate", s.gate, dtypes=kinds)
        if tuple(s.gate.shape) not in ((dim,), (tokens, 1), (tokens, dim)):
            raise ValueError("saved.gate must be [dim], [tokens, 1] or [tokens, dim]: got %s" % (tuple(s.gate.shape),))


def _fits_grads(group, s: ReduceNormSaved, grad_hidden, grad_normed):
    """The checks below of the gradients."""
    size, dtype, device = s.residual.shape, s.residual.dtype, group.device
    if grad_hidden is not None and not (isinstance(grad_hidden, torch.Tensor) and grad_hidden.shape == size and grad_hidden.dtype is dtype
                                        and grad_hidden.get_device() == device and grad_hidden.is_contiguous()):
        return False
    return grad_normed is None or (
        s.pre_weight is not None and isinstance(grad_normed, torch.Tensor) and grad_normed.dtype is dtype and grad_normed.get_device() == device
        and grad_normed.is_contiguous() and (grad_normed.shape == (s.copies, *size) or (s.copies == 1 and grad_normed.shape == size)))


def _check_reduce_norm_backward(group, saved, grad_hidden, grad_normed):
    """Says what is wrong with the arguments of reduce_norm_backward."""
    _check_saved(saved)
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
    _on_device(group, grad_hidden=grad_hidden, grad_normed=grad_normed, residual=saved.residual, total=saved.total, stats=saved.stats,
               pre_weight=saved.pre_weight, post_weight=saved.post_weight, gate=saved.gate)
    raise ValueError("the arguments do not fit each other")


def reduce_norm_backward(group, saved: ReduceNormSaved, grad_hidden=None, grad_normed=None) -> ReduceNormGrads:
    _refuse_tracers()
    if not isinstance(saved, ReduceNormSaved):
        raise TypeError("saved must come from reduce_norm(..., save=True)")
    if not _fits_saved(group, saved) or not _fits_grads(group, saved, grad_hidden, grad_normed):
        _check_reduce_norm_backward(group, saved, grad_hidden, grad_normed)
    _refuse_tangents(grad_hidden, grad_normed, saved.total, saved.residual, saved.pre_weight, saved.post_weight, saved.gate)
    return _reduce_norm_backward(group, saved, grad_hidden, grad_normed, (True,) * 5)
