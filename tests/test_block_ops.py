"""Refusals of the block operators (routing, dispatch, combine, reduce_norm): none of them needs a device, every one is
said before anything is launched."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from stragglar_amd import block_ops, capi  # noqa: E402
from stragglar_amd.torch_emulation import EmulatedGroup  # noqa: E402


@pytest.fixture()
def group(sarlib):
    """A group without a context: the argument checks run before the device is touched."""
    g = object.__new__(EmulatedGroup)
    g.n, g.device, g._lib = 4, 0, sarlib
    return g


def routing(tokens=3, topk=2, experts=8):
    return block_ops.Routing(torch.zeros(tokens, topk, dtype=torch.int32), torch.zeros(tokens * topk, dtype=torch.int32),
                             torch.zeros(experts + 1, dtype=torch.int32), experts, 4)


def test_route_refuses(group):
    ids = torch.zeros(3, 2, dtype=torch.int64)
    for bad, experts, why in [(ids.float(), 8, "dtype"), (ids.view(-1), 8, "tokens, topk"), (ids, 7, "multiple"), (ids, 0, "multiple"),
                              (ids, 1028, "multiple"), (torch.zeros(3, 0, dtype=torch.int64), 8, "topk"),
                              (torch.zeros(1, 65, dtype=torch.int32), 8, "topk"), (ids.t(), 8, "contiguous"), (ids, 8, "CUDA"),
                              ([[0]], 8, "tokens, topk"), (torch.zeros(1, 1, dtype=torch.int64).expand(1 << 30, 2), 8, "contiguous")]:
        with pytest.raises((ValueError, TypeError), match=why):
            group.route(bad, experts)


def test_routing_refuses():
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32)
    for args in [(i(6), i(6), i(9), 8, 4), (i(3, 2), i(5), i(9), 8, 4), (i(3, 2), i(6), i(8), 8, 4), (i(3, 2), i(6), i(9), 8, 3),
                 (i(3, 2).long(), i(6), i(9), 8, 4), (i(2, 3).t(), i(6), i(9), 8, 4), (i(3, 2), i(6), i(9).float(), 8, 4)]:
        with pytest.raises(ValueError):
            block_ops.Routing(*args)
    r = block_ops.Routing(i(3, 2), i(6), torch.arange(9, dtype=torch.int32), 8, 4)
    assert (r.tokens, r.topk) == (3, 2) and r.rank_offsets.tolist() == [0, 2, 4, 6, 8]


def test_dispatch_and_combine_refuse(group):
    r = routing()
    for call, why in [(lambda: group.dispatch(torch.zeros(4, 8), r), "tokens must be"),
                      (lambda: group.dispatch(torch.zeros(3, 8, dtype=torch.float64), r), "dtype"),
                      (lambda: group.dispatch(torch.zeros(3, 0), r), "columns"),
                      (lambda: group.dispatch(torch.zeros(8, 3).t(), r), "must be|contiguous"),
                      (lambda: group.dispatch(torch.zeros(3, 8), (1, 2, 3)), "routing"),
                      (lambda: group.dispatch(torch.zeros(3, 8), r), "CUDA"),
                      (lambda: group.combine(torch.zeros(5, 8), r), "rows must be"),
                      (lambda: group.combine(torch.zeros(6, 8), r, torch.zeros(2, 3)), "weights has shape"),
                      (lambda: group.combine(torch.zeros(6, 8), r, torch.zeros(3, 2).half()), "weights has dtype"),
                      (lambda: group.combine(torch.zeros(6, 8).bfloat16(), r, torch.zeros(3, 2).half()), "weights has dtype"),
                      (lambda: group.combine(torch.zeros(6, 8), r, torch.zeros(2, 3).t()), "contiguous"),
                      (lambda: group.combine(torch.zeros(6, 8), r, torch.zeros(3, 2)), "CUDA"),
                      (lambda: group.dispatch_backward(torch.zeros(3, 8), r), "grad must be"),
                      (lambda: group.combine_backward(torch.zeros(3, 7), torch.zeros(6, 8), r), "grad has shape"),
                      (lambda: group.combine_backward(torch.zeros(3, 8).half(), torch.zeros(6, 8), r), "grad has dtype")]:
        with pytest.raises((ValueError, TypeError), match=why):
            call()


def test_reduce_norm_refuses(group):
    t, d = 3, 8
    x, w = torch.zeros(t, d), torch.ones(d)
    for call, why in [(lambda: group.reduce_norm([x] * 3, x, w), "per emulated rank"),
                      (lambda: group.reduce_norm([x] * 3 + [x[:2]], x, w), "shape"),
                      (lambda: group.reduce_norm([x] * 3 + [x.half()], x, w), "dtype"),
                      (lambda: group.reduce_norm(torch.zeros(3, t, d), x, w), "partials must be"),
                      (lambda: group.reduce_norm(torch.zeros(t, d + 1), x, w), "partials must be"),
                      (lambda: group.reduce_norm(x, x.double(), w), "dtype"),
                      (lambda: group.reduce_norm(x, x.view(-1), w), "residual must be"),
                      (lambda: group.reduce_norm(x, x, w[:4]), "pre_weight has shape"),
                      (lambda: group.reduce_norm(x, x, w.half()), "pre_weight has dtype"),
                      (lambda: group.reduce_norm(x, x, w, post_weight=torch.ones(1, d)), "post_weight has shape"),
                      (lambda: group.reduce_norm(x, x, w, gate=torch.ones(1, d)), "gate must be"),
                      (lambda: group.reduce_norm(x, x, w, gate=torch.ones(t)), "gate must be"),
                      (lambda: group.reduce_norm(x, x, w, gate=torch.ones(1, d).expand(t, d)), "contiguous"),
                      (lambda: group.reduce_norm(x, x, w, eps=-1.0), "eps"),
                      (lambda: group.reduce_norm(x, x, w, eps=float("nan")), "eps"),
                      (lambda: group.reduce_norm(torch.zeros(1, 16385), torch.zeros(1, 16385)), "dim must be"),
                      (lambda: group.reduce_norm(torch.zeros(1, 0), torch.zeros(1, 0)), "dim must be"),
                      (lambda: group.reduce_norm(x, x, w), "CUDA")]:
        with pytest.raises((ValueError, TypeError), match=why):
            call()


def test_reduce_norm_backward_refuses(group):
    x = torch.zeros(3, 8)
    saved = block_ops.ReduceNormSaved(1, 4, (3, 8), x, torch.zeros(2, 3), x, torch.ones(8), None, None, 1.0, 1e-6)
    for call, why in [(lambda: group.reduce_norm_backward((1, 2)), "saved"),
                      (lambda: group.reduce_norm_backward(saved, torch.zeros(3, 7)), "grad_hidden has shape"),
                      (lambda: group.reduce_norm_backward(saved, None, torch.zeros(3, 8)), "grad_normed has shape"),
                      (lambda: group.reduce_norm_backward(saved, None, torch.zeros(4, 3, 8).half()), "dtype"),
                      (lambda: group.reduce_norm_backward(saved._replace(pre_weight=None), None, torch.zeros(4, 3, 8)), "without a pre_weight"),
                      (lambda: group.reduce_norm_backward(saved, x, None), "CUDA")]:
        with pytest.raises((ValueError, TypeError), match=why):
            call()


def test_a_capturing_stream_refuses_autograd(monkeypatch):
    """Neither the recording nor the backward pass of a recorded call goes into a capture; without gradients the check
    is not even made."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    x = torch.zeros(2, 2, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        block_ops._recording(None, x)
    with torch.no_grad():
        assert not block_ops._recording(x)
    assert not block_ops._recording(x.detach(), None)
    for node in (block_ops._Dispatch, block_ops._Combine, block_ops._ReduceNorm):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            node._backward(None, x)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert block_ops._recording(x)


def refused(lib, rc, why):
    assert rc == -1 and why in lib.lib.sar_last_error().decode(), (rc, lib.lib.sar_last_error())


def test_c_entries_refuse(sarlib):
    """The C entry points say SAR_EINVAL before they look for a device (addresses here are never used)."""
    L, p, odd = sarlib.lib, 0x10000, 0x10001
    big = 1 << 40
    route = lambda **k: L.sar_route(0, None, *[{**dict(experts=p, ib=8, t=4, k=2, e=8, r=p, s=p, o=p, w=None, wb=0), **k}[n]
                                               for n in ("experts", "ib", "t", "k", "e", "r", "s", "o", "w", "wb")])
    for k, why in [(dict(ib=2), "index_bytes"), (dict(t=-1), "negative"), (dict(k=0), "topk"), (dict(k=65), "topk"), (dict(e=0), "num_experts"),
                   (dict(e=1025), "num_experts"), (dict(t=1 << 30), "2^31"), (dict(o=None), "offsets"), (dict(experts=None), "null"),
                   (dict(experts=p + 4), "aligned"), (dict(r=odd), "aligned"), (dict(t=8192), "workspace"),
                   (dict(t=8192, w=p, wb=8), "workspace")]:
        refused(sarlib, route(**k), why)
    assert L.sar_route_workspace(16, 8, 64) == 0 and L.sar_route_workspace(8192, 2, 8) == (4 + 1) * 8 * 4 and L.sar_route_workspace(-1, 2, 8) == 0

    dispatch = lambda **k: L.sar_dispatch(0, None, *[{**dict(dt=0, x=p, t=4, k=2, d=8, r=p, o=p, e=8, w=None, wd=0, out=p), **k}[n]
                                                     for n in ("dt", "x", "t", "k", "d", "r", "o", "e", "w", "wd", "out")])
    combine = lambda **k: L.sar_combine(0, None, *[{**dict(dt=0, x=p, t=4, k=2, d=8, r=p, w=None, wd=0, out=p), **k}[n]
                                                   for n in ("dt", "x", "t", "k", "d", "r", "w", "wd", "out")])
    back = lambda **k: L.sar_combine_backward(0, None, *[{**dict(dt=0, g=p, x=p, t=4, k=2, d=8, r=p, o=p, e=8, w=p, wd=0, gr=p, gw=p), **k}[n]
                                                         for n in ("dt", "g", "x", "t", "k", "d", "r", "o", "e", "w", "wd", "gr", "gw")])
    for call in (dispatch, combine, back):
        for k, why in [(dict(dt=3), "dtype"), (dict(t=-1), "negative"), (dict(k=0), "topk"), (dict(k=65), "topk"), (dict(d=0), "dim"),
                       (dict(d=big), "dim"), (dict(t=1 << 30), "2^31"), (dict(r=None), "row_of_slot"), (dict(r=odd), "row_of_slot"),
                       (dict(w=p, wd=1), "weights"), (dict(w=odd, wd=0), "weights"), (dict(x=None), "null"), (dict(x=odd), "aligned")]:
            refused(sarlib, call(**k), why)
        assert call(t=0) == 0
    for call in (dispatch, combine):
        refused(sarlib, call(out=None), "null")
    refused(sarlib, dispatch(e=0), "num_experts")
    refused(sarlib, dispatch(o=None), "null")
    for k in (dict(g=None), dict(w=None), dict(gw=None), dict(o=None)):
        refused(sarlib, back(**k), "null")

    def norm(backward=False, grads=None, **k):
        a = capi.ReduceNormArgs(dtype=0, sources=1, copies=1, tokens=4, dim=8, eps=1e-6, residual_scale=1.0, residual=p, hidden=p)
        a.partials = (ctypes.c_void_p * 1)(p)
        for n, v in k.items():
            setattr(a, n, v)
        if not backward:
            return L.sar_reduce_norm(0, None, ctypes.byref(a))
        g = capi.ReduceNormGrads(total=p, grad_hidden=p, grad_partials=p, workspace=p, workspace_bytes=1 << 30)
        for n, v in (grads or {}).items():
            setattr(g, n, v)
        a.stats = k.get("stats", p)
        return L.sar_reduce_norm_backward(0, None, ctypes.byref(a), ctypes.byref(g))

    both = [(dict(dtype=3), "dtype"), (dict(tokens=-1), "negative"), (dict(tokens=1 << 41), "many"), (dict(dim=0), "dim"), (dict(dim=16385), "dim"),
            (dict(sources=0), "sources"), (dict(sources=65), "sources"), (dict(copies=0), "copies"), (dict(copies=65), "copies"),
            (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
            (dict(pre_weight=p, pre_dtype=1), "pre_weight"), (dict(post_weight=p, post_dtype=2), "post_weight"), (dict(gate_kind=4), "gate kind"),
            (dict(gate_kind=1), "gate is null"), (dict(gate_kind=1, gate=p, gate_dtype=1), "gate must"), (dict(residual=None), "residual"),
            (dict(residual=odd), "aligned"), (dict(post_weight=odd), "aligned")]
    for k, why in both:
        refused(sarlib, norm(**k), why)
        refused(sarlib, norm(backward=True, **k), why)
    refused(sarlib, norm(pre_weight=p), "go together")
    refused(sarlib, norm(normed=p), "go together")
    refused(sarlib, norm(partials=None), "partials")
    refused(sarlib, norm(sources=1, partials=(ctypes.c_void_p * 1)(None)), "partial")
    refused(sarlib, norm(total=odd), "aligned")
    refused(sarlib, L.sar_reduce_norm(0, None, None), "null")
    assert norm(tokens=0) == 0
    for g, why in [(dict(grad_normed=p), "without pre_weight"), (dict(grad_pre_weight=p), "without pre_weight"), (dict(grad_post_weight=p), "without post_weight"),
                   (dict(grad_gate=p), "without a gate"), (dict(total=None), "null"), (dict(total_dtype=2), "total"), (dict(workspace=None), "workspace"),
                   (dict(workspace_bytes=16), "workspace"), (dict(grad_hidden=odd), "aligned")]:
        refused(sarlib, norm(backward=True, grads=g, tokens=100), why)
    refused(sarlib, norm(backward=True, stats=None), "null")
    assert L.sar_reduce_norm_workspace(100, 8, 0) >= 3 * 8 * 4 and L.sar_reduce_norm_workspace(1, 8, 0) == 0 and L.sar_reduce_norm_workspace(4, 0, 0) == 0


def test_struct_sizes_follow_the_header(tmp_path):
    """The ctypes structures against what a C compiler makes of the header."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "sar.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", sizeof(sar_reduce_norm_args), '
                   'offsetof(sar_reduce_norm_args, stats), sizeof(sar_reduce_norm_grads), offsetof(sar_reduce_norm_grads, workspace_bytes)); return 0; }\n')
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(capi.ReduceNormArgs), capi.ReduceNormArgs.stats.offset,
                   ctypes.sizeof(capi.ReduceNormGrads), capi.ReduceNormGrads.workspace_bytes.offset]


# ---- calls that get past the checks: on the CPU, with nothing behind the C entries ---------------------------------

@pytest.fixture()
def recorder(monkeypatch):
    """A group whose tensors lie on the CPU and whose C entries only note their names in `calls`."""
    class Entries:
        def __getattr__(self, name):
            return lambda *args: g.calls.append(name) or 0

    class Lib:
        lib = Entries()

        def check(self, rc):
            assert rc == 0
    g = object.__new__(EmulatedGroup)
    g.n, g.device, g._lib, g.calls = 4, -1, Lib(), []
    monkeypatch.setattr(block_ops, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return g


def test_a_routing_written_again_is_noticed_by_the_backward_pass(recorder):
    g = recorder
    for field in ("row_of_slot", "offsets"):
        r = routing()
        x, rows = torch.zeros(3, 8, requires_grad=True), torch.zeros(6, 8, requires_grad=True)
        w = torch.zeros(3, 2, requires_grad=True)
        outs = [(g.combine(rows, r, w), (rows, w)), (g.combine(rows, r), (rows,))]
        if field == "row_of_slot":                        # (what dispatch's gradient reads)
            outs.append((g.dispatch(x, r), (x,)))
        getattr(r, field).copy_(torch.ones_like(getattr(r, field)))
        g.calls.clear()
        for out, leaves in outs:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(out.sum(), leaves)
        assert not g.calls
    r = routing()                                          # left alone, it is what the backward pass gets
    torch.autograd.grad(g.combine(rows, r, w).sum(), (rows, w))
    assert g.calls == ["sar_combine", "sar_combine_backward"]


def test_a_routing_made_in_inference_mode_takes_part_in_autograd(recorder):
    with torch.inference_mode():
        r = routing()
    x, rows = torch.zeros(3, 8, requires_grad=True), torch.zeros(6, 8, requires_grad=True)
    assert torch.autograd.grad(recorder.dispatch(x, r).sum(), x)[0].shape == (3, 8)
    assert torch.autograd.grad(recorder.combine(rows, r).sum(), rows)[0].shape == (6, 8)


def every_call(g, r, make=lambda t: t):
    """One call of each kind per floating-point input, that input passed through `make`: (name, call)."""
    t, k, d = 3, 2, 8
    z = lambda *shape: torch.zeros(*shape)
    yield "dispatch", lambda: g.dispatch(make(z(t, d)), r)
    yield "combine rows", lambda: g.combine(make(z(t * k, d)), r, z(t, k))
    yield "combine rows alone", lambda: g.combine(make(z(t * k, d)), r)
    yield "combine weights", lambda: g.combine(z(t * k, d), r, make(z(t, k)))
    yield "dispatch_backward", lambda: g.dispatch_backward(make(z(t * k, d)), r)
    yield "combine_backward grad", lambda: g.combine_backward(make(z(t, d)), z(t * k, d), r, z(t, k))
    yield "combine_backward rows", lambda: g.combine_backward(z(t, d), make(z(t * k, d)), r, z(t, k))
    yield "combine_backward weights", lambda: g.combine_backward(z(t, d), z(t * k, d), r, make(z(t, k)))
    args = dict(partials=lambda: z(t, d), residual=lambda: z(t, d), pre_weight=lambda: z(d), post_weight=lambda: z(d), gate=lambda: z(t, 1))
    for name in args:
        yield "reduce_norm " + name, lambda name=name: g.reduce_norm(**{n: make(f()) if n == name else f() for n, f in args.items()})
    yield "reduce_norm one of the partials", lambda: g.reduce_norm([z(t, d), z(t, d), make(z(t, d)), z(t, d)], z(t, d), z(d))
    saved = block_ops.ReduceNormSaved(1, 4, (t, d), z(t, d), z(2, t), z(t, d), z(d), z(d), z(t, 1), 1.0, 1e-6)
    yield "reduce_norm_backward hidden", lambda: g.reduce_norm_backward(saved, make(z(t, d)), None)
    yield "reduce_norm_backward normed", lambda: g.reduce_norm_backward(saved, None, make(z(4, t, d)))


def test_tangents_are_refused(recorder):
    """Forward-mode derivatives: an output without a tangent would be a derivative of zero."""
    from torch.autograd import forward_ad
    g, r = recorder, routing()
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for grad in (True, False):                           # no_grad does not switch them off
            for name, call in every_call(g, r, dual):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
                    pytest.fail(name)
        with pytest.raises(NotImplementedError):
            g.dispatch(dual(torch.zeros(3, 8)).requires_grad_(True), r)
        assert not g.calls
        for name, call in every_call(g, r):                  # a level alone changes nothing
            call()
        with torch.inference_mode():                         # nobody asks for derivatives
            g.dispatch(dual(torch.zeros(3, 8)), r)
    assert len(g.calls) == len(list(every_call(g, r))) + 1


def test_tracers_are_refused(recorder):
    """A recorder of torch's operations would keep the allocation of the outputs and none of the kernels."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    g, r, x = recorder, routing(), torch.zeros(3, 8)
    ids = torch.zeros(3, 2, dtype=torch.int64)
    calls = list(every_call(g, r)) + [("route", lambda: g.route(ids, 8))]

    def also(call):
        def f(t):
            call()
            return t + 1
        return f
    for name, call in calls:
        for how in (lambda f: make_fx(f)(x), lambda f: make_fx(f, pre_dispatch=True)(x), lambda f: make_fx(f, tracing_mode="symbolic")(x),
                    lambda f: torch.jit.trace(f, x, check_trace=False), lambda f: torch.func.functionalize(f)(x),
                    lambda f: torch.func.functionalize(torch.vmap(f))(x)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                how(also(call))
                pytest.fail(name)
        with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(RuntimeError, match="cannot be traced"):
            call()
    leaf = x.clone().requires_grad_(True)
    out = g.dispatch(leaf, r)
    g.calls.clear()
    with pytest.raises(RuntimeError, match="cannot be traced"):       # the backward pass of a call made before
        make_fx(lambda t: torch.autograd.grad(out, leaf, t)[0])(torch.zeros(6, 8))
    assert not g.calls


def test_a_mode_that_watches_changes_nothing(recorder):
    from torch.utils.flop_counter import FlopCounterMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    g, r = recorder, routing()
    leaf = torch.zeros(3, 8, requires_grad=True)
    for mode in (FlopCounterMode(display=False), Log()):
        with mode:
            assert torch.autograd.grad(g.dispatch(leaf, r).sum(), leaf)[0].shape == (3, 8)
    assert g.calls == ["sar_dispatch", "sar_combine"] * 2


def test_combine_keeps_its_rows_for_the_gradient_of_weights_alone(recorder):
    g, r = recorder, routing()
    leaf = torch.zeros(6, 8, requires_grad=True)
    for weights, kept in [(None, False), (torch.zeros(3, 2), False), (torch.zeros(3, 2, requires_grad=True), True)]:
        rows = leaf.clone()
        out = g.combine(rows, r, weights)
        address = rows.data_ptr()
        assert (address in [t.data_ptr() for t in out.grad_fn.saved_tensors if t is not None]) == kept
        rows.add_(1)                                       # in place: only the gradient that reads the rows minds
        if kept:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(out.sum(), leaf)
        else:
            g.calls.clear()
            assert torch.autograd.grad(out.sum(), leaf)[0].shape == (6, 8)
            assert g.calls == ["sar_dispatch"]


def test_a_saved_call_is_checked_part_by_part(recorder):
    """The kernels take a saved call's sizes from its residual: parts that do not fit it would be read past their ends."""
    g, t, d = recorder, 3, 8
    z = torch.zeros
    saved = block_ops.ReduceNormSaved(4, 4, (4, t, d), z(t, d), z(2, t), z(t, d).half(), z(d), z(d).half(), z(t, 1), 1.0, 1e-6)
    grad = z(t, d).half()
    assert g.reduce_norm_backward(saved, grad).partials.shape == (4, t, d) and g.calls == ["sar_reduce_norm_backward"]
    one = saved._replace(sources=1, partial_shape=(t, d), total=z(t, d).half())
    assert g.reduce_norm_backward(one, grad).partials.shape == (t, d)
    g.calls.clear()
    for part in [dict(total=z(t - 1, d)), dict(total=z(t, d).double()), dict(total=z(d, t).t()), dict(total=None), dict(stats=z(2, t - 1)), dict(stats=z(2, t).half()),
                 dict(stats=z(t, 2).t()), dict(residual=z(t * d).half()), dict(residual=None), dict(residual=z(t + 1, d).half()), dict(partial_shape=(3, t, d)),
                 dict(partial_shape=(t, d)), dict(partial_shape=()), dict(sources=5), dict(pre_weight=z(d - 1)), dict(pre_weight=z(d).double()),
                 dict(post_weight=z(2 * d)[::2]), dict(gate=z(t)), dict(gate=z(t, 1).double()), dict(gate=z(1, d))]:
        with pytest.raises((ValueError, TypeError), match=list(part)[0] if "residual" not in part and "sources" not in part else "saved"):
            g.reduce_norm_backward(saved._replace(**part), grad)
            pytest.fail(str(part))
    g.device = 0
    with pytest.raises(ValueError, match="CUDA"):
        g.reduce_norm_backward(saved)
    assert not g.calls


def test_what_saved_tensor_hooks_give_back_is_checked(recorder):
    """Hooks may move saved tensors away and bring them back; what comes back in another type, size or order is refused
    before a kernel reads it as what it was."""
    g, r, z = recorder, routing(), torch.zeros
    x, rows, w = z(3, 8, requires_grad=True), z(6, 8, requires_grad=True), z(3, 2, requires_grad=True)
    d = z(8, requires_grad=True)
    calls = [("sar_combine", lambda: g.dispatch(x, r), x), ("sar_dispatch", lambda: g.combine(rows, r), rows), ("sar_dispatch", lambda: g.combine(rows, r, w.detach()), rows),
             ("sar_combine_backward", lambda: g.combine(rows, r, w), w), ("sar_reduce_norm_backward", lambda: g.reduce_norm([x] * 4, x, d, d, d)[0], d)]
    bad = [lambda t: t.to(torch.float16), lambda t: t[:-1], lambda t: t.unsqueeze(0), lambda t: torch.stack([t, t], -1)[..., 0]]
    for entry, call, leaf in calls:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.numpy(force=True).copy(), torch.from_numpy):
            out = call()
            g.calls.clear()
            torch.autograd.grad(out.sum(), leaf)
        assert g.calls == [entry]
        for change in bad:
            at = 0                                       # each saved tensor in turn
            while True:
                seen = []

                def unpack(t):
                    seen.append(t)
                    return change(t) if len(seen) == at + 1 else t
                with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
                    out = call()
                if at == sum(t is not None for t in out.grad_fn.saved_tensors):
                    break
                g.calls.clear(), seen.clear()
                with pytest.raises(RuntimeError, match="saved-tensor hook"):
                    torch.autograd.grad(out.sum(), leaf)
                assert not g.calls, (entry, at)
                at += 1


def test_scale_and_eps_are_numbers(recorder):
    """A tensor would be turned into a number behind autograd's back, its gradient lost."""
    x, learned = torch.zeros(3, 8), torch.tensor(0.5, requires_grad=True)
    for bad in (learned, learned.detach()):
        with pytest.raises(TypeError, match="numbers"):
            recorder.reduce_norm(x, x, residual_scale=bad)
        with pytest.raises(TypeError, match="numbers"):
            recorder.reduce_norm(x, x, eps=bad)
    assert not recorder.calls
    for scale, eps in ((1, 0), (0.5, 1e-6), (-0.25, 1e-5)):
        recorder.reduce_norm(x, x, residual_scale=scale, eps=eps)


def test_the_capture_check_asks_the_tensors_own_device(monkeypatch):
    """With another device current it is the stream of the tensors' device that counts, in either direction."""
    import contextlib
    now = [0]

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], d
        yield
        now[0] = before

    class Leaf:
        requires_grad = True

        def __init__(self, device):
            self.device_index = device

        def get_device(self):
            return self.device_index
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == 1)
    with pytest.raises(RuntimeError, match="captured"):
        block_ops._recording(None, Leaf(1))
    assert block_ops._recording(Leaf(0)) and now == [0]
    now[0] = 1
    assert block_ops._recording(Leaf(0)) and now == [1]


def test_the_parts_of_a_routing_stay(recorder):
    """They are checked when a routing is made and believed afterwards."""
    import copy
    import pickle
    r = routing()
    for name, value in [("row_of_slot", torch.zeros(2, 3, dtype=torch.int32).t()), ("row_of_slot", r.row_of_slot.long()), ("offsets", r.offsets[:3]),
                        ("num_experts", 1 << 20), ("ranks", 0)]:
        with pytest.raises(AttributeError, match="make another"):
            setattr(r, name, value)
    for again in (copy.copy(r), copy.deepcopy(r), pickle.loads(pickle.dumps(r)), recorder.route(torch.zeros(3, 2, dtype=torch.int64), 8)):
        assert isinstance(again, block_ops.Routing) and again.row_of_slot.shape == (3, 2) and (again.num_experts, again.ranks, again.tokens) == (8, 4, 3)
        assert again.rank_offsets.shape == (5,)
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32)
    for experts, ranks in [(8, 0), (8, -4), (0, 4)]:
        with pytest.raises(ValueError):
            block_ops.Routing(i(3, 2), i(6), i(experts + 1), experts, ranks)


def test_the_backward_pass_of_no_tokens_wants_its_channel_gate(sarlib):
    """The kernel runs even then and reads the gate's `dim` elements: a null pointer has to end on the host."""
    p = 0x10000
    a = capi.ReduceNormArgs(dtype=0, sources=1, copies=1, tokens=0, dim=8, eps=1e-6, residual_scale=1.0, gate_kind=1, post_weight=p)
    g = capi.ReduceNormGrads(total_dtype=0, grad_post_weight=p)
    refused(sarlib, sarlib.lib.sar_reduce_norm_backward(0, None, ctypes.byref(a), ctypes.byref(g)), "gate is null")
