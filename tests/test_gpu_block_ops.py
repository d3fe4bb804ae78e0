"""The block operators of an emulated group on the GPU against plain implementations in 64 bits.

Tolerances follow from the arithmetic: `B` carries a value and a bound on what 32-bit operations in the kernels' order
of magnitude can have added to it (each operation rounds by at most 2^-24 of its result; a sum over `depth` additions in
a row by depth * 2^-24 of the sum of magnitudes), and a result is then rounded once to its type by at most half a step.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

E32 = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# sums over a row: at most 16 elements in one lane, 6 steps over the lanes, 16 waves
ROW = 40
# column sums: tokens of one workgroup (all of them up to 4096 tokens: 16), a 16th of up to 1024 workgroups, 16 waves
COLUMN = 100


class B:
    """A float64 value with a bound on the error of its 32-bit counterpart."""

    def __init__(self, v, e=None):
        self.v = v.double() if isinstance(v, torch.Tensor) else v
        self.e = torch.zeros_like(self.v) if e is None else e

    def __add__(self, o):
        v = self.v + o.v
        return B(v, self.e + o.e + E32 * v.abs())

    def __sub__(self, o):
        v = self.v - o.v
        return B(v, self.e + o.e + E32 * v.abs())

    def __mul__(self, o):
        if not isinstance(o, B):
            o = B(torch.full((), float(np.float32(o)), dtype=torch.float64, device=self.v.device))
        v = self.v * o.v
        return B(v, self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e + E32 * v.abs())

    def sum(self, dim, depth, keepdim=False):
        return B(self.v.sum(dim, keepdim=keepdim), self.e.sum(dim, keepdim=keepdim) + depth * E32 * (self.v.abs() + self.e).sum(dim, keepdim=keepdim))

    def rsqrt(self, eps):
        v = (self.v + eps).rsqrt()
        return B(v, 0.5 * v / (self.v + eps).clamp(min=1e-300) * (self.e + E32 * (self.v + eps)) * 1.01 + 4 * E32 * v)


def check(got, want, what, dtype=None):
    """`got` within the bound of `want` plus one rounding to its type (and half the smallest step of fp16)."""
    g, dtype = got.detach().double(), dtype or got.dtype
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    allowed = (want.e * (1 + half) + half * want.v.abs() + tiny).expand_as(g)
    off = (g - want.v).abs()
    assert g.shape == want.v.shape, what
    bad = ~(off <= allowed)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of what is allowed" % (what, int(bad.sum()), bad.numel(), float((off / allowed)[bad].max()))


@pytest.fixture(scope="module")
def groups():
    from stragglar_amd.torch_emulation import EmulatedGroup
    made = {}

    def get(n):
        if n not in made:
            made[n] = EmulatedGroup(n, algorithm="ring")
        return made[n]
    yield get
    for g in made.values():
        g.close()


def randn(seed, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype).cuda()


def choices(seed, tokens, topk, experts, drop=0.0, ids=torch.int64):
    rng = np.random.default_rng(seed)
    out = rng.integers(0, experts, (tokens, topk))
    out[rng.random((tokens, topk)) < drop] = -1
    return torch.from_numpy(out).to(ids).cuda()


def plain_route(experts, num_experts):
    flat = experts.cpu().numpy().astype(np.int64).reshape(-1)
    key = np.where((flat < 0) | (flat >= num_experts), num_experts, flat)
    order = np.argsort(key, kind="stable")
    total = int((key < num_experts).sum())
    rows = np.full(flat.size, -1)
    rows[order[:total]] = np.arange(total)
    slots = np.full(flat.size, -1)
    slots[:total] = order[:total]
    return rows, slots, np.searchsorted(key[order], np.arange(num_experts + 1), side="left")


def assert_route(r, experts, num_experts, what=""):
    rows, slots, offsets = plain_route(experts, num_experts)
    assert np.array_equal(r.row_of_slot.cpu().numpy().reshape(-1), rows), what
    assert np.array_equal(r.slot_of_row.cpu().numpy(), slots), what
    assert np.array_equal(r.offsets.cpu().numpy(), offsets), what
    assert np.array_equal(r.rank_offsets.cpu().numpy(), offsets[::num_experts // r.ranks]), what


# ---- route ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,topk,experts,ranks", [
    (0, 2, 8, 4), (1, 1, 4, 4), (1, 8, 64, 8), (7, 3, 12, 3), (16, 8, 64, 8), (333, 2, 8, 8), (1023, 8, 256, 8), (1024, 8, 1024, 8),
    (1025, 8, 1024, 8), (8193, 1, 3, 3), (5000, 5, 60, 6), (100, 64, 128, 4), (40000, 8, 256, 8), (300001, 2, 33, 3)])
@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
def test_route_sorts_stably(groups, tokens, topk, experts, ranks, ids):
    for seed, drop in [(1, 0.0), (2, 0.3)]:
        e = choices(seed, tokens, topk, experts, drop, ids)
        assert_route(groups(ranks).route(e, experts), e, experts, (tokens, topk, experts, drop))


@pytest.mark.parametrize("tokens", [5, 4096, 20000])
def test_route_at_the_edges(groups, tokens):
    g = groups(4)
    same = torch.full((tokens, 2), 3, dtype=torch.int64, device="cuda")
    assert_route(g.route(same, 8), same, 8, "all to one expert, twice each")
    none = torch.full((tokens, 2), -1, dtype=torch.int32, device="cuda")
    r = g.route(none, 8)
    assert_route(r, none, 8, "nobody goes anywhere")
    assert int(r.offsets[-1]) == 0
    odd = choices(3, tokens, 2, 8)
    odd[::3, 0] = 8                       # one past the last expert, and numbers that only look right in 32 bits
    odd[1::3, 1] = (1 << 32) + 2
    odd[2::5, 0] = -(1 << 40) + 1
    assert_route(g.route(odd, 8), odd, 8, "numbers outside the experts")


# ---- dispatch, combine ---------------------------------------------------------------------------------------

MOVES = [(1, 1, 4, 1, 0.0), (5, 2, 8, 3, 0.3), (3, 4, 8, 7, 0.0), (17, 3, 8, 8, 0.0), (40, 2, 4, 9, 0.5), (64, 8, 64, 64, 0.0), (129, 5, 16, 511, 0.2),
         (33, 2, 8, 1001, 0.1), (32, 8, 64, 2048, 0.0), (21, 6, 12, 4104, 0.1), (6, 64, 64, 130, 0.1), (5000, 2, 8, 1000, 0.1), (4200, 3, 8, 1003, 0.0)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("tokens,topk,experts,dim,drop", MOVES)
def test_dispatch_and_its_gradient(groups, tokens, topk, experts, dim, drop, dtype):
    g, dt = groups(4), DT[dtype]
    e = choices(tokens + dim, tokens, topk, experts, drop)
    r = g.route(e, experts)
    x = randn(1, tokens, dim, dtype=dt).requires_grad_(True)
    rows = g.dispatch(x, r)
    slots = r.slot_of_row.long()
    want = torch.where((slots >= 0).unsqueeze(1), x.detach()[slots.clamp(min=0) // topk], torch.zeros((), dtype=dt, device="cuda"))
    assert torch.equal(rows, want)
    grad = randn(2, tokens * topk, dim, dtype=dt)
    total = int(r.offsets[-1])
    grad[total:] = float("nan")                                      # rows nobody reads
    gx, = torch.autograd.grad(rows, x, grad)
    kept = B(torch.zeros(tokens, topk, dim, dtype=torch.float64, device="cuda"))
    index = r.row_of_slot.long()
    kept.v[index >= 0] = grad.double()[index[index >= 0]]
    check(gx, kept.sum(1, topk), "grad_tokens")
    assert torch.equal(g.dispatch_backward(grad, r), gx)


@pytest.mark.parametrize("dtype,weights", [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("tokens,topk,experts,dim,drop", MOVES)
def test_combine_and_its_gradients(groups, tokens, topk, experts, dim, drop, dtype, weights):
    g, dt = groups(4), DT[dtype]
    r = g.route(choices(tokens + dim, tokens, topk, experts, drop), experts)
    index = r.row_of_slot.long()
    has = index >= 0
    total = int(r.offsets[-1])
    rows = randn(3, tokens * topk, dim, dtype=dt)
    rows[total:] = float("inf")                                      # rows nobody was sent to
    w = randn(4, tokens, topk, dtype=DT[weights], scale=0.5)
    w[~has] = float("nan")                                           # weights of dropped slots
    rows.requires_grad_(True), w.requires_grad_(True)
    y = g.combine(rows, r, w)
    taken = torch.zeros(tokens, topk, dim, dtype=torch.float64, device="cuda")
    taken[has] = rows.detach().double()[index[has]]
    ww = torch.where(has, w.detach().double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    check(y, (B(taken) * B(ww.unsqueeze(2))).sum(1, topk), "combine")
    grad = randn(5, tokens, dim, dtype=dt)
    gr, gw = torch.autograd.grad(y, (rows, w), grad)
    want = torch.zeros(tokens * topk, dim, dtype=torch.float64, device="cuda")
    want[index[has]] = (grad.double().unsqueeze(1) * ww.unsqueeze(2))[has]
    check(gr, B(want, E32 * want.abs()), "grad_rows")
    # dot products: a lane adds at most 8 elements of 4 vectors a segment of 64 lanes, 6 steps over the lanes, then segments
    depth = dim // 64 + 64
    check(gw, (B(grad.double().unsqueeze(1).expand_as(taken)) * B(taken)).sum(2, depth), "grad_weights")
    assert not gw[~has].any() and not gr[total:].any()
    er, ew = g.combine_backward(grad, rows.detach(), r, w.detach())
    assert torch.equal(er, gr) and torch.equal(ew, gw)
    # one gradient without the other
    y = g.combine(rows, r, w.detach())
    assert torch.equal(torch.autograd.grad(y, rows, grad)[0], gr)
    y = g.combine(rows.detach(), r, w)
    assert torch.equal(torch.autograd.grad(y, w, grad)[0], gw)
    # without weights
    y = g.combine(rows, r)
    check(y, B(taken).sum(1, topk), "plain sum")
    want = torch.zeros(tokens * topk, dim, dtype=dt, device="cuda")
    want[index[has]] = grad.unsqueeze(1).expand(-1, topk, -1)[has]
    assert torch.equal(torch.autograd.grad(y, rows, grad)[0], want)


def test_moves_on_rows_off_every_boundary(groups):
    """Views that start in the middle of an allocation: rows on element boundaries only."""
    g = groups(4)
    for dt, dim in [(torch.bfloat16, 77), (torch.float16, 1001), (torch.float32, 33)]:
        base = randn(6, 31, dim, dtype=dt)
        r = g.route(choices(7, 30, 2, 8, 0.2), 8)
        x = base[1:]
        assert torch.equal(g.dispatch(x, r), g.dispatch(x.clone(), r))
        rows = g.dispatch(x, r)
        big = torch.cat([rows[:1], rows])[1:]
        assert torch.equal(g.combine(big, r), g.combine(rows, r))
        res, w = base[1:], randn(8, dim + 1, dtype=dt)[1:]
        a, b = g.reduce_norm(x, res, pre_weight=w, post_weight=w, gate=w), g.reduce_norm(x.clone(), res.clone(), w.clone(), w.clone(), w.clone())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_outputs_leave_their_neighbours_alone(groups, sarlib):
    """The C entries on outputs in the middle of larger buffers: what lies in front of and behind them stays."""
    g = groups(4)
    for dt, code, dim in [(torch.bfloat16, 2, 77), (torch.float32, 0, 6), (torch.float16, 1, 3), (torch.float16, 1, 520)]:
        tokens, topk = 19, 2
        r = g.route(choices(9, tokens, topk, 8, 0.3), 8)
        x = randn(10, tokens, dim, dtype=dt)
        pad = 64 + 1
        buf = torch.full((2 * pad + tokens * topk * dim,), 7.0, dtype=dt, device="cuda")
        es = buf.element_size()
        stream = torch.cuda.current_stream().cuda_stream
        sarlib.check(sarlib.lib.sar_dispatch(0, stream, code, x.data_ptr(), tokens, topk, dim, r.row_of_slot.data_ptr(), r.offsets.data_ptr(), 8,
                                             None, 0, buf.data_ptr() + pad * es))
        assert torch.equal(buf[pad:-pad].view(-1, dim), g.dispatch(x, r))
        assert (buf[:pad] == 7).all() and (buf[-pad:] == 7).all()
        buf.fill_(7.0)
        rows = g.dispatch(x, r)
        sarlib.check(sarlib.lib.sar_combine(0, stream, code, rows.data_ptr(), tokens, topk, dim, r.row_of_slot.data_ptr(), None, 0, buf.data_ptr() + pad * es))
        end = pad + tokens * dim
        assert torch.equal(buf[pad:end].view(-1, dim), g.combine(rows, r))
        assert (buf[:pad] == 7).all() and (buf[end:] == 7).all()


# ---- reduce_norm -----------------------------------------------------------------------------------------------

def norm_inputs(seed, n, tokens, dim, dtype, weights, partials, pre, post, gate):
    dt, wt = DT[dtype], DT[weights]
    if partials == "ranks":
        p = [randn(seed + 10 + r, tokens, dim, dtype=dt, scale=n ** -0.5) for r in range(n)]
    elif partials == "block":
        p = randn(seed + 10, n, tokens, dim, dtype=dt, scale=n ** -0.5)
    else:
        p = randn(seed + 10, tokens, dim, dtype=dt)
    shape = {"none": None, "channel": (dim,), "token": (tokens, 1), "full": (tokens, dim)}[gate]
    return dict(partials=p, residual=randn(seed + 1, tokens, dim, dtype=dt),
                pre_weight=randn(seed + 2, dim, dtype=wt, scale=0.2, mean=1.0) if pre else None,
                post_weight=randn(seed + 3, dim, dtype=wt, scale=0.2, mean=1.0) if post else None,
                gate=None if shape is None else randn(seed + 4, *shape, dtype=wt, scale=0.3, mean=0.5))


def plain_norm(s, scale, eps, grad_hidden=None, grad_normed=None):
    """reduce_norm and its gradients by the formulas, with bounds.  grad_normed: [copies, tokens, dim]."""
    p = s["partials"]
    parts = list(p) if isinstance(p, list) or p.dim() == 3 else [p]
    dim = s["residual"].shape[1]
    f32eps = float(np.float32(eps))
    y = B(parts[0])
    for q in parts[1:]:
        y = y + B(q)

    def norm(x):
        return ((x * x).sum(1, ROW, keepdim=True) * (1.0 / dim)).rsqrt(f32eps)
    u, yhat, r1 = y, y, None
    if s["post_weight"] is not None:
        r1 = norm(y)
        yhat = y * r1
        u = yhat * B(s["post_weight"])
    gate = B(s["gate"]) if s["gate"] is not None else B(torch.ones(1, device="cuda"))
    h = B(s["residual"]) * scale + gate * u
    x = None
    if s["pre_weight"] is not None:
        r2 = norm(h)
        hhat = h * r2
        x = hhat * B(s["pre_weight"])
    if grad_hidden is None and grad_normed is None:
        return h, x
    zero = B(torch.zeros_like(h.v))
    dh = B(grad_hidden) if grad_hidden is not None else zero
    d_pre = None
    if grad_normed is not None and x is not None:
        G = B(grad_normed[0])
        for q in grad_normed[1:]:
            G = G + B(q)
        t = G * B(s["pre_weight"])
        c = (t * hhat).sum(1, ROW, keepdim=True) * (1.0 / dim)
        dh = dh + r2 * (t - hhat * c)
        d_pre = (G * hhat).sum(0, COLUMN)
    elif x is not None:
        d_pre = B(torch.zeros(dim, device="cuda"))
    du = dh * gate
    dy, d_post = du, None
    if r1 is not None:
        t = du * B(s["post_weight"])
        c = (t * yhat).sum(1, ROW, keepdim=True) * (1.0 / dim)
        dy = r1 * (t - yhat * c)
        d_post = (du * yhat).sum(0, COLUMN)
    d_gate = None
    if s["gate"] is not None:
        dg = dh * u
        d_gate = dg.sum(0, COLUMN) if s["gate"].dim() == 1 else dg.sum(1, ROW, keepdim=True) if s["gate"].shape[1] == 1 and dim > 1 else dg
    return h, x, dict(partials=dy, residual=dh * scale, pre_weight=d_pre, post_weight=d_post, gate=d_gate)


def run_norm(group, s, scale, eps, gather, save=False):
    return group.reduce_norm(s["partials"], s["residual"], pre_weight=s["pre_weight"], post_weight=s["post_weight"], gate=s["gate"],
                             residual_scale=scale, eps=eps, gather=gather, save=save)


NORMS = [  # ranks, tokens, dim, partials, gather, pre, post, gate
    (4, 1, 1, "ranks", True, True, True, "channel"), (4, 3, 1, "one", False, True, True, "token"), (3, 5, 3, "ranks", True, True, True, "full"),
    (4, 2, 7, "block", False, True, False, "token"), (4, 9, 8, "ranks", True, True, True, "none"), (6, 33, 64, "ranks", True, True, True, "channel"),
    (8, 17, 1001, "ranks", True, True, True, "token"), (8, 130, 511, "one", False, True, True, "full"), (8, 7, 2048, "block", True, False, True, "channel"),
    (8, 64, 4096, "ranks", True, True, True, "channel"), (3, 5, 4100, "one", True, True, False, "none"), (5, 6, 8192, "ranks", False, True, True, "channel"),
    (4, 3, 9001, "ranks", True, True, True, "full"), (3, 4, 16384, "ranks", True, True, True, "channel"), (3, 2, 16383, "one", False, False, False, "token"),
    (16, 40, 320, "ranks", True, True, True, "channel"), (64, 5, 96, "ranks", True, True, True, "token"), (4, 2500, 200, "one", True, True, True, "channel"),
    (4, 0, 64, "ranks", True, True, True, "channel"), (3, 4000, 37, "ranks", False, True, True, "token")]


@pytest.mark.parametrize("dtype,weights", [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("n,tokens,dim,partials,gather,pre,post,gate", NORMS)
def test_reduce_norm_and_its_gradients(groups, n, tokens, dim, partials, gather, pre, post, gate, dtype, weights):
    g, dt, scale, eps = groups(n), DT[dtype], 0.8125, 1e-5
    s = norm_inputs(tokens + dim, n, tokens, dim, dtype, weights, partials, pre, post, gate)
    hidden, normed = run_norm(g, s, scale, eps, gather)
    copies = n if gather else 1
    grad_hidden = randn(90, tokens, dim, dtype=dt)
    grad_normed = randn(91, copies, tokens, dim, dtype=dt, scale=copies ** -0.5) if pre else None
    h, x, want = plain_norm(s, scale, eps, grad_hidden, grad_normed)
    check(hidden, h, "hidden")
    if pre:
        assert normed.shape == ((n, tokens, dim) if gather else (tokens, dim))
        for copy in (normed if gather else [normed]):
            check(copy, x, "normed")
    else:
        assert normed is None
    leaves = [t.requires_grad_(True) for t in (s["partials"] if isinstance(s["partials"], list) else [s["partials"]])]
    names = [k for k in ("residual", "pre_weight", "post_weight", "gate") if s[k] is not None]
    for k in names:
        s[k].requires_grad_(True)
    h2, x2 = run_norm(g, s, scale, eps, gather)
    assert torch.equal(h2, hidden) and (not pre or torch.equal(x2, normed))
    outs, grads = ([h2, x2], [grad_hidden, grad_normed if gather else grad_normed[0]]) if pre else ([h2], [grad_hidden])
    got = torch.autograd.grad(outs, leaves + [s[k] for k in names], grads)
    for p in got[:len(leaves)]:
        for q in (p if p.dim() == 3 else [p]):
            check(q, want["partials"], "partials")
    for k, v in zip(names, got[len(leaves):]):
        assert v.shape == s[k].shape and v.dtype == s[k].dtype
        check(v, want[k], "grad of " + k)
    # the explicit pair gives the same bits
    with torch.no_grad():
        h3, x3, saved = run_norm(g, s, scale, eps, gather, save=True)
        again = g.reduce_norm_backward(saved, grad_hidden, grad_normed if gather or not pre else grad_normed[0])
    assert torch.equal(h3, hidden)
    flat = list(again.partials) if isinstance(s["partials"], list) else [again.partials]
    assert all(torch.equal(a, b) for a, b in zip(flat, got))
    for k, v in zip(names, got[len(leaves):]):
        assert torch.equal(getattr(again, k), v), k


def test_reduce_norm_with_one_gradient_missing(groups):
    g, scale, eps = groups(4), 1.0, 1e-6
    s = norm_inputs(5, 4, 12, 100, "f32", "f32", "ranks", True, True, "channel")
    gh, gx = randn(1, 12, 100), randn(2, 4, 12, 100)
    with torch.no_grad():
        _, _, saved = run_norm(g, s, scale, eps, True, save=True)
        for a, b in [(gh, None), (None, gx)]:
            got = g.reduce_norm_backward(saved, a, b)
            want = plain_norm(s, scale, eps, a, b)[2]
            for k in ("residual", "pre_weight", "post_weight", "gate"):
                check(getattr(got, k), want[k], k)
            for p in got.partials:
                check(p, want["partials"], "partials")
        none = g.reduce_norm_backward(saved)
        assert not any(t.any() for t in none)
    # only some inputs ask for a gradient; gradients that come expanded (stride 0) and only through one output
    s["gate"].requires_grad_(True), s["partials"][2].requires_grad_(True)
    hidden, normed = run_norm(g, s, scale, eps, True)
    a, b = torch.autograd.grad(normed.sum(), (s["gate"], s["partials"][2]))
    want = plain_norm(s, scale, eps, None, torch.ones(4, 12, 100, device="cuda"))[2]
    check(a, want["gate"], "gate"), check(b, want["partials"], "partial 2")


def test_reduce_norm_gradients_against_differences(groups):
    """Directional derivatives of the 64-bit formulas by central differences: step 2^-20, so the cubic term is below 1e-11
    and the cancellation below 1e-9 of the loss."""
    g, n, t, d, eps, scale = groups(3), 3, 4, 24, 1e-5, 0.75
    for gate in ("none", "channel", "token", "full"):
        s = norm_inputs(3, n, t, d, "f32", "f32", "ranks", True, True, gate)
        gh, gx = randn(1, t, d), randn(2, n, t, d)
        with torch.no_grad():
            saved = run_norm(g, s, scale, eps, True, save=True)[2]
            got = g.reduce_norm_backward(saved, gh, gx)
        bound = plain_norm(s, scale, eps, gh, gx)[2]

        def loss(q):
            h, x = plain_norm(q, scale, eps)
            return float((h.v * gh.double()).sum() + (x.v.unsqueeze(0) * gx.double()).sum())
        for k in ("residual", "pre_weight", "post_weight", "gate", 0, 2):
            if k == "gate" and gate == "none":
                continue
            base = (s["partials"][k] if isinstance(k, int) else s[k]).double()
            v = randn(50, *base.shape).double()
            vals = []
            for step in (2.0 ** -20, -2.0 ** -20):
                q = dict(s, partials=[p.double() for p in s["partials"]], **{j: s[j].double() for j in ("residual", "pre_weight", "post_weight", "gate") if s[j] is not None})
                if isinstance(k, int):
                    q["partials"][k] = base + step * v
                else:
                    q[k] = base + step * v
                vals.append(loss(q))
            slope = (vals[0] - vals[1]) / 2.0 ** -19
            mine, b = (got.partials[k], bound["partials"]) if isinstance(k, int) else (getattr(got, k), bound[k])
            allowed = float(((b.e + E32 * b.v.abs()) * v.abs()).sum()) + 1e-6 * (1 + abs(slope))
            assert abs(float((mine.double() * v).sum()) - slope) <= allowed, (gate, k)


def test_reduce_norm_of_zeros_infinities_and_nan(groups):
    g, d = groups(4), 300
    x = torch.zeros(5, d, device="cuda")
    x[1] = 1.0
    x[2, 7] = float("inf")
    x[3, 299] = float("nan")
    w = torch.ones(d, device="cuda")
    hidden, normed = g.reduce_norm(x, torch.zeros(5, d, device="cuda"), pre_weight=w, post_weight=w, gather=False)
    assert not hidden[0].any() and not normed[0].any()                        # zeros stay zeros (eps > 0)
    assert torch.allclose(normed[1], torch.ones_like(normed[1]), rtol=0, atol=2e-6)    # eps 1e-6 twice: 1 - 1e-6
    for row, col in ((2, 7), (3, 299)):                                          # inf * 0 and NaN, in their own rows only
        assert torch.isnan(hidden[row, col]) and torch.isnan(normed[row]).all()
    assert torch.isfinite(hidden[4]).all() and torch.isfinite(normed[4]).all()
    # 16-bit values whose squares leave the type: statistics are kept in 32 bits
    big = torch.full((3, d), 60000.0, dtype=torch.float16, device="cuda")
    _, normed = g.reduce_norm([big] * 4, torch.zeros_like(big), pre_weight=w.half(), post_weight=w.half())
    assert torch.allclose(normed.float(), torch.ones_like(normed.float()), rtol=0, atol=2 ** -10)


def test_more_rows_than_one_pass_of_the_grid(groups):
    """Row counts at which every kernel's grid goes round: 2^20 workgroups of norms, 2^20 of four tokens."""
    g = groups(4)
    x, res, w = randn(1, 1100003, 8, dtype=torch.float16), randn(2, 1100003, 8, dtype=torch.float16), randn(3, 8, mean=1.0, scale=0.1)
    gh, gx = randn(4, 1100003, 8, dtype=torch.float16), randn(5, 1100003, 8, dtype=torch.float16)
    s = dict(partials=x, residual=res, pre_weight=w, post_weight=w, gate=w)
    with torch.no_grad():
        hidden, normed, saved = run_norm(g, s, 0.5, 1e-6, False, save=True)
        back = g.reduce_norm_backward(saved, gh, gx)
    h, n, want = plain_norm(s, 0.5, 1e-6, gh, gx.unsqueeze(0))
    check(hidden, h, "hidden"), check(normed, n, "normed"), check(back.partials, want["partials"], "partials")
    # column sums: 1100003 tokens over 512 workgroups of 8 rows is 269 additions in a row, in front of the rest of COLUMN
    for k in ("pre_weight", "post_weight", "gate"):
        check(getattr(back, k), B(want[k].v, want[k].e * 4), k)
    t = 4200003
    e = choices(6, t, 1, 8, 0.1)
    r = g.route(e, 8)
    assert_route(r, e, 8)
    rows, wt, gy = randn(7, t, 8, dtype=torch.bfloat16), randn(8, t, 1), randn(9, t, 8, dtype=torch.bfloat16)
    index, has = r.row_of_slot.long()[:, 0], r.row_of_slot[:, 0] >= 0
    y = g.combine(rows, r, wt)
    taken = torch.where(has.unsqueeze(1), rows.double()[index.clamp(min=0)], torch.zeros((), dtype=torch.float64, device="cuda"))
    check(y, B(taken) * B(wt), "combine")
    gr, gw = g.combine_backward(gy, rows, r, wt)
    check(gw, (B(gy) * B(taken)).sum(1, 16, keepdim=True), "grad_weights")
    check(gr[index[has]], B(gy[has]) * B(wt[has]), "grad_rows")
    assert not gr[int(r.offsets[-1]):].any()
    assert torch.equal(g.dispatch(gy, r)[index[has]], gy[has])


@pytest.mark.parametrize("dtype,dim", [("bf16", 4096), ("f16", 2050), ("f32", 1028)])
def test_calls_large_enough_to_stream(groups, dtype, dim):
    """Calls of 512 MiB and more go past the caches, in kernels of their own: every kind of call at such a size, looked at in
    a few places."""
    n, dt = 8, DT[dtype]
    g = groups(n)
    es = torch.finfo(dt).bits // 8
    t = (600 << 20) // (18 * dim * es)
    base = [randn(r, 499, dim, dtype=dt) for r in range(4)]
    spread = torch.arange(t, device="cuda")
    s = dict(partials=[base[r % 4][(spread * (r + 1) + r) % 499] for r in range(n)], residual=base[3][(spread * 3) % 499],
             pre_weight=randn(5, dim, mean=1.0, scale=0.2), post_weight=randn(6, dim, mean=1.0, scale=0.2), gate=randn(7, dim, mean=0.5, scale=0.2))
    gh, gx = base[0][(spread * 7) % 499], torch.stack([base[r % 4][(spread * 11 + r) % 499] for r in range(n)])
    with torch.no_grad():
        hidden, normed, saved = run_norm(g, s, 0.75, 1e-6, True, save=True)
        back = g.reduce_norm_backward(saved, gh, gx)
    for a in (0, t // 2, t - 30):
        part = slice(a, a + 30)
        h, x, want = plain_norm(dict(s, partials=[p[part] for p in s["partials"]], residual=s["residual"][part]), 0.75, 1e-6, gh[part], gx[:, part])
        check(hidden[part], h, a), check(back.residual[part], want["residual"], a)
        for r in range(n):
            check(normed[r, part], x, (a, r)), check(back.partials[r, part], want["partials"], (a, r))
    # the column sums, over all tokens
    sums = {k: torch.zeros(dim, dtype=torch.float64, device="cuda") for k in ("pre_weight", "post_weight", "gate")}
    bounds = {k: torch.zeros(dim, dtype=torch.float64, device="cuda") for k in sums}
    for a in range(0, t, 1000):
        part = slice(a, min(t, a + 1000))
        want = plain_norm(dict(s, partials=[p[part] for p in s["partials"]], residual=s["residual"][part]), 0.75, 1e-6, gh[part], gx[:, part])[2]
        for k in sums:
            sums[k] += want[k].v
            bounds[k] += want[k].e
    for k in sums:
        check(getattr(back, k), B(sums[k], bounds[k]), k)
    del hidden, normed, saved, back, gx, s
    topk = 4
    t = (560 << 20) // (topk * dim * es)
    r = g.route(choices(1, t, topk, 16, 0.05), 16)
    x = base[0][torch.arange(t, device="cuda") % 499]
    rows = g.dispatch(x, r)
    slots = r.slot_of_row.long()
    want = torch.where((slots >= 0).unsqueeze(1), x[slots.clamp(min=0) // topk], torch.zeros((), dtype=dt, device="cuda"))
    assert torch.equal(rows, want)
    del want
    w = torch.softmax(randn(3, t, topk), 1)
    y = g.combine(rows, r, w)
    gr, gw = g.combine_backward(x, rows, r, w)
    assert not gr[int(r.offsets[-1]):].any()
    for a in (0, t // 2, t - 30):
        part = slice(a, a + 30)
        index, has = r.row_of_slot[part].long(), r.row_of_slot[part] >= 0
        taken = torch.where(has.unsqueeze(2), rows[index.clamp(min=0)].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
        check(y[part], (B(taken) * B(w[part].unsqueeze(2))).sum(1, topk), a)
        check(gw[part], (B(x[part].unsqueeze(1).expand_as(taken)) * B(taken)).sum(2, dim // 64 + 64), a)
        check(gr[index[has]], B(x[part].unsqueeze(1).expand(-1, topk, -1)[has]) * B(w[part][has].unsqueeze(1)), a)


def test_row_numbers_out_of_range_count_as_dropped(groups):
    """A routing whose numbers were overwritten: the kernels hold every row number against the number of rows."""
    from stragglar_amd.block_ops import Routing
    g = groups(4)
    r = g.route(choices(1, 10, 2, 8), 8)
    rows = r.row_of_slot.clone()
    rows[3, 0], rows[5, 1], rows[7, 0] = 20, -12345, 2 ** 31 - 1
    offsets = r.offsets.clone()
    offsets[-1] = 2 ** 31 - 1
    bad = Routing(rows, r.slot_of_row, offsets, 8, 4)
    x, w = randn(2, 10, 24), torch.ones(10, 2, device="cuda")
    out = g.dispatch(x, bad)
    keep = torch.ones(10, 2, dtype=torch.bool, device="cuda")
    keep[3, 0] = keep[5, 1] = keep[7, 0] = False
    src = randn(3, 20, 24)
    want = (src[r.row_of_slot.long()] * keep.unsqueeze(2)).sum(1)
    assert torch.equal(out[r.row_of_slot[keep].long()], x.unsqueeze(1).expand(-1, 2, -1)[keep])
    assert torch.equal(g.combine(src, bad, w), want)
    gr, gw = g.combine_backward(x, src, bad, w)
    assert not gw[~keep].any() and torch.equal(gr[r.row_of_slot[keep].long()], x.unsqueeze(1).expand(-1, 2, -1)[keep])


def test_not_differentiable_twice(groups):
    g = groups(4)
    x = randn(1, 6, 16).requires_grad_(True)
    r = g.route(choices(2, 6, 2, 8), 8)
    w = torch.softmax(randn(3, 6, 2), 1).requires_grad_(True)
    hidden, normed = g.reduce_norm(x, x.detach(), pre_weight=torch.ones(16, device="cuda"), gather=False)
    for out, leaf in [(g.dispatch(x, r), x), (g.combine(g.dispatch(x, r).detach(), r, w), w), (normed, x)]:
        grad, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)      # once is fine
        with pytest.raises(RuntimeError, match="once_differentiable|twice"):
            grad.sum().backward()


# ---- together, and in a program ----------------------------------------------------------------------------------

def block(g, partials, residual, experts, weights, mats, w, gate, num_experts):
    """The second half of a block: attention's partial outputs come in, the experts' block goes out."""
    hidden, x = g.reduce_norm(partials, residual, pre_weight=w[0], post_weight=w[1], gate=gate, gather=False)
    r = g.route(experts, num_experts)
    rows = g.dispatch(x, r)
    ends = r.offsets.tolist()
    out = [torch.tanh(rows[a:b] @ m) for a, b, m in zip(ends, ends[1:], mats)] + [rows[ends[-1]:]]
    y = g.combine(torch.cat(out), r, weights)
    return g.reduce_norm(y, hidden, pre_weight=w[2], post_weight=w[3], gate=gate, residual_scale=0.5, gather=True)


def plain_block(partials, residual, experts, weights, mats, w, gate, num_experts, n, eps=1e-6):
    def rms(x, v):
        return x / torch.sqrt(x.square().mean(1, keepdim=True) + eps) * v
    hidden = residual + gate * rms(sum(partials), w[1])
    x = rms(hidden, w[0])
    y = torch.zeros_like(x)
    for e in range(num_experts):
        for k in range(experts.shape[1]):
            at = (experts[:, k] == e).nonzero()[:, 0]
            y = y.index_add(0, at, weights[at, k].unsqueeze(1) * torch.tanh(x[at] @ mats[e]))
    hidden2 = 0.5 * hidden + gate * rms(y, w[3])
    return hidden2, rms(hidden2, w[2]).unsqueeze(0).expand(n, -1, -1)


def test_a_block_forward_and_backward(groups):
    """All operators in a row as a model uses them, in 32 bits, against autograd in 64 bits.  What the chain of about ten
    operators with condition numbers of a few tens can lose stays below 2^-24 * 1000 = 6e-5 of the largest value."""
    n, t, d, e, k = 4, 37, 48, 8, 3
    g = groups(n)
    leaves = ([randn(r, t, d, scale=0.5) for r in range(n)] + [randn(9, t, d)] + [torch.softmax(randn(10, t, k), 1)] +
              [randn(20 + i, d, d, scale=d ** -0.5) for i in range(e)] + [randn(40 + i, d, scale=0.1, mean=1.0) for i in range(4)] + [randn(50, d, scale=0.1, mean=0.7)])
    ids = choices(11, t, k, e, 0.1)
    gh, gx = randn(60, t, d), randn(61, n, t, d)

    def split(v):
        return v[:n], v[n], ids, v[n + 1], v[n + 2:n + 2 + e], v[n + 2 + e:n + 6 + e], v[-1], e
    mine = [v.clone().requires_grad_(True) for v in leaves]
    out = block(g, *split(mine))
    got = list(out) + list(torch.autograd.grad(out, mine, (gh, gx)))
    theirs = [v.double().requires_grad_(True) for v in leaves]
    ref = plain_block(*split(theirs), n)
    want = list(ref) + list(torch.autograd.grad(ref, theirs, (gh.double(), gx.double())))
    for i, (a, b) in enumerate(zip(got, want)):
        assert float((a.detach().double() - b.detach()).abs().max()) <= 6e-5 * float(b.detach().abs().max()), i


def test_block_operators_beside_all_reduce(groups):
    """A training step's pieces on one group: block gradients, then the gradient AllReduce on the same ranks."""
    from stragglar_amd.torch_emulation import EmulatedGroup
    group = EmulatedGroup(4)
    try:
        s = norm_inputs(1, 4, 30, 60, "f32", "f32", "ranks", True, True, "channel")
        with torch.no_grad():
            saved = run_norm(group, s, 1.0, 1e-6, True, save=True)[2]
            grads = [group.reduce_norm_backward(saved, randn(70 + r, 30, 60)) for r in range(4)]
        want = sum(q.post_weight.double() for q in grads) / 4
        per_rank = [[q.post_weight, q.gate] for q in grads]
        group.allreduce_gradients(per_rank)
        for r in range(4):
            assert torch.allclose(per_rank[r][0].double(), want, rtol=0, atol=1e-5)
    finally:
        group.close()


def test_the_same_inputs_give_the_same_bits(groups):
    g = groups(8)
    s = norm_inputs(8, 8, 1500, 264, "bf16", "f32", "ranks", True, True, "channel")
    gh, gx = randn(1, 1500, 264, dtype=torch.bfloat16), randn(2, 8, 1500, 264, dtype=torch.bfloat16)
    e = choices(1, 9000, 4, 64, 0.1)
    rows, w, gy = randn(3, 36000, 40), randn(4, 9000, 4), randn(5, 9000, 40)

    def once():
        with torch.no_grad():
            h, x, saved = run_norm(g, s, 1.0, 1e-6, True, save=True)
            r = g.route(e, 64)
            return [h, x] + list(g.reduce_norm_backward(saved, gh, gx)) + [r.row_of_slot, r.slot_of_row, r.offsets, g.combine(rows, r, w)] + list(g.combine_backward(gy, rows, r, w))
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(once(), first))


def test_on_another_stream(groups):
    g = groups(4)
    e = choices(1, 3000, 3, 8, 0.2)
    x = randn(2, 3000, 129)
    r0 = g.route(e, 8)
    want = g.combine(g.dispatch(x, r0), r0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = torch.randn(2048, 2048, device="cuda")
        for _ in range(20):
            a = torch.tanh(a @ a)                       # keeps the side stream busy
        y = x + 0 * a[0, 0].clamp(-1, 1)               # made on the side stream, late
        r = g.route(e + (0 * a[0, 0].clamp(-1, 1)).long(), 8)
        got = g.combine(g.dispatch(y, r), r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_two_streams_at_once(groups):
    """Calls of different sizes on two streams, one after the other without waiting: nothing is shared between them."""
    g = groups(4)
    jobs = []
    for i, (t, d) in enumerate([(9000, 264), (700, 1001)]):
        e, x, res = choices(i, t, 4, 16, 0.1), randn(10 + i, t, d), randn(20 + i, t, d)
        w, gw, gh = randn(30 + i, d, mean=1.0, scale=0.1), torch.softmax(randn(40 + i, t, 4), 1), randn(50 + i, t, d)
        jobs.append((e, x, res, w, gw, gh))

    def work(e, x, res, w, gw, gh):
        with torch.no_grad():
            r = g.route(e, 16)
            y = g.combine(g.dispatch(x, r), r, gw)
            h, n, saved = g.reduce_norm([x, y, x, y], res, pre_weight=w, post_weight=w, gate=w, save=True)
            return [y, h, n, *g.reduce_norm_backward(saved, gh, n), *g.combine_backward(gh, g.dispatch(x, r), r, gw)]
    want = [work(*j) for j in jobs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(*jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i])), i


def test_no_tokens(groups):
    g = groups(4)
    r = g.route(torch.zeros(0, 2, dtype=torch.int64, device="cuda"), 8)
    assert r.offsets.tolist() == [0] * 9 and r.slot_of_row.numel() == 0
    x, w = torch.zeros(0, 16, device="cuda", requires_grad=True), torch.zeros(0, 2, device="cuda", requires_grad=True)
    rows = g.dispatch(x, r)
    y = g.combine(rows, r, w)
    assert rows.shape == (0, 16) and y.shape == (0, 16)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == (0, 16) and gw.shape == (0, 2)


def test_captured_and_replayed(groups):
    """Forward and explicit backward in two graphs, replayed in turn with eager work in between, on changing inputs."""
    g, n, t, d, e, k = groups(4), 4, 700, 136, 16, 4
    ids = choices(1, t, k, e, 0.1)                          # few slots: one launch
    many = choices(2, 5000, k, e, 0.1)                      # many: three
    parts = [randn(r, t, d, dtype=torch.bfloat16) for r in range(n)]
    res, w = randn(5, t, d, dtype=torch.bfloat16), randn(6, d, mean=1.0, scale=0.1)
    gw = torch.softmax(randn(7, t, k), 1)
    gh, gx = randn(8, t, d, dtype=torch.bfloat16), randn(9, n, t, d, dtype=torch.bfloat16)

    def step():
        with torch.no_grad():
            h, x, saved = g.reduce_norm(parts, res, pre_weight=w, post_weight=w, gate=w, save=True)
            grads = g.reduce_norm_backward(saved, gh, gx)
            r = g.route(ids, e)
            rows = g.dispatch(x[0], r)
            y = g.combine(rows, r, gw)
            gr, gww = g.combine_backward(gh, rows, r, gw)
            m = g.route(many, e)
            return [h, x, *grads, rows, y, gr, gww, g.dispatch_backward(gr, r), m.row_of_slot, m.slot_of_row, m.offsets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(4):
        for t_ in parts:
            t_.copy_(randn(100 + i, t, d, dtype=torch.bfloat16))
        ids.copy_(choices(200 + i, t, k, e, 0.2))
        many.copy_(choices(300 + i, 5000, k, e, 0.2))
        want = step()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_autograd_is_refused_while_capturing(groups):
    g = groups(4)
    x = randn(1, 8, 16).requires_grad_(True)
    r = g.route(choices(2, 8, 2, 8), 8)
    rows = g.dispatch(x, r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = x.detach() * 2
        with pytest.raises(RuntimeError, match="captured"):
            g.dispatch(x, r)
        with pytest.raises(RuntimeError, match="captured"):
            g.reduce_norm(x, x.detach())
        with torch.no_grad():
            out = g.dispatch(x, r)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, rows) and torch.equal(keep, x.detach() * 2)
    assert torch.autograd.grad(rows.sum(), x)[0].shape == x.shape


def test_offsets_beyond_32_bits(groups):
    """Rows whose byte offsets pass 2^32 (and element offsets 2^31): 600000 x 4096 in 16 bits."""
    g, t, k, d = groups(4), 300000, 2, 4096
    e = choices(1, t, k, 8)
    r = g.route(e, 8)
    base = randn(2, 997, d, dtype=torch.bfloat16)
    x = base[torch.arange(t, device="cuda") % 997]
    rows = g.dispatch(x, r)
    slots = r.slot_of_row.long()
    for a in (0, 262140, 524280, t * k - 50):
        assert torch.equal(rows[a:a + 50], x[slots[a:a + 50] // k]), a
    w = torch.softmax(randn(3, t, k), 1)
    y = g.combine(rows, r, w)
    for a in (0, 262140, t - 50):
        want = (B(x[a:a + 50].unsqueeze(1).expand(-1, k, -1)) * B(w[a:a + 50].unsqueeze(2))).sum(1, k)
        check(y[a:a + 50], want, a)
    gr, gw = g.combine_backward(y, rows, r, w)
    at = r.row_of_slot[t - 50:].long()
    check(gr[at[:, 1]], B(y[t - 50:]) * B(w[t - 50:, 1:]), "grad_rows")
    del gr, gw, y, x
    s = dict(partials=rows, residual=rows, pre_weight=randn(4, d, dtype=torch.bfloat16), post_weight=None, gate=None)
    with torch.no_grad():
        hidden, normed, saved = g.reduce_norm(rows, rows, pre_weight=s["pre_weight"], gather=False, save=True)
        back = g.reduce_norm_backward(saved, rows, normed)
    for a in (0, 524280, t * k - 20):
        part = rows[a:a + 20]
        h, x, want = plain_norm(dict(s, partials=part, residual=part), 1.0, 1e-6, part, normed[a:a + 20].unsqueeze(0))
        check(hidden[a:a + 20], h, a), check(normed[a:a + 20], x, a), check(back.residual[a:a + 20], want["residual"], a)


def test_a_routing_between_forward_and_backward(groups):
    """Written again in place it is refused; what route() made under inference_mode gives the gradients of any other."""
    g, t, k, d = groups(4), 50, 2, 40
    e = choices(1, t, k, 8, 0.2)
    x, rows = randn(2, t, d).requires_grad_(True), randn(3, t * k, d).requires_grad_(True)
    w, gx, gr = randn(4, t, k).requires_grad_(True), randn(5, t * k, d), randn(6, t, d)

    def forward(r):
        return (g.dispatch(x, r), g.combine(rows, r, w)), (x, rows, w), (gx, gr)
    r = g.route(e, 8)
    want = torch.autograd.grad(*forward(r))
    with torch.inference_mode():
        made = g.route(e, 8)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(*forward(made)), want))
    for outs in ((g.dispatch(x, r),), (g.combine(rows, r, w),), (g.combine(rows, r),)):
        again = g.route(choices(7, t, k, 8, 0.2), 8)
        r.row_of_slot.copy_(again.row_of_slot), r.offsets.copy_(again.offsets)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            outs[0].sum().backward()


def test_combine_lets_go_of_rows_that_no_gradient_reads(groups):
    """Without a gradient of the weights the rows' memory comes back before the backward pass, with the same gradient."""
    g, t, k, d = groups(4), 4096, 8, 512
    r = g.route(choices(1, t, k, 8), 8)
    leaf, w = randn(2, t * k, d).requires_grad_(True), torch.softmax(randn(3, t, k), 1)
    grad = randn(4, t, d)
    want = g.combine_backward(grad, leaf.detach(), r, w)[0]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    rows = leaf * 1.0
    y = g.combine(rows, r, w)
    del rows
    assert torch.cuda.memory_allocated() - before < 2 * t * d * 4           # y, not the 64 MiB of rows
    assert torch.equal(torch.autograd.grad(y, leaf, grad)[0], want)


def test_saved_tensors_kept_on_the_host(groups):
    """Offloaded and brought back they give the same bits; left on the host they are refused before a kernel sees them."""
    g, t, k, d = groups(4), 60, 2, 72
    r = g.route(choices(1, t, k, 8, 0.2), 8)
    x, w, v = randn(2, t, d).requires_grad_(True), torch.softmax(randn(3, t, k), 1).requires_grad_(True), randn(4, d, mean=1.0, scale=0.1).requires_grad_(True)

    def forward():
        y = g.combine(g.dispatch(x, r), r, w)
        return g.reduce_norm([y, x, y, x], x, pre_weight=v, post_weight=v, gate=v)[1]
    want = torch.autograd.grad(forward().square().sum(), (x, w, v))
    with torch.autograd.graph.save_on_cpu():
        out = forward()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out.square().sum(), (x, w, v)), want))
    for call in (lambda: g.dispatch(x, r), lambda: g.combine(x[:1].expand(t * k, -1).contiguous(), r, w), lambda: g.reduce_norm(x, x, v)[1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s.cpu(), lambda s: s):
            out = call()
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            out.backward(torch.ones_like(out))


# ---- every kernel's streaming form (calls of 512 MiB and more) -----------------------------------------------------

@pytest.mark.parametrize("dtype,dim", [("bf16", 512), ("f16", 505), ("f32", 520), ("bf16", 1001), ("f16", 2041), ("f32", 1024)])
def test_streaming_gradients_of_short_rows(groups, dtype, dim):
    """combine's gradients where a wave has a token to itself: rows of up to 64, 128 and 256 vectors.  With and without a
    gradient of the weights (then the rows' is a weighted dispatch)."""
    g, dt, topk = groups(8), DT[dtype], 8
    row = dim * torch.finfo(dt).bits // 8
    t = (530 << 20) // (topk * row)                                # rows alone pass 512 MiB
    assert t >= 2048 and row <= 256 * 16
    r = g.route(choices(dim, t, topk, 16, 0.05), 16)
    index, has, total = r.row_of_slot.long(), r.row_of_slot >= 0, int(r.offsets[-1])
    base = randn(1, 499, dim, dtype=dt)
    rows = base[torch.arange(t * topk, device="cuda") % 499].requires_grad_(True)
    grad = base[torch.arange(t, device="cuda") * 5 % 499]
    w = randn(2, t, topk, scale=0.5)
    alone, = torch.autograd.grad(g.combine(rows, r, w), rows, grad)
    gr, gw = g.combine_backward(grad, rows.detach(), r, w)
    assert torch.equal(alone, gr)
    assert not gr[total:].any() and not gw[~has].any()
    y = g.combine(rows.detach(), r, w)
    for a in (0, t // 3, t - 40):
        part = slice(a, a + 40)
        i, h = index[part], has[part]
        taken = torch.where(h.unsqueeze(2), rows.detach()[i.clamp(min=0)].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
        check(y[part], (B(taken) * B(w[part].unsqueeze(2))).sum(1, topk), a)
        check(gw[part], (B(grad[part].unsqueeze(1).expand_as(taken)) * B(taken)).sum(2, dim // 64 + 64), a)
        check(gr[i[h]], B(grad[part].unsqueeze(1).expand(-1, topk, -1)[h]) * B(w[part][h].unsqueeze(1)), a)


@pytest.mark.parametrize("dtype,dim,n,partials,gather,gate", [
    ("bf16", 9001, 3, "ranks", True, "channel"), ("f16", 16384, 4, "ranks", False, "full"), ("f32", 5000, 3, "ranks", True, "token"),
    ("f32", 16384, 3, "ranks", True, "channel"), ("f32", 8193, 3, "one", False, "channel"), ("bf16", 16383, 3, "one", False, "channel"),
    ("bf16", 256, 4, "ranks", True, "channel"), ("f16", 250, 4, "one", False, "channel"), ("f32", 516, 8, "ranks", True, "none"), ("bf16", 4096, 3, "one", False, "token")])
def test_streaming_norms(groups, dtype, dim, n, partials, gather, gate):
    """Rows of two and four vectors a thread (their column sums in LDS), rows that share a workgroup, and finished outputs.
    Column sums add at most tokens / (workgroups * rows) + rows + workgroups / 32 + 32 times in a row: 122 for rows of 250, 82
    and less for the others, so 1.25 times what COLUMN allows holds for all."""
    g, dt, scale, eps = groups(n), DT[dtype], 0.75, 1e-6
    sources, copies = n if partials == "ranks" else 1, n if gather else 1
    row = dim * torch.finfo(dt).bits // 8
    t = (513 << 20) // ((sources + copies + 2) * row) + 1           # the rows that the smallest pass counts
    spread = torch.arange(t, device="cuda")
    base = [randn(r, 499, dim, dtype=dt) for r in range(4)]
    parts = [base[r % 4][(spread * (r + 1) + r) % 499] * n ** -0.5 for r in range(sources)]
    shape = {"none": None, "channel": (dim,), "token": (t, 1), "full": (t, dim)}[gate]
    s = dict(partials=parts if partials == "ranks" else parts[0], residual=base[3][(spread * 3) % 499],
             pre_weight=randn(5, dim, mean=1.0, scale=0.2), post_weight=randn(6, dim, mean=1.0, scale=0.2),
             gate=None if shape is None else randn(7, *shape, mean=0.5, scale=0.2))
    gh = base[0][(spread * 7) % 499]
    gx = torch.stack([base[r % 4][(spread * 11 + r) % 499] for r in range(copies)])
    with torch.no_grad():
        hidden, normed, saved = run_norm(g, s, scale, eps, gather, save=True)
        back = g.reduce_norm_backward(saved, gh, gx if gather else gx[0])
        again = run_norm(g, s, scale, eps, gather)                                  # without a total to write
    assert torch.equal(again[0], hidden) and torch.equal(again[1], normed)
    del again

    def cut(part):
        p = [q[part] for q in s["partials"]] if partials == "ranks" else s["partials"][part]
        q = dict(s, partials=p, residual=s["residual"][part])
        if gate in ("token", "full"):
            q["gate"] = s["gate"][part]
        return plain_norm(q, scale, eps, gh[part], gx[:, part])
    sums = {}
    for a in range(0, t, 2000):
        part = slice(a, min(t, a + 2000))
        h, x, want = cut(part)
        for k in ("pre_weight", "post_weight") + (("gate",) if gate == "channel" else ()):
            v, e = sums.get(k, (0, 0))
            sums[k] = (v + want[k].v, e + want[k].e)
        if a in (0, t // 4000 * 2000) or part.stop == t:
            check(hidden[part], h, a), check(back.residual[part], want["residual"], a)
            for q in (normed if gather else [normed]):
                check(q[part], x, a)
            for q in (back.partials if partials == "ranks" else [back.partials]):
                check(q[part], want["partials"], a)
            if gate in ("token", "full"):
                check(back.gate[part], want["gate"], a)
    for k, (v, e) in sums.items():
        check(getattr(back, k), B(v, 1.25 * e), k)


# ---- inside other parts of torch ------------------------------------------------------------------------------------

def small_block(g, r):
    def f(x, w, v):
        y = g.combine(torch.tanh(g.dispatch(x * 2, r)), r, w)
        hidden, normed = g.reduce_norm([y, x, y, x], x, pre_weight=v, post_weight=v, gate=v, gather=False)
        return hidden + normed
    return f


def small_inputs():
    return (randn(2, 60, 72).requires_grad_(True), torch.softmax(randn(3, 60, 2), 1).requires_grad_(True),
            randn(4, 72, mean=1.0, scale=0.1).requires_grad_(True))


@pytest.mark.parametrize("reentrant", [False, True])
def test_under_activation_checkpointing(groups, reentrant):
    from torch.utils.checkpoint import checkpoint
    g = groups(4)
    f, leaves = small_block(g, g.route(choices(1, 60, 2, 8, 0.2), 8)), small_inputs()
    for t in leaves:
        t.grad = None
    f(*leaves).square().sum().backward()
    want = [t.grad.clone() for t in leaves]
    for t in leaves:
        t.grad = None
    checkpoint(f, *leaves, use_reentrant=reentrant).square().sum().backward()
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


def test_under_torch_compile(groups):
    """The graph breaks at the calls, which run as they are (no code is generated: the eager backend)."""
    g = groups(4)
    f, leaves = small_block(g, g.route(choices(1, 60, 2, 8, 0.2), 8)), small_inputs()
    out, got = f(*leaves), torch.compile(f, backend="eager")(*leaves)
    assert torch.equal(out, got)
    for a, b in zip(torch.autograd.grad(out.sum(), leaves), torch.autograd.grad(got.sum(), leaves)):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(torch.compile(f, backend="eager")(*leaves), out)


def test_two_threads_at_once(groups):
    """Each on a stream of its own."""
    import threading
    g, want, got, went_wrong = groups(4), {}, {}, []
    jobs = {i: (choices(i, 500 + 300 * i, 3, 8, 0.1), randn(i, 500 + 300 * i, 136)) for i in range(2)}

    def work(e, x):
        r = g.route(e, 8)
        return g.reduce_norm(g.combine(g.dispatch(x, r), r), x, pre_weight=x[0].contiguous(), gather=False)
    for i, job in jobs.items():
        want[i] = work(*job)
    torch.cuda.synchronize()

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = [work(*jobs[i]) for _ in range(30)]
                torch.cuda.current_stream().synchronize()
        except Exception as e:          # noqa: BLE001 (told to the test's own thread)
            went_wrong.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not went_wrong, went_wrong
    for i in jobs:
        assert all(torch.equal(a, b) for run_ in got[i] for a, b in zip(run_, want[i])), i


def test_the_most_slots_there_are(groups):
    """2^31 - 1 of them: expert 3 i mod 8 for slot i, so its row is the expert's first plus i / 8.  One element a row."""
    g, n, step = groups(4), 2 ** 31 - 1, 1 << 26
    ids = torch.empty(n, 1, dtype=torch.int32, device="cuda")
    x = torch.empty(n, 1, dtype=torch.float16, device="cuda")
    for a in range(0, n, step):
        i = torch.arange(a, min(n, a + step), device="cuda")
        ids[a:a + step, 0] = (3 * i % 8).int()
        x[a:a + step, 0] = (i % 2039).half()
    r = g.route(ids, 8)
    counts = [(n - first + 7) // 8 for first in range(8)]                     # of slots i = first mod 8
    per_expert = {3 * first % 8: c for first, c in enumerate(counts)}
    starts = np.concatenate([[0], np.cumsum([per_expert[e] for e in range(8)])])
    assert np.array_equal(r.offsets.cpu().numpy(), starts)
    first = torch.from_numpy(starts).cuda()
    rows = g.dispatch(x, r)
    for a in range(0, n, step):
        i = torch.arange(a, min(n, a + step), device="cuda")
        row = first[3 * i % 8] + i // 8
        assert torch.equal(r.row_of_slot[a:a + step, 0].long(), row), a
        assert torch.equal(r.slot_of_row[row].long(), i), a
        assert torch.equal(rows[row, 0], x[a:a + step, 0]), a
    del ids
    assert torch.equal(g.combine(rows, r), x)
    with pytest.raises(ValueError, match="2\\^31"):
        g.route(torch.empty(2 ** 30, 2, dtype=torch.int32, device="cuda"), 8)
