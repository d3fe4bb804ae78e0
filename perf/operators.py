"""The block operators of ``stragglar_amd.torch_emulation.EmulatedGroup``: cases, inputs, plain forms and exact values.

A transformer block over n emulated ranks, its tokens sharded over the ranks by rows:

* ``route``: every token's expert choices sorted by expert (stable, rank r owns experts [r * E / n, (r + 1) * E / n));
* ``dispatch``: every chosen copy of a token goes to its row in expert order, and back in the backward pass;
* ``combine``: a token's rows come back as their weighted sum; its gradients to rows and weights;
* ``reduce_norm``: the ranks' partial block outputs are summed, normed, gated, added to the scaled residual, normed for
  the next block and given to every rank; its gradients.

``own`` False: elementary torch operations in 32 bits.  ``own`` True: the calls a user makes.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
RESIDUAL_SCALE = 0.8125


def _tokens(op, direction, ranks, tokens, topk, experts, dim, dtype, drop, ids="i64", weights="f32"):
    return {"op": op, "direction": direction, "ranks": ranks, "tokens": tokens, "topk": topk, "experts": experts, "dim": dim,
            "dtype": dtype, "drop": drop, "ids": ids, "weights": weights}


def _norm(direction, ranks, tokens, dim, dtype, partials, gather, gate, weights):
    return {"op": "reduce_norm", "direction": direction, "ranks": ranks, "tokens": tokens, "dim": dim, "dtype": dtype,
            "partials": partials, "gather": gather, "gate": gate, "weights": weights}


def listed():
    cases = [
        # one decoding step of a small batch: the latency of a single sort
        ("route decode", _tokens("route", "forward", 8, 16, 8, 64, 0, "bf16", 0.0)),
        # a large training batch over many experts, some slots over capacity
        ("route batch", _tokens("route", "forward", 8, 131072, 8, 256, 0, "bf16", 0.02)),
        # one decoding step: a few tokens to their experts' rows
        ("dispatch decode", _tokens("dispatch", "forward", 8, 32, 8, 64, 2048, "bf16", 0.0)),
        # a training step's tokens to the experts and their gradients back
        ("dispatch training", _tokens("dispatch", "training", 8, 16384, 8, 128, 2048, "bf16", 0.0)),
        # rows that are no whole vectors, over capacity, two experts a token
        ("dispatch ragged", _tokens("dispatch", "forward", 4, 4099, 2, 8, 1001, "f16", 0.1, ids="i32")),
        # one decoding step: the experts' rows back to their tokens
        ("combine decode", _tokens("combine", "forward", 8, 32, 8, 64, 2048, "bf16", 0.0)),
        # a training step's expert outputs back, and the gradients of rows and weights
        ("combine training", _tokens("combine", "training", 8, 16384, 4, 64, 4096, "bf16", 0.0)),
        # 32-bit training with odd rows and dropped slots
        ("combine ragged f32", _tokens("combine", "training", 6, 2053, 6, 48, 1023, "f32", 0.1)),
        # one decoding step's block boundary: eight partial outputs of a few tokens
        ("norm decode", _norm("forward", 8, 8, 4096, "bf16", "ranks", True, "channel", "bf16")),
        # a long prompt's block boundary, every rank's copy written
        ("norm prompt", _norm("forward", 8, 8192, 4096, "bf16", "ranks", True, "channel", "bf16")),
        # a training step's block boundary with all its gradients
        ("norm training", _norm("training", 8, 4096, 4096, "bf16", "ranks", True, "channel", "f32")),
        # a finished block output (no partial sums), kept sharded, odd sizes, a gate for each token
        ("norm ragged", _norm("training", 6, 1537, 1001, "f16", "one", False, "token", "f32")),
    ]
    return [dict(c, name=name) for name, c in cases]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["route", "dispatch", "combine", "reduce_norm", "reduce_norm"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    ranks = rng.choice([3, 4, 6, 8, 8, 16])
    dim = _spread(rng, 64, 8192)
    if rng.random() < 0.6:
        dim = max(64, dim // 64 * 64)
    if op == "reduce_norm":
        partials = rng.choice(["ranks", "ranks", "one"])
        gather = rng.random() < 0.6
        copies = (ranks if partials == "ranks" else 1) + (ranks if gather else 1) + 2
        tokens = _spread(rng, 1, max(1, min(16384, (150 << 20) // (copies * dim))))
        return _norm(rng.choice(["forward", "training"]), ranks, tokens, dim, dtype, partials, gather,
                     rng.choice(["none", "channel", "token", "full"]), rng.choice(["f32", dtype]))
    experts = ranks * _spread(rng, 1, 512 // ranks)
    topk = min(experts, _spread(rng, 1, 10))
    drop = rng.choice([0.0, 0.0, 0.05, 0.3])
    ids = rng.choice(["i64", "i32"])
    if op == "route":
        return _tokens("route", "forward", ranks, _spread(rng, 1, 1048576 // topk), topk, experts, 0, "bf16", drop, ids)
    tokens = _spread(rng, 1, max(1, min(32768, (150 << 20) // ((topk + 1) * dim))))
    return _tokens(op, rng.choice(["forward", "training"]), ranks, tokens, topk, experts, dim, dtype, drop, ids, rng.choice(["f32", dtype]))


# ---- inputs ------------------------------------------------------------------------------------------------------

def _choices(case, g):
    """Distinct experts for each token, some experts asked for more often than others; a dropped slot is -1."""
    tokens, topk, experts = case["tokens"], case["topk"], case["experts"]
    liking = 0.5 * torch.randn(experts, device="cuda", generator=g)
    logits = torch.randn(tokens, experts, device="cuda", generator=g) + liking
    ids = logits.topk(topk, dim=1).indices
    if case["drop"]:
        ids = torch.where(torch.rand(tokens, topk, device="cuda", generator=g) < case["drop"], torch.full_like(ids, -1), ids)
    return ids.to(torch.int64 if case["ids"] == "i64" else torch.int32).contiguous()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + mean).to(dtype)

    s = {}
    if case["op"] == "reduce_norm":
        n, t, d, wt = case["ranks"], case["tokens"], case["dim"], DTYPES[case["weights"]]
        if case["partials"] == "ranks":
            s["partials"] = [normal(t, d, scale=n ** -0.5) for _ in range(n)]
        else:
            s["partials"] = normal(t, d)
        s["residual"] = normal(t, d)
        s["pre_weight"] = normal(d, dtype=wt, scale=0.1, mean=1.0)
        s["post_weight"] = normal(d, dtype=wt, scale=0.1, mean=1.0)
        shape = {"none": None, "channel": (d,), "token": (t, 1), "full": (t, d)}[case["gate"]]
        s["gate"] = None if shape is None else normal(*shape, dtype=wt, scale=0.2, mean=0.5)
        if case["direction"] == "training":
            s["grad_hidden"] = normal(t, d)
            s["grad_normed"] = normal(n, t, d, scale=n ** -0.5) if case["gather"] else normal(t, d)
        return s
    s["experts"] = _choices(case, g)
    t, k, d = case["tokens"], case["topk"], case["dim"]
    if case["op"] == "dispatch":
        s["tokens"] = normal(t, d)
        if case["direction"] == "training":
            s["grad"] = normal(t * k, d)
    elif case["op"] == "combine":
        s["rows"] = normal(t * k, d)
        s["weights"] = torch.softmax(torch.randn(t, k, device="cuda", generator=g), dim=1).to(DTYPES[case["weights"]])
        if case["direction"] == "training":
            s["grad"] = normal(t, d)
    return s


_groups = {}


def _group(ranks):
    if ranks not in _groups:
        from stragglar_amd.torch_emulation import EmulatedGroup
        _groups[ranks] = EmulatedGroup(ranks, algorithm="ring")
    return _groups[ranks]


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["group"] = _group(case["ranks"])
        s["routing"] = s["group"].route(s["experts"], case["experts"]) if case["op"] in ("dispatch", "combine") else None
    elif case["op"] in ("dispatch", "combine"):
        s["routing"] = _plain_route(s["experts"], case["experts"])
    s["case"] = case
    if case["direction"] == "training":
        for name in ("tokens", "rows", "weights", "residual", "pre_weight", "post_weight", "gate"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
        if case["op"] == "reduce_norm":
            for p in (s["partials"] if isinstance(s["partials"], list) else [s["partials"]]):
                p.requires_grad_(True)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------

def _plain_route(experts, num_experts):
    flat = experts.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= num_experts), torch.full_like(flat, num_experts), flat)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=num_experts + 1)
    offsets = (torch.cumsum(counts, 0) - counts).int()
    index = torch.arange(key.numel(), device=key.device)
    slots = torch.where(index < offsets[-1], order, torch.full_like(order, -1)).int()
    rows = torch.empty_like(order)
    rows[order] = index
    rows = torch.where(key < num_experts, rows, torch.full_like(rows, -1)).int()
    return rows.view(experts.shape), slots, offsets


def _plain_dispatch(x, routing):
    rows, slots, offsets = routing
    kept = slots >= 0
    token = torch.div(slots, rows.shape[1], rounding_mode="floor").clamp(min=0).long()
    return (x.float()[token] * kept.unsqueeze(1)).to(x.dtype)


def _plain_combine(r, routing, weights):
    rows = routing[0]
    kept = rows >= 0
    w = torch.where(kept, weights.float(), torch.zeros((), device=r.device))
    taken = r.float()[rows.clamp(min=0).long()]
    return (taken * w.unsqueeze(2)).sum(1).to(r.dtype)


def _plain_norm(x, weight):
    return x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * weight.float()


def _plain_reduce_norm(s):
    case = s["case"]
    p = s["partials"]
    y = p.float() if isinstance(p, torch.Tensor) else sum(q.float() for q in p)
    u = _plain_norm(y, s["post_weight"])
    if s["gate"] is not None:
        u = u * s["gate"].float()
    h = RESIDUAL_SCALE * s["residual"].float() + u
    x = _plain_norm(h, s["pre_weight"])
    if case["gather"]:                      # every rank's copy is rounded by itself, so that their gradients add in 32 bits
        x = x.unsqueeze(0).expand(case["ranks"], -1, -1)
    return h.to(s["residual"].dtype), x.to(s["residual"].dtype).contiguous()


# ---- one pass ----------------------------------------------------------------------------------------------------

def _wanted(s):
    p = s["partials"]
    return (p if isinstance(p, list) else [p]) + [s[k] for k in ("residual", "pre_weight", "post_weight", "gate") if s[k] is not None]


def run(s):
    case = s["case"]
    op, training = case["op"], case["direction"] == "training"
    if op == "route":
        if own:
            r = s["group"].route(s["experts"], case["experts"])
            return {"rows": r.row_of_slot, "slots": r.slot_of_row, "offsets": r.offsets}
        rows, slots, offsets = _plain_route(s["experts"], case["experts"])
        return {"rows": rows, "slots": slots, "offsets": offsets}
    if op == "dispatch":
        out = s["group"].dispatch(s["tokens"], s["routing"]) if own else _plain_dispatch(s["tokens"], s["routing"])
        if not training:
            return {"rows": out}
        return {"rows": out.detach(), "grad_tokens": torch.autograd.grad(out, s["tokens"], s["grad"])[0]}
    if op == "combine":
        call = s["group"].combine if own else _plain_combine
        out = call(s["rows"], s["routing"], s["weights"])
        if not training:
            return {"tokens": out}
        gr, gw = torch.autograd.grad(out, (s["rows"], s["weights"]), s["grad"])
        return {"tokens": out.detach(), "grad_rows": gr, "grad_weights": gw}
    if own:
        hidden, normed = s["group"].reduce_norm(s["partials"], s["residual"], pre_weight=s["pre_weight"], post_weight=s["post_weight"],
                                                gate=s["gate"], residual_scale=RESIDUAL_SCALE, eps=EPS, gather=case["gather"])
    else:
        hidden, normed = _plain_reduce_norm(s)
    if not training:
        return {"hidden": hidden, "normed": normed}
    grads = torch.autograd.grad((hidden, normed), _wanted(s), (s["grad_hidden"], s["grad_normed"]))
    return {"hidden": hidden.detach(), "normed": normed.detach(), "grads": list(grads)}


def work(case):
    es, t = SIZE[case["dtype"]], case["tokens"]
    training = case["direction"] == "training"
    if case["op"] == "reduce_norm":
        d, n = case["dim"], case["ranks"]
        ws = SIZE[case["weights"]]
        src, dst = (n if case["partials"] == "ranks" else 1), (n if case["gather"] else 1)
        gate = {"none": 0, "channel": d, "token": t, "full": t * d}[case["gate"]] * ws
        b = (src + dst + 2) * t * d * es + 2 * d * ws + gate
        f = (src + 10) * t * d
        if training:
            b += (src + dst + 2) * t * d * es + 2 * d * ws + gate
            f += (dst + 25) * t * d
        return {"bytes": b, "flops": f}
    n, ids = t * case["topk"], 8 if case["ids"] == "i64" else 4
    if case["op"] == "route":
        return {"bytes": n * (ids + 8) + 4 * (case["experts"] + 1), "flops": n}
    d, ws = case["dim"], SIZE[case["weights"]]
    b = (n + t) * d * es + 4 * n
    if case["op"] == "dispatch":
        return {"bytes": b * 2 - 4 * n if training else b, "flops": n * d if training else 0}
    b += n * ws
    return {"bytes": b + (n + t) * d * es + n * ws if training else b, "flops": (5 if training else 2) * n * d}


# ---- exact values ------------------------------------------------------------------------------------------------

def _exact_route(experts, num_experts):
    """By counting, expert after expert, on the host."""
    import numpy as np
    flat = experts.reshape(-1).cpu().numpy().astype(np.int64)
    rows = np.full(flat.size, -1, np.int64)
    slots = np.full(flat.size, -1, np.int64)
    offsets = [0]
    for e in range(num_experts):
        mine = np.flatnonzero(flat == e)
        rows[mine] = offsets[-1] + np.arange(mine.size)
        slots[offsets[-1]:offsets[-1] + mine.size] = mine
        offsets.append(offsets[-1] + mine.size)
    dev = experts.device
    return torch.from_numpy(rows).to(dev).view(experts.shape), torch.from_numpy(slots).to(dev), torch.tensor(offsets, device=dev)


def _mean_square(x):
    return (x * x).sum(1, keepdim=True) / x.shape[1]


def exact(case, seed):
    s = _inputs(case, seed)
    training = case["direction"] == "training"
    if case["op"] == "reduce_norm":
        return _exact_reduce_norm(case, s, training)
    rows, slots, offsets = _exact_route(s["experts"], case["experts"])
    if case["op"] == "route":
        return {"rows": rows, "slots": slots, "offsets": offsets}
    total, k = int(offsets[-1]), case["topk"]
    row_token = torch.div(slots[:total], k, rounding_mode="floor")
    if case["op"] == "dispatch":
        x = s["tokens"].double()
        out = torch.zeros(slots.numel(), x.shape[1], dtype=torch.float64, device=x.device)
        out[:total] = x[row_token]
        if not training:
            return {"rows": out}
        g = torch.zeros_like(x)
        for j in range(k):
            has = rows[:, j] >= 0
            g[has] += s["grad"].double()[rows[has, j]]
        return {"rows": out, "grad_tokens": g}
    r, w = s["rows"].double(), s["weights"].double()
    y = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device=r.device)
    for j in range(k):
        has = rows[:, j] >= 0
        y[has] += w[has, j].unsqueeze(1) * r[rows[has, j]]
    if not training:
        return {"tokens": y}
    g = s["grad"].double()
    row_weight = w.reshape(-1)[slots[:total]]
    gr = torch.zeros_like(r)
    gr[:total] = g[row_token] * row_weight.unsqueeze(1)
    gw = torch.zeros_like(w)
    for j in range(k):
        has = rows[:, j] >= 0
        gw[has, j] = (g[has] * r[rows[has, j]]).sum(1)
    return {"tokens": y, "grad_rows": gr, "grad_weights": gw}


def _exact_reduce_norm(case, s, training):
    n = case["ranks"]
    p = s["partials"] if isinstance(s["partials"], list) else [s["partials"]]
    y = torch.zeros_like(s["residual"], dtype=torch.float64)
    for q in p:
        y += q.double()
    wp, wq = s["post_weight"].double(), s["pre_weight"].double()
    gate = torch.ones(1, dtype=torch.float64, device=y.device) if s["gate"] is None else s["gate"].double()
    r1 = 1.0 / torch.sqrt(_mean_square(y) + EPS)
    yhat = y * r1
    h = RESIDUAL_SCALE * s["residual"].double() + gate * (yhat * wp)
    r2 = 1.0 / torch.sqrt(_mean_square(h) + EPS)
    hhat = h * r2
    x = hhat * wq
    normed = x.unsqueeze(0).expand(n, -1, -1) if case["gather"] else x
    if not training:
        return {"hidden": h, "normed": normed}
    gx = s["grad_normed"].double().sum(0) if case["gather"] else s["grad_normed"].double()
    a = gx * wq
    gh = s["grad_hidden"].double() + r2 * (a - hhat * ((a * hhat).sum(1, keepdim=True) / y.shape[1]))
    gu = gh * gate
    b = gu * wp
    gy = r1 * (b - yhat * ((b * yhat).sum(1, keepdim=True) / y.shape[1]))
    grads = [gy] * len(p) + [RESIDUAL_SCALE * gh, (gx * hhat).sum(0), (gu * yhat).sum(0)]
    if s["gate"] is not None:
        gg = gh * yhat * wp
        grads.append({"channel": lambda: gg.sum(0), "token": lambda: gg.sum(1, keepdim=True), "full": lambda: gg}[case["gate"]]())
    return {"hidden": h, "normed": normed, "grads": grads}
