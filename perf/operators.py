"""Cases of the expert and matrix-update operators, for timing and for comparison: rows sorted by expert and back (`experts.expert_plan`,
`expert_dispatch`, `expert_combine`), the experts' products (`experts.expert_linear`), the orthogonalised update (`optim.newton_schulz`)
and the optimizer step that applies it (`optim.HipMuon`).

`run` computes a case in elementary torch operations (own = False) or through the framework (own = True); `exact` gives the same outputs
from the definitions in 64 bits.  Sizes: 16 sub-fields, 64-wide layers and batches of 65536 are this repository's own; the wide ones are
generic."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one query point blended from its two nearest of 16 sub-fields: latency alone
        dict(name="exchange_one_row", op="exchange", rows=1, k=2, experts=16, width=64, dtype="f32", drop=0.0, skew=False, grad=False),
        # a training batch of 65536 rays, two sub-fields each, 64 features; one assignment in twenty lies outside every sub-field
        dict(name="exchange_subfields", op="exchange", rows=65536, k=2, experts=16, width=64, dtype="f32", drop=0.05, skew=False, grad=True),
        # odd everything: rows whose length is no multiple of a vector, crowded experts, dropped assignments
        dict(name="exchange_odd", op="exchange", rows=10007, k=3, experts=37, width=195, dtype="f16", drop=0.1, skew=True, grad=True),
        # the training exchange of a wide mixture layer: 131072 assignments of 2048 features
        dict(name="exchange_wide", op="exchange", rows=16384, k=8, experts=128, width=2048, dtype="bf16", drop=0.0, skew=False, grad=True),
        # answering single tokens: a few rows, each expert's weights read for one row or two
        dict(name="linear_few_rows", op="linear", rows=16, experts=64, n_in=1024, n_out=2048, dtype="bf16", bias=False, skew=False, tail=0, grad=False),
        # one 64 -> 64 layer of 16 sub-fields, trained on 131072 points
        dict(name="linear_subfields", op="linear", rows=131072, experts=16, n_in=64, n_out=64, dtype="f32", bias=True, skew=False, tail=1000, grad=True),
        # odd widths, crowded and empty experts
        dict(name="linear_odd", op="linear", rows=5003, experts=7, n_in=129, n_out=385, dtype="f16", bias=True, skew=True, tail=17, grad=True),
        # a wide expert layer in training
        dict(name="linear_wide", op="linear", rows=65536, experts=32, n_in=2048, n_out=1024, dtype="bf16", bias=False, skew=False, tail=0, grad=True),
        # three tall gradients of odd size
        dict(name="orthogonalise_odd", op="orthogonalise", batch=3, m=385, n=129, dtype="bf16"),
        # the gradient of one wide layer
        dict(name="orthogonalise_wide", op="orthogonalise", batch=1, m=2048, n=4096, dtype="f32"),
        # the step over the layers of 16 sub-fields, stacked by layer
        dict(name="muon_subfields", op="muon", shapes="16x64x40,16x80x64,16x64x64,16x64x47,16x3x64", dtype="f32", nesterov=True),
        # the step over one wide expert layer
        dict(name="muon_wide", op="muon", shapes="8x1024x2048", dtype="f32", nesterov=True),
    ]


def _log(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["exchange", "linear", "orthogonalise", "muon"])
    if op == "exchange":
        k = rng.randint(1, 8)
        width = _log(rng, 1, 2048)
        rows = _log(rng, 1, min(65536, 16384 * 8 * 2048 // (k * width)))
        return dict(op=op, rows=rows, k=k, experts=_log(rng, k, 256), width=width, dtype=rng.choice(sorted(DTYPES)) if width * rows < 1 << 23 else "bf16",
                    drop=rng.choice([0.0, 0.05, 0.5]), skew=rng.random() < 0.5, grad=rng.random() < 0.7)
    if op == "linear":
        n_in, n_out, experts = _log(rng, 8, 2048), _log(rng, 8, 2048), _log(rng, 1, 64)
        dtype = rng.choice(sorted(DTYPES))
        most = 65536 * 2048 * 1024 // (4 if dtype == "f32" else 1)
        rows = _log(rng, 1, min(131072, most // (n_in * n_out)))
        return dict(op=op, rows=rows, experts=experts, n_in=n_in, n_out=n_out, dtype=dtype, bias=rng.random() < 0.5, skew=rng.random() < 0.3,
                    tail=rng.randint(0, rows // 8), grad=rng.random() < 0.7)
    m, n = _log(rng, 4, 4096), _log(rng, 4, 4096)
    small, large = min(m, n), max(m, n)
    most = 2048 * 2048 * 4096 // (small * small * large)
    if most < 1:
        m, n, most = 2048, rng.randint(1024, 4096), 1
    batch = _log(rng, 1, min(64, most))
    if op == "orthogonalise":
        return dict(op=op, batch=batch, m=m, n=n, dtype=rng.choice(sorted(DTYPES)))
    shapes = [(batch, m, n)]
    while len(shapes) < 3 and rng.random() < 0.5:
        shapes.append((rng.randint(1, 16), rng.randint(4, 128), rng.randint(4, 128)))
    return dict(op=op, shapes=",".join("%dx%dx%d" % s for s in shapes), dtype="f32", nesterov=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "exchange":
        N, k, E, D = case["rows"], case["k"], case["experts"], case["width"]
        scores = _normal(gen, N, E)
        if case["skew"]:  # a few experts are wanted by nearly everybody, the last ones by nobody
            scores = scores - 6.0 * torch.arange(E, device="cuda") / E
        value, ids = torch.topk(scores, k, dim=1)
        if case["drop"]:
            ids = torch.where(torch.rand(N, k, generator=gen, device="cuda") < case["drop"], torch.full_like(ids, -1), ids)
        state.update(ids=ids, weights=torch.softmax(value, 1), x=_normal(gen, N, D, dtype=dtype), answers=_normal(gen, N * k, D, dtype=dtype))
        if case["grad"]:
            state.update(dy=_normal(gen, N, D, dtype=dtype), drows=_normal(gen, N * k, D, dtype=dtype))
            state["x"].requires_grad_(True), state["answers"].requires_grad_(True), state["weights"].requires_grad_(True)
    elif case["op"] == "linear":
        M, E, I, O = case["rows"], case["experts"], case["n_in"], case["n_out"]
        share = torch.arange(E, 0, -1).double() ** 3 if case["skew"] else torch.ones(E).double()
        chosen = torch.multinomial(share, M - case["tail"], replacement=True, generator=torch.Generator().manual_seed(seed))
        counts = torch.bincount(chosen, minlength=E)
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32)
        state.update(offsets=offsets.cuda(), longest=int(counts.max()), x=_normal(gen, M, I, dtype=dtype),
                     weight=_normal(gen, E, O, I, dtype=dtype, scale=1 / math.sqrt(I)), bias=_normal(gen, E, O, dtype=dtype) if case["bias"] else None)
        if case["grad"]:
            state["dy"] = _normal(gen, M, O, dtype=dtype)
            state["x"].requires_grad_(True), state["weight"].requires_grad_(True)
            if case["bias"]:
                state["bias"].requires_grad_(True)
    elif case["op"] == "orthogonalise":
        state["g"] = _normal(gen, case["batch"], case["m"], case["n"], dtype=dtype, scale=1e-3)
    else:
        state["params"] = [_normal(gen, *s, scale=1 / math.sqrt(s[-1])) for s in _shapes(case)]
        state["grads"] = [_normal(gen, *s, scale=1e-3) for s in _shapes(case)]
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_exchange(s):
    E, grad = s["case"]["experts"], s["case"]["grad"]
    ids, w, x, answers = s["ids"], s["weights"].detach(), s["x"].detach(), s["answers"].detach()
    N, k = ids.shape
    flat = ids.reshape(-1)
    held = (flat >= 0) & (flat < E)
    key, order = torch.sort(torch.where(held, flat, torch.full_like(flat, E)), stable=True)
    offsets = torch.searchsorted(key, torch.arange(E + 1, device=key.device)).to(torch.int32)
    src = torch.where(key < E, order, torch.full_like(order, -1)).to(torch.int32)
    place = torch.empty_like(order)
    place[order] = torch.arange(N * k, device=order.device)
    dst = torch.where(held, place, torch.full_like(place, -1)).reshape(N, k).to(torch.int32)
    there = (key < E)[:, None]
    rows = torch.where(there, x[order // k], torch.zeros_like(x[:1]))
    at = place.reshape(N, k)
    seen = held.reshape(N, k, 1)
    mine = torch.where(seen, answers[at].float(), torch.zeros((), device=x.device))
    y = (mine * w[..., None]).sum(1).to(x.dtype)
    if not grad:
        return offsets, src, dst, rows, y
    dy = s["dy"].float()
    dw = torch.where(seen[..., 0], (mine * dy[:, None, :]).sum(2), torch.zeros((), device=x.device))
    danswers = torch.where(there, dy[order // k] * w.reshape(-1)[order][:, None], torch.zeros((), device=x.device)).to(x.dtype)
    dx = torch.where(seen, s["drows"][at].float(), torch.zeros((), device=x.device)).sum(1).to(x.dtype)
    return offsets, src, dst, rows, y, danswers, dw, dx


def _plain_linear(s):
    x, weight, bias, offsets = s["x"].detach().float(), s["weight"].detach().float(), s["bias"], s["offsets"].long()
    out_type = s["x"].dtype
    # every expert's rows, filled up with zeros to the longest expert's length
    at = offsets[:-1, None] + torch.arange(s["longest"], device=x.device)
    there = at < offsets[1:, None]
    at = torch.where(there, at, torch.zeros_like(at))
    zero = torch.zeros((), device=x.device)
    xe = torch.where(there[..., None], x[at], zero)
    ye = torch.matmul(xe, weight.transpose(1, 2).contiguous())
    if bias is not None:
        ye = ye + bias.detach().float()[:, None, :]
    y = torch.zeros(x.shape[0], weight.shape[1], device=x.device)
    y[at[there]] = ye[there]
    if not s["case"]["grad"]:
        return (y.to(out_type),)
    dye = torch.where(there[..., None], s["dy"].float()[at], zero)
    dxe = torch.matmul(dye, weight)
    dx = torch.zeros_like(x)
    dx[at[there]] = dxe[there]
    dweight = torch.matmul(dye.transpose(1, 2).contiguous(), xe)
    out = (y.to(out_type), dx.to(out_type), dweight.to(out_type))
    return out if bias is None else out + (dye.sum(1).to(out_type),)


def _plain_orthogonal(g):
    """the matrices' singular values pushed to about one by an odd polynomial, five times over"""
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS).float()
    for _ in range(NS_STEPS):
        s = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return x.transpose(-2, -1).contiguous() if tall else x


def _plain_muon(s):
    nesterov = s["case"]["nesterov"]
    bufs = s.setdefault("bufs", [torch.zeros_like(p) for p in s["params"]])
    for p, g, buf in zip(s["params"], s["grads"], bufs):
        buf.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
        update = _plain_orthogonal((1 - MOMENTUM) * g + MOMENTUM * buf if nesterov else buf)
        p.mul_(1 - LR * DECAY).sub_(update, alpha=LR * math.sqrt(max(1.0, p.shape[-2] / p.shape[-1])))
    return s["params"] + bufs


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_exchange(s):
    from presight_amd import experts

    plan = experts.expert_plan(s["ids"], s["case"]["experts"])
    rows = experts.expert_dispatch(s["x"], plan)
    y = experts.expert_combine(s["answers"], s["weights"], plan)
    if not s["case"]["grad"]:
        return plan.offsets, plan.src, plan.dst, rows, y
    dx, danswers, dw = torch.autograd.grad([rows, y], [s["x"], s["answers"], s["weights"]], [s["drows"], s["dy"]])
    return plan.offsets, plan.src, plan.dst, rows.detach(), y.detach(), danswers, dw, dx


def _own_linear(s):
    from presight_amd import experts

    y = experts.expert_linear(s["x"], s["weight"], s["bias"], s["offsets"])
    if not s["case"]["grad"]:
        return (y,)
    leaves = [s["x"], s["weight"]] + ([s["bias"]] if s["bias"] is not None else [])
    return (y.detach(),) + torch.autograd.grad(y, leaves, s["dy"])


def _own_muon(s):
    from presight_amd import optim

    if "opt" not in s:
        params = [torch.nn.Parameter(p) for p in s["params"]]
        s["opt"] = optim.HipMuon(params, lr=LR, momentum=MOMENTUM, nesterov=s["case"]["nesterov"], weight_decay=DECAY, ns_steps=NS_STEPS,
                                 ns_coefficients=COEFFICIENTS, eps=NS_EPS)
        for p, g in zip(params, s["grads"]):
            p.grad = g
    s["opt"].step()
    return [p.detach() for p in s["opt"].params] + s["opt"].momentum_buffers


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "exchange":
            return _own_exchange(state)
        if op == "linear":
            return _own_linear(state)
        if op == "muon":
            return _own_muon(state)
        from presight_amd import optim

        return optim.newton_schulz(state["g"], steps=NS_STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    if op == "exchange":
        return _plain_exchange(state)
    if op == "linear":
        return _plain_linear(state)
    if op == "muon":
        return _plain_muon(state)
    return _plain_orthogonal(state["g"]).to(state["g"].dtype)


# ------------------------------------------------------------------------------------------------ work
def _ns_flops(batch, m, n):
    """per step: the product of the matrix with its transpose and that product's square, which are symmetric (half of each is computed),
    and their product with the matrix"""
    s, t = min(m, n), max(m, n)
    return batch * NS_STEPS * (s * (s + 1) * t + s * s * (s + 1) + 2 * s * s * t)


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "exchange":
        N, k, D = case["rows"], case["k"], case["width"]
        kept = N * k * (1 - case["drop"])
        moved = size * (N * D + N * k * D + kept * D + N * D) + N * k * (8 + 4 + 4 + 4) + 4 * (case["experts"] + 1)
        flops = 2 * kept * D
        if case["grad"]:
            moved += size * (N * D + N * k * D + kept * D + N * D) + N * k * 4
            flops += 4 * kept * D
        return {"bytes": moved, "flops": flops}
    if case["op"] == "linear":
        M, I, O = case["rows"], case["n_in"], case["n_out"]
        kept, E = M - case["tail"], case["experts"]
        used = min(E, kept)
        moved = size * (kept * I + used * O * I + M * O + (used * O if case["bias"] else 0)) + 4 * (E + 1)
        flops = 2.0 * kept * I * O
        if case["grad"]:
            moved += size * (kept * O + M * I + E * O * I + (E * O if case["bias"] else 0))
            flops *= 3
        return {"bytes": moved, "flops": flops}
    if case["op"] == "orthogonalise":
        return {"bytes": 2 * size * case["batch"] * case["m"] * case["n"], "flops": _ns_flops(case["batch"], case["m"], case["n"])}
    shapes = _shapes(case)
    return {"bytes": sum(5 * 4 * b * m * n for b, m, n in shapes), "flops": sum(_ns_flops(b, m, n) for b, m, n in shapes)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_orthogonal(g):
    """x p(x^T x) with the polynomial applied from the short side: U p(S) V^T, whichever side the products are formed on"""
    a, b, c = COEFFICIENTS
    x = g.double()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + NS_EPS)
    wide = x.shape[-1] > x.shape[-2]
    for _ in range(NS_STEPS):
        t = x.transpose(-2, -1).contiguous()
        gram = torch.matmul(x, t) if wide else torch.matmul(t, x)
        poly = torch.matmul(gram, c * gram + b * torch.eye(gram.shape[-1], device=x.device, dtype=x.dtype)) \
            + a * torch.eye(gram.shape[-1], device=x.device, dtype=x.dtype)
        x = torch.matmul(poly, x) if wide else torch.matmul(x, poly)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "orthogonalise":
        return _exact_orthogonal(s["g"])
    if case["op"] == "muon":
        params, bufs = [], []
        for p, g in zip(s["params"], s["grads"]):
            buf = (1 - MOMENTUM) * g.double()  # of a momentum that starts at zero
            u = _exact_orthogonal((1 - MOMENTUM) * g.double() + MOMENTUM * buf if case["nesterov"] else buf)
            params.append((1 - LR * DECAY) * p.double() - LR * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5 * u)
            bufs.append(buf)
        return params + bufs
    if case["op"] == "linear":
        x, w = s["x"].detach().double(), s["weight"].detach().double()
        b = s["bias"].detach().double() if case["bias"] else None
        cut = s["offsets"].tolist()
        y = torch.zeros(x.shape[0], w.shape[1], device=x.device, dtype=x.dtype)
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(w.shape[:2], device=x.device, dtype=x.dtype)
        for e in range(case["experts"]):
            lo, hi = cut[e], cut[e + 1]
            y[lo:hi] = x[lo:hi] @ w[e].T + (b[e] if b is not None else 0)
            if case["grad"]:
                dy = s["dy"][lo:hi].double()
                dx[lo:hi], dw[e], db[e] = dy @ w[e], dy.T @ x[lo:hi], dy.sum(0)
        return ((y, dx, dw, db) if case["bias"] else (y, dx, dw)) if case["grad"] else (y,)
    # exchange: per assignment, in the rows' own order
    ids, w = s["ids"], s["weights"].detach().double()
    N, k, E, D = case["rows"], case["k"], case["experts"], case["width"]
    flat = ids.reshape(-1).cpu()
    kept = torch.nonzero((flat >= 0) & (flat < E)).reshape(-1)
    src = kept[torch.argsort(flat[kept] * (N * k) + kept)].to(ids.device)  # expert first, then the assignment's own number
    P = src.numel()
    x, answers = s["x"].detach().double(), s["answers"].detach().double()
    rows = torch.zeros(N * k, D, device=x.device, dtype=x.dtype)
    rows[:P] = x[src // k]
    spread = torch.zeros(N * k, D, device=x.device, dtype=x.dtype)
    spread[src] = answers[:P] * w.reshape(-1)[src][:, None]
    y = spread.reshape(N, k, D).sum(1)
    if not case["grad"]:
        return None, None, None, rows, y
    dy = s["dy"].double()
    danswers = torch.zeros_like(rows)
    danswers[:P] = dy[src // k] * w.reshape(-1)[src][:, None]
    dw = torch.zeros(N * k, device=x.device, dtype=x.dtype)
    dw[src] = (answers[:P] * dy[src // k]).sum(1)
    spread.zero_()
    spread[src] = s["drows"].double()[:P]
    return None, None, None, rows, y, danswers, dw.reshape(N, k), spread.reshape(N, k, D).sum(1)
