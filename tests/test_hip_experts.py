"""Rows sorted by expert and back, and the experts' linear layers (presight_amd.experts), against plain 64-bit restatements.

Tolerances.  Layouts are compared exactly.  A sum of n terms t_i held in fp32 in any order is off by at most n * 2^-23 * sum |t_i| (each of
the n additions by one unit in the last place of a partial sum that sum |t_i| bounds; matrix instructions are given that whole unit
instead of the half of round-to-nearest), and the one rounding to the output type T by finfo(T).eps / 2 of the value, or by half a step of T's
subnormals (finfo(T).smallest_normal * eps / 2)."""
import pytest
import torch

from presight_amd import experts

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch.device("cuda:0")


def within(got, ref, terms, absum):
    """|got - ref| <= one rounding to got's type + `terms` fp32 additions over terms of absolute sum `absum`"""
    f = torch.finfo(got.dtype)
    bound = (ref.abs() * f.eps / 2 + f.smallest_normal * f.eps / 2 + (1 + f.eps) * terms * 2.0 ** -23 * absum).cpu()
    err = (got.detach().cpu().double() - ref.cpu()).abs()
    assert got.shape == ref.shape
    assert torch.isfinite(err).all() and (err <= bound).all(), f"worst {float((err / bound.clamp_min(1e-300)).max()):.2f} x the bound"


def plan_ref(ids, E):
    """the stable sort, assignment by assignment"""
    N, k = ids.shape
    flat = ids.reshape(-1).tolist()
    order = sorted((f for f in range(N * k) if 0 <= flat[f] < E), key=lambda f: (flat[f], f))
    dst = [-1] * (N * k)
    for p, f in enumerate(order):
        dst[f] = p
    counts = [0] * E
    for f in order:
        counts[flat[f]] += 1
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return t(offsets), t(order + [-1] * (N * k - len(order))), t(dst).reshape(N, k)


def some_ids(N, k, E, seed, kind):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, E, (N, k), generator=g)
    if kind == "dropped":
        ids[torch.rand(N, k, generator=g) < 0.4] = -1
        ids[torch.rand(N, k, generator=g) < 0.1] = E + 3
        ids[: N // 3] = -1  # whole rows that nobody takes
    elif kind == "one":
        ids[:] = E // 2
    elif kind == "nobody":
        ids[:] = -1
    elif kind == "twice":
        ids[:] = ids[:, :1]
    return ids


# ------------------------------------------------------------------------------------------------ refusals (no GPU needed)
def test_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        experts.expert_plan(torch.zeros(4, 2, dtype=torch.int64), 3)
    plan = experts.ExpertPlan(torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32), 3)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        experts.expert_dispatch(torch.zeros(4, 5), plan)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        experts.expert_combine(torch.zeros(8, 5), torch.zeros(4, 2), plan)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        experts.expert_linear(torch.zeros(8, 5), torch.zeros(3, 6, 5), None, plan)
    with pytest.raises(TypeError):
        experts.expert_dispatch(torch.zeros(4, 5), plan.dst)


def test_library_refuses_bad_sizes():
    """the C entries check what they can before anything is launched: an error code and a text, no launch"""
    from presight_amd._lib import check, lib

    h = lib()
    for rc in (h.ps_expert_plan(None, 0, 8, 0, None, None, None, None, None), h.ps_expert_plan(None, 0, 8, 1025, None, None, None, None, None),
               h.ps_expert_plan(None, 0, -1, 4, None, None, None, None, None), h.ps_expert_plan(None, 0, 1 << 31, 4, None, None, None, None, None),
               h.ps_expert_plan(None, 0, 8, 4, None, None, None, None, None),
               h.ps_expert_dispatch(None, 4, None, None, 4, 0, 4, 0, None, None), h.ps_expert_dispatch(None, 4, None, None, 4, 2, 4, 0, None, None),
               h.ps_expert_combine(None, 4, None, None, 1 << 30, 2, 4, 0, None, None),
               h.ps_expert_linear_fwd(None, 4, None, None, None, 8, 2, 5, 4, 0, None, None, None),
               h.ps_expert_linear_fwd(None, 5, None, None, None, 8, 2, 5, 4, 0, None, None, None),
               h.ps_expert_linear_dx(None, 3, None, None, 8, 2, 5, 4, 0, None, None, None),
               h.ps_expert_linear_dw(None, 4, None, 5, None, 8, 0, 5, 4, 0, None, None, None, None)):
        assert rc != 0
    with pytest.raises(Exception, match="experts"):
        check(h.ps_expert_plan(None, 0, 8, 0, None, None, None, None, None), "ps_expert_plan")


def test_plan_made_by_hand_is_checked():
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    experts.ExpertPlan(i32(4), i32(8), i32(4, 2), 3)
    for bad in ((i32(5), i32(8), i32(4, 2)), (i32(4), i32(7), i32(4, 2)), (i32(4), i32(8), i32(8))):
        with pytest.raises(ValueError):
            experts.ExpertPlan(*bad, 3)
    for bad in ((i32(4).long(), i32(8), i32(4, 2)), (i32(4), i32(8), i32(2, 4).t()), (i32(8)[::2], i32(8), i32(4, 2))):
        with pytest.raises(TypeError):
            experts.ExpertPlan(*bad, 3)


@pytest.mark.gpu
def test_refusals(dev):
    ids = torch.zeros(6, 2, dtype=torch.int64, device=dev)
    for bad, exc in ((ids.float(), TypeError), (ids[:, 0], ValueError), (ids[:, :0], ValueError)):
        with pytest.raises(exc):
            experts.expert_plan(bad, 4)
    for E in (0, 1025):
        with pytest.raises(ValueError):
            experts.expert_plan(ids, E)
    plan = experts.expert_plan(ids, 4)
    x = torch.zeros(6, 8, device=dev)
    with pytest.raises(ValueError):
        experts.expert_dispatch(x[:5], plan)
    with pytest.raises(TypeError):
        experts.expert_dispatch(x.double(), plan)
    with pytest.raises(ValueError):
        experts.expert_combine(x, None, plan)
    with pytest.raises(ValueError):
        experts.expert_combine(torch.zeros(12, 8, device=dev), torch.zeros(6, 3, device=dev), plan)
    with pytest.raises(RuntimeError, match="GPU"):
        experts.expert_combine(torch.zeros(12, 8, device=dev), torch.zeros(6, 2), plan)
    rows, w = torch.zeros(12, 8, device=dev), torch.zeros(4, 5, 8, device=dev)
    for args, exc in (((rows, w[:, :, :7], None, plan), ValueError), ((rows, w.half(), None, plan), TypeError), ((rows, w[:3], None, plan), ValueError),
                      ((rows, w, torch.zeros(4, 4, device=dev), plan), ValueError), ((rows[:11], w, None, plan), ValueError),
                      ((rows, w, None, plan.offsets.float()), ValueError), ((rows, w, None, plan.offsets[:4]), ValueError),
                      ((rows, w[:, :0], None, plan), ValueError)):
        with pytest.raises(exc):
            experts.expert_linear(*args)


# ------------------------------------------------------------------------------------------------ the layout
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["all", "dropped", "one", "nobody", "twice"])
@pytest.mark.parametrize("N,k,E", [(0, 2, 5), (1, 1, 1), (1, 8, 16), (63, 1, 3), (65, 3, 64), (1000, 2, 16), (4096, 2, 37), (4097, 2, 1024),
                                   (3001, 5, 1), (20000, 4, 130)])
def test_plan(dev, N, k, E, kind):
    ids = some_ids(N, k, E, N + E, kind)
    want = plan_ref(ids, E)
    for t in (torch.int64, torch.int32):
        plan = experts.expert_plan(ids.to(t).to(dev), E)
        for got, ref in zip((plan.offsets, plan.src, plan.dst), want):
            assert got.dtype == torch.int32 and torch.equal(got.cpu(), ref)
    assert int(plan.held) == int(want[0][-1])


@pytest.mark.gpu
def test_plan_of_a_million_and_strided_ids(dev):
    """many counting workgroups, chunks longer than their least; ids that are a slice of a wider tensor"""
    g = torch.Generator().manual_seed(5)
    wide = torch.randint(-1, 300, (400_000, 5), generator=g)
    ids = wide[:, 1:4]
    plan = experts.expert_plan(wide.to(dev)[:, 1:4], 300)
    flat = ids.reshape(-1)
    key, order = torch.sort(torch.where(flat >= 0, flat, 300), stable=True)
    held = int((key < 300).sum())
    assert torch.equal(plan.src.cpu()[:held].long(), order[:held]) and bool((plan.src[held:] == -1).all())
    assert torch.equal(plan.offsets.cpu().long(), torch.searchsorted(key, torch.arange(301)))
    dst = torch.full_like(flat, -1)
    dst[order[:held]] = torch.arange(held)
    assert torch.equal(plan.dst.cpu().long().reshape(-1), dst)


# ------------------------------------------------------------------------------------------------ the exchange
def exchange_ref(ids, E, x, rows, w, dy, drows):
    """every output of the exchange, in 64 bits"""
    offsets, src, dst = plan_ref(ids, E)
    N, k = ids.shape
    held = int(offsets[-1])
    at = src[:held].long()
    sorted_x = torch.zeros(N * k, x.shape[1], dtype=torch.float64)
    sorted_x[:held] = x[at // k]
    wf = w.reshape(-1)
    spread, spread_abs = torch.zeros(N * k, x.shape[1], dtype=torch.float64), None
    spread[at] = rows[:held] * wf[at][:, None]
    spread_abs = spread.abs()
    drows_out = torch.zeros_like(sorted_x)
    drows_out[:held] = dy[at // k] * wf[at][:, None]
    dw, dw_abs = torch.zeros(N * k, dtype=torch.float64), torch.zeros(N * k, dtype=torch.float64)
    dw[at] = (rows[:held] * dy[at // k]).sum(1)
    dw_abs[at] = (rows[:held] * dy[at // k]).abs().sum(1)
    back = torch.zeros_like(spread)
    back[at] = drows[:held]
    shape = (N, k, x.shape[1])
    return dict(rows=sorted_x, y=spread.reshape(shape).sum(1), y_abs=spread_abs.reshape(shape).sum(1), drows=drows_out, dw=dw.reshape(N, k),
                dw_abs=dw_abs.reshape(N, k), dx=back.reshape(shape).sum(1), dx_abs=back.abs().reshape(shape).sum(1))


def exchange_case(dev, N, k, E, D, dtype, kind, seed=0, poison=True):
    g = torch.Generator().manual_seed(seed + 7 * N + D)
    ids = some_ids(N, k, E, seed + N, kind)
    T = TYPES[dtype]
    x, rows, dy, drows = (torch.randn(n, D, generator=g).to(T) for n in (N, N * k, N, N * k))
    w = torch.randn(N, k, generator=g)
    held = int(((ids >= 0) & (ids < E)).sum())
    ref = exchange_ref(ids, E, x.double(), rows.double(), w.double(), dy.double(), drows.double())
    if poison:  # what belongs to nobody is never read
        rows[held:], drows[held:] = float("nan"), float("inf")
        w = torch.where((ids >= 0) & (ids < E), w, torch.full_like(w, float("nan")))
    return ids, [t.to(dev) for t in (x, rows, w, dy, drows)], ref


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,k,E,D,kind", [(1, 1, 1, 1, "all"), (1, 2, 16, 64, "all"), (257, 3, 37, 195, "dropped"), (100, 8, 5, 2, "twice"),
                                          (77, 2, 9, 130, "nobody"), (64, 4, 300, 1028, "dropped"), (33, 1, 4, 4096, "one"), (5, 2, 3, 2056, "all")])
def test_exchange_and_gradients(dev, N, k, E, D, kind, dtype):
    ids, (x, rows, w, dy, drows), ref = exchange_case(dev, N, k, E, D, dtype, kind)
    for t in (x, rows, w):
        t.requires_grad_(True)
    plan = experts.expert_plan(ids.to(dev), E)
    got_rows = experts.expert_dispatch(x, plan)
    y = experts.expert_combine(rows, w, plan)
    assert torch.equal(got_rows.detach().cpu().double(), ref["rows"])
    within(y, ref["y"], k, ref["y_abs"])
    dx, da, dw = torch.autograd.grad([got_rows, y], [x, rows, w], [drows, dy])
    within(dx, ref["dx"], k, ref["dx_abs"])
    within(da, ref["drows"], 1, ref["drows"].abs())
    within(dw, ref["dw"], D + 6, ref["dw_abs"])
    assert y.dtype == da.dtype == dx.dtype == TYPES[dtype] and dw.dtype == torch.float32
    # one gradient at a time gives the same bits
    y = experts.expert_combine(rows, w.detach(), plan)
    assert torch.equal(torch.autograd.grad(y, rows, dy)[0], da)
    y = experts.expert_combine(rows.detach(), w, plan)
    assert torch.equal(torch.autograd.grad(y, w, dy)[0], dw)


@pytest.mark.gpu
def test_combine_without_weights_and_with_16_bit_ones(dev):
    ids, (x, rows, w, dy, drows), ref = exchange_case(dev, 90, 3, 11, 72, "bf16", "all")
    plan = experts.expert_plan(ids.to(dev), 11)
    rows.requires_grad_(True)
    y = experts.expert_combine(rows, None, plan)
    held = rows.detach().double().cpu()[plan.dst.cpu().long().reshape(-1)].reshape(90, 3, 72)
    within(y, held.sum(1), 3, held.abs().sum(1))
    assert torch.equal(torch.autograd.grad(y, rows, dy)[0].cpu(), dy.cpu()[plan.src.cpu().long() // 3])
    wh = w.half().requires_grad_(True)
    y = experts.expert_combine(rows, wh, plan)
    ref = exchange_ref(ids, 11, x.cpu().double(), rows.detach().cpu().double(), wh.detach().cpu().double(), dy.cpu().double(), drows.cpu().double())
    within(y, ref["y"], 3, ref["y_abs"])
    dw = torch.autograd.grad(y, wh, dy)[0]
    assert dw.dtype == torch.float16
    within(dw, ref["dw"], 72 + 6, ref["dw_abs"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_exchange_of_strided_and_unaligned_rows(dev, dtype):
    """rows at a distance, columns of a wider tensor at an odd start, a transposed tensor, an expanded gradient: the same bits as copies"""
    T = TYPES[dtype]
    g = torch.Generator().manual_seed(1)
    ids = some_ids(50, 2, 7, 3, "dropped").to(dev)
    plan = experts.expert_plan(ids, 7)
    w = torch.randn(50, 2, generator=g).to(dev)
    wide = torch.randn(100, 261, generator=g).to(T).to(dev)
    tall = torch.randn(64, 100, generator=g).to(T).to(dev)
    for v in (wide[:, 3:67], wide[:, 8:72], wide[:, 1:2], tall.t()):
        for n, f in ((50, lambda t: experts.expert_dispatch(t, plan)), (100, lambda t: experts.expert_combine(t, w, plan))):
            a, b = v[:n].detach().requires_grad_(True), v[:n].detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
            ya, yb = f(a), f(b)
            assert torch.equal(ya, yb)
            one = torch.ones((), device=dev, dtype=T).expand(ya.shape)  # (strides of zero)
            assert torch.equal(torch.autograd.grad(ya, a, one)[0], torch.autograd.grad(yb, b, one.contiguous())[0])


@pytest.mark.gpu
def test_places_behind_32_bits(dev):
    """the sorted rows hold more than 2^31 elements"""
    N, k, D = 300_000, 8, 1024
    ids = (torch.arange(N * k, device=dev) % 11).reshape(N, k)
    plan = experts.expert_plan(ids, 11)
    x = torch.arange(N, device=dev, dtype=torch.float32).remainder(251).to(torch.bfloat16)[:, None].expand(N, D)
    rows = experts.expert_dispatch(x, plan)
    at = torch.tensor([0, N * k // 2, N * k - 1], device=dev)
    assert torch.equal(rows[at], x[plan.src[at].long() // k])
    y = experts.expert_combine(rows, torch.full((N, k), 0.125, device=dev), plan)
    assert torch.equal(y, x)


@pytest.mark.gpu
def test_places_of_a_plan_made_by_hand_are_bounded(dev):
    """places outside the sorted rows count as no expert"""
    N, k = 50, 2
    ids = some_ids(N, k, 4, 1, "dropped")
    plan = experts.expert_plan(ids.to(dev), 4)
    dst = plan.dst.clone()
    dst[dst < 0] = N * k
    dst[0, 0], dst[1, 1] = 2 ** 30, -(2 ** 30)  # (rows that nobody takes)
    other = experts.ExpertPlan(plan.offsets, plan.src, dst, 4)
    x, gates = torch.randn(N, 7, device=dev, requires_grad=True), torch.rand(N, k, device=dev, requires_grad=True)
    rows = [experts.expert_dispatch(x, p) for p in (plan, other)]
    y = [experts.expert_combine(r, gates, p) for r, p in zip(rows, (plan, other))]
    assert torch.equal(rows[0], rows[1]) and torch.equal(y[0], y[1])
    dy = torch.randn(N, 7, device=dev)
    for a, b in zip(*[torch.autograd.grad(v, [x, gates], dy) for v in y]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_more_lanes_than_a_launch_holds(dev):
    """rows whose lanes number more than 2^32: every workgroup takes several; values are whole numbers, so all results are exact"""
    N, D = (1 << 26) + 1000, 33
    x = torch.randint(-128, 128, (N, D), device=dev, dtype=torch.int8).to(torch.bfloat16)
    plan = experts.expert_plan((torch.arange(N, device=dev, dtype=torch.int32) % 7)[:, None], 7)
    rows = experts.expert_dispatch(x, plan).requires_grad_(True)
    w = torch.ones(N, 1, device=dev, requires_grad=True)
    y = experts.expert_combine(rows, w, plan)
    assert torch.equal(y, x)
    drows, dw = torch.autograd.grad(y, [rows, w], x)
    assert torch.equal(drows, rows)
    for part in range(0, N, 1 << 22):
        assert torch.equal(dw[part:part + (1 << 22), 0], x[part:part + (1 << 22)].float().square().sum(1))


# ------------------------------------------------------------------------------------------------ the experts' linear layers
def lengths(M, E, kind, seed):
    """offsets [E+1] of M rows"""
    g = torch.Generator().manual_seed(seed)
    if kind == "even":
        who = torch.arange(M) * E // max(M, 1)
    elif kind == "one":
        who = torch.full((M,), E - 1)
    elif kind == "nobody":
        who = torch.zeros(0, dtype=torch.int64)
    else:  # crowded and empty experts, rows behind the last
        share = torch.rand(E, generator=g) ** 4
        share[::3] = 0 if E > 3 else share[::3]
        who = torch.multinomial(share + 1e-9, M - M // 9, replacement=True, generator=g) if M > 8 else torch.zeros(M, dtype=torch.int64)
    return torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(who, minlength=E).cumsum(0)])


def linear_ref(x, w, b, offsets, dy):
    M, E = x.shape[0], w.shape[0]
    out = dict(y=torch.zeros(M, w.shape[1]).double(), dx=torch.zeros_like(x), dw=torch.zeros_like(w), db=torch.zeros(w.shape[:2]).double())
    ab = {k + "_abs": v.clone() for k, v in out.items()}
    for e in range(E):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        for o, n, (X, W, G, B) in ((out, "", (x[s], w[e], dy[s], b[e])), (ab, "_abs", (x[s].abs(), w[e].abs(), dy[s].abs(), b[e].abs()))):
            o["y" + n][s], o["dx" + n][s] = X @ W.T + B, G @ W
            o["dw" + n][e], o["db" + n][e] = G.T @ X, G.sum(0)
    return out, ab


def check_linear(dev, M, E, n_in, n_out, dtype, kind, bias=True, seed=0):
    T = TYPES[dtype]
    g = torch.Generator().manual_seed(seed + M + n_in)
    offsets = lengths(M, E, kind, seed + M)
    x, w, b, dy = (torch.randn(*s, generator=g).to(T) for s in ((M, n_in), (E, n_out, n_in), (E, n_out), (M, n_out)))
    if not bias:
        b.zero_()
    ref, ab = linear_ref(x.double(), w.double(), b.double(), offsets, dy.double())
    held = int(offsets[-1])
    x[held:], dy[held:] = float("nan"), float("inf")  # rows of nobody are never read
    x, w, b = (t.to(dev).requires_grad_(True) for t in (x, w, b))
    y = experts.expert_linear(x, w, b if bias else None, offsets.to(torch.int32).to(dev))
    within(y, ref["y"], n_in + 2, ab["y_abs"])
    grads = torch.autograd.grad(y, [x, w] + ([b] if bias else []), dy.to(dev))
    longest = int((offsets[1:] - offsets[:-1]).max())
    within(grads[0], ref["dx"], n_out + 2, ab["dx_abs"])
    within(grads[1], ref["dw"], longest + 66, ab["dw_abs"])
    if bias:
        within(grads[2], ref["db"], longest + 66, ab["db_abs"])
    return x, w, b, y, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,E,n_in,n_out,kind", [(1, 1, 1, 1, "even"), (1, 3, 64, 64, "one"), (16, 64, 256, 128, "even"), (300, 7, 129, 385, "ragged"),
                                                 (513, 5, 64, 80, "ragged"), (200, 130, 40, 24, "ragged"), (1000, 2, 30, 3, "ragged"),
                                                 (130, 4, 512, 200, "one"), (64, 3, 96, 48, "nobody"), (2500, 3, 200, 136, "ragged"),
                                                 (9, 4, 1030, 66, "even")])
def test_linear_and_gradients(dev, M, E, n_in, n_out, kind, dtype):
    check_linear(dev, M, E, n_in, n_out, dtype, kind, bias=(M + E) % 2 == 0 or kind == "nobody")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,E,n_in,n_out,kind", [(40000, 8, 264, 300, "ragged"), (33000, 64, 301, 265, "ragged"), (6500, 64, 264, 300, "even"),
                                                 (5000, 64, 201, 130, "ragged")])
def test_linear_of_every_tile(dev, M, E, n_in, n_out, kind, dtype):
    """sizes that take the largest tiles, whole weights' gradients and gradients in pieces, rows of whole 16 bytes and others"""
    check_linear(dev, M, E, n_in, n_out, dtype, kind, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,E,n_in,n_out", [(4200, 64, 512, 520), (24000, 1, 776, 1000)])
def test_gradients_of_the_largest_tiles(dev, M, E, n_in, n_out, dtype):
    """weights' gradients by 256 x 256, whole and in pieces"""
    check_linear(dev, M, E, n_in, n_out, dtype, "even", bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,E,kind", [(16, 1000, "ragged"), (700, 65, "ragged"), (700, 129, "even"), (2000, 5000, "ragged"), (9, 8200, "even"), (40, 4097, "one")])
def test_linear_of_many_experts(dev, M, E, kind, dtype):
    """more experts than lanes, and than lanes times lanes"""
    check_linear(dev, M, E, 24, 40, dtype, kind, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,E,n_in,n_out,kind", [(1, 1, 4096, 130, "one"), (5, 2, 2100, 70, "ragged"), (217, 9, 1789, 667, "ragged"), (7, 3, 60, 5000, "even"),
                                                 (30, 4, 2048, 2049, "ragged"), (16, 3, 2000, 64, "nobody")])
def test_linear_of_few_rows_and_long_sums(dev, M, E, n_in, n_out, kind, dtype):
    """sums that are shared out over workgroups and joined, forward and in the rows' gradient"""
    check_linear(dev, M, E, n_in, n_out, dtype, kind, bias=True)


@pytest.mark.gpu
def test_linear_of_rows_far_apart(dev):
    """rows more than 2^20 elements apart are copied first"""
    x = torch.zeros(5, (1 << 20) + 4, device=dev)
    x[:, :40] = torch.randn(5, 40, generator=torch.Generator().manual_seed(1)).to(dev)
    w = torch.randn(2, 24, 40, generator=torch.Generator().manual_seed(2)).to(dev).requires_grad_(True)
    offsets = torch.tensor([0, 2, 5], device=dev)
    results = []
    for t in (x[:, :40], x[:, :40].contiguous()):
        t.requires_grad_(True)
        y = experts.expert_linear(t, w, None, offsets)
        results.append((y,) + torch.autograd.grad(y, [t, w], x[:, 8:32]))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("M,E", [(300, 4), (3000, 64), (4000, 4), (2000, 100)])
def test_linear_of_offsets_that_do_not_ascend(dev, M, E):
    """ask for more tiles and pieces than the rows make: every access stays inside, what follows is right"""
    x, w = torch.ones(M, 40, device=dev, requires_grad=True), torch.ones(E, 72, 40, device=dev, requires_grad=True)
    for first, second in ((0, M), (M, 0), (M + 7, -9)):
        offsets = torch.tensor([first, second] * E, dtype=torch.int32, device=dev)[: E + 1]
        y = experts.expert_linear(x, w, None, offsets)
        torch.autograd.grad(y, [x, w], torch.ones_like(y))
    offsets = torch.tensor([0] * E + [M], device=dev)
    y = experts.expert_linear(x, w, None, offsets)
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert (y == 40).all() and (dx == 72).all() and (dw[-1] == M).all() and not dw[:-1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_of_no_rows(dev, dtype):
    x = torch.zeros(0, 24, device=dev, dtype=TYPES[dtype], requires_grad=True)
    w = torch.randn(3, 8, 24, device=dev).to(TYPES[dtype]).requires_grad_(True)
    y = experts.expert_linear(x, w, None, torch.zeros(4, dtype=torch.int32, device=dev))
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros(0, 8, device=dev, dtype=TYPES[dtype]))
    assert y.shape == (0, 8) and dx.shape == x.shape and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_linear_of_a_piece_of_the_experts(dev, dtype):
    """a piece of the plan's offsets: rows of the other experts, before and behind, are zero and do not enter the gradients"""
    T = TYPES[dtype]
    g = torch.Generator().manual_seed(4)
    offsets = lengths(400, 9, "ragged", 2)
    x, w, dy = torch.randn(400, 40, generator=g).to(T), torch.randn(9, 56, 40, generator=g).to(T), torch.randn(400, 56, generator=g).to(T)
    ref, ab = linear_ref(x.double(), w.double(), torch.zeros(9, 56).double(), offsets, dy.double())
    lo, hi = int(offsets[2]), int(offsets[6])
    xd, wd = x.to(dev).requires_grad_(True), w[2:6].to(dev).requires_grad_(True)
    y = experts.expert_linear(xd, wd, None, offsets[2:7].to(dev))  # (int64 offsets)
    dx, dw = torch.autograd.grad(y, [xd, wd], dy.to(dev))
    for t in (ref["y"], ref["dx"], ab["y_abs"], ab["dx_abs"]):
        t[:lo], t[hi:] = 0, 0
    within(y, ref["y"], 42, ab["y_abs"])
    within(dx, ref["dx"], 58, ab["dx_abs"])
    within(dw, ref["dw"][2:6], 400, ab["dw_abs"][2:6])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_of_other_layouts(dev, dtype):
    """strided rows, columns at an odd start, a transposed weight, a transposed and an expanded gradient: the values of the copies"""
    T = TYPES[dtype]
    g = torch.Generator().manual_seed(9)
    offsets = lengths(150, 3, "ragged", 1).to(torch.int32).to(dev)
    wide = torch.randn(150, 133, generator=g).to(T).to(dev)
    wt = torch.randn(3, 64, 72, generator=g).to(T).to(dev)  # [E, in, out]
    grads = (torch.randn(72, 150, generator=g).to(T).to(dev).t(), torch.ones((), device=dev, dtype=T).expand(150, 72), wide[:, :72])
    for x in (wide[:, 5:69], wide[:, 64:128], wide[:, 1:65].t().contiguous().t()):
        leaves = [x.detach().requires_grad_(True), wt.transpose(1, 2).detach().requires_grad_(True)]
        copies = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in leaves]
        y, z = experts.expert_linear(*leaves, None, offsets), experts.expert_linear(*copies, None, offsets)
        assert torch.equal(y, z)
        for dy in grads:
            for a, b in zip(torch.autograd.grad(y, leaves, dy, retain_graph=True), torch.autograd.grad(z, copies, dy.contiguous(), retain_graph=True)):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_linear_infinities_stay_in_their_rows(dev):
    """an infinite or undefined value reaches the outputs that its row enters, and no others"""
    g = torch.Generator().manual_seed(3)
    offsets = torch.tensor([0, 40, 90], dtype=torch.int32, device=dev)
    x, w = torch.randn(90, 70, generator=g).to(dev), torch.randn(2, 50, 70, generator=g).to(dev)
    clean = experts.expert_linear(x, w, None, offsets)
    x[39, 69], x[40, 0] = float("inf"), float("nan")
    y = experts.expert_linear(x, w, None, offsets)
    keep = torch.ones(90, dtype=torch.bool, device=dev)
    keep[39:41] = False
    assert torch.equal(y[keep], clean[keep]) and not torch.isfinite(y[39:41]).any()


@pytest.mark.gpu
def test_gradients_by_differences(dev):
    """the whole chain's gradients against central differences of it, in fp32: a step of 2^-6 along a random direction; the chain is
    linear in each leaf, so the difference quotient is exact but for the rounding of the two losses"""
    g = torch.Generator().manual_seed(12)
    N, k, E, D, H = 60, 2, 5, 24, 20
    plan = experts.expert_plan(some_ids(N, k, E, 1, "dropped").to(dev), E)
    leaves = [torch.randn(*s, generator=g).to(dev).requires_grad_(True) for s in ((N, D), (E, H, D), (E, H), (N, k))]
    c = torch.randn(N, H, generator=g).to(dev)

    def loss(x, w, b, gates):
        y = experts.expert_combine(experts.expert_linear(experts.expert_dispatch(x, plan), w, b, plan), gates, plan)
        return (y.double() * c).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    with torch.no_grad():
        size = float(sum((t.abs() for t in [loss(*[v.abs() for v in leaves])])))
        for i, (leaf, grad) in enumerate(zip(leaves, grads)):
            d = torch.randn(leaf.shape, generator=g).to(dev)
            h = 2.0 ** -6
            up, down = [list(leaves), list(leaves)]
            up[i], down[i] = leaf + h * d, leaf - h * d
            quotient = float(loss(*up) - loss(*down)) / (2 * h)
            # each loss carries the rounding of its fp32 values: at most D + k + 3 units over terms whose absolute sum is of the order of
            # the loss of absolute values (c enters by its own size), and the leaf's own rounding
            bound = 2 * (D + k + 4) * 2.0 ** -23 * (float(c.abs().max()) + 1) * (size + abs(float(loss(*up)))) / (2 * h)
            assert abs(quotient - float((grad.double() * d).sum())) <= bound


# ------------------------------------------------------------------------------------------------ streams, graphs, a second device
def moe_step(x, ids, E, w, b, gates, dy):
    plan = experts.expert_plan(ids, E)
    rows = experts.expert_dispatch(x, plan)
    y = experts.expert_combine(experts.expert_linear(rows, w, b, plan), gates, plan)
    return (y,) + torch.autograd.grad(y, [x, w, b, gates], dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N", [("f32", 96), ("bf16", 5000)])
def test_captured_and_replayed(dev, dtype, N):
    """plan, exchange, products and all gradients in one graph, replayed on new contents with eager work in between: the eager bits"""
    T, E, D, H, k = TYPES[dtype], 6, 72, 40, 2
    g = torch.Generator().manual_seed(2)

    def fresh(seed):
        q = torch.Generator().manual_seed(seed)
        return [some_ids(N, k, E, seed, "dropped").to(dev), torch.randn(N, D, generator=q).to(T).to(dev), torch.randn(N, H, generator=q).to(T).to(dev)]

    w, b = (torch.randn(*s, generator=g).to(T).to(dev).requires_grad_(True) for s in ((E, H, D), (E, H)))
    gates = torch.rand(N, k, generator=g).to(dev).requires_grad_(True)
    ids, x, dy = fresh(0)
    x.requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        moe_step(x, ids, E, w, b, gates, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = moe_step(x, ids, E, w, b, gates, dy)
    for seed in (1, 2, 3, 1):
        new = fresh(seed)
        with torch.no_grad():
            ids.copy_(new[0]), x.copy_(new[1]), dy.copy_(new[2])
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, r in zip(kept, moe_step(x, ids, E, w, b, gates, dy)):
            assert torch.equal(a, r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_few_rows_captured(dev, dtype):
    """sums shared out over workgroups, in two graphs that are replayed in turn with eager calls between them: the eager bits"""
    T = TYPES[dtype]
    g = torch.Generator().manual_seed(21)
    w = [torch.randn(3, 130, n, generator=g).to(T).to(dev) for n in (4096, 2051)]
    x = [torch.zeros(5, n, device=dev, dtype=T) for n in (4096, 2051)]
    offsets = [torch.zeros(4, device=dev, dtype=torch.int32) for _ in x]
    for a in zip(x, w, offsets):
        experts.expert_linear(a[0], a[1], None, a[2])
    graphs, out = [torch.cuda.CUDAGraph() for _ in x], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            out.append(experts.expert_linear(x[i], w[i], None, offsets[i]))
    for replay in range(4):
        for i, graph in enumerate(graphs):
            x[i].copy_(torch.randn(x[i].shape, generator=g).to(T))
            offsets[i].copy_(torch.tensor([0, replay, 3, 3 + replay % 3], dtype=torch.int32))
            graph.replay()
        eager = [experts.expert_linear(x[i], w[i], None, offsets[i]) for i in range(2)]
        torch.cuda.synchronize()
        for kept, now, n in zip(out, eager, range(2)):
            assert torch.equal(kept, now) and not now[3 + replay % 3:].any() and now[:1].any()


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """two chains of different inputs side by side on two streams give what they give alone"""
    g = torch.Generator().manual_seed(8)
    jobs = []
    for seed, N in ((0, 3000), (1, 20000)):
        ids = some_ids(N, 2, 12, seed, "dropped").to(dev)
        t = [torch.randn(*s, generator=g).to(dev).requires_grad_(True) for s in ((N, 64), (12, 48, 64), (12, 48), (N, 2))]
        jobs.append((t[0], ids, 12, t[1], t[2], t[3], torch.randn(N, 48, generator=g).to(dev)))
    alone = [moe_step(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        both = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                both.append(moe_step(*j))
        torch.cuda.synchronize()
        for a, r in zip(alone, both):
            assert all(torch.equal(p, q) for p, q in zip(a, r))


@pytest.mark.gpu
def test_second_derivatives_are_refused(dev):
    plan = experts.expert_plan(torch.zeros(4, 1, dtype=torch.int64, device=dev), 1)
    x = torch.randn(4, 8, device=dev, requires_grad=True)
    (g,) = torch.autograd.grad(experts.expert_dispatch(x, plan).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
def test_a_tangent_is_not_dropped():
    """an input that carries a tangent takes the way through autograd, which refuses it; without one nothing changes"""
    from torch.autograd import forward_ad

    t = torch.zeros(3, 4)
    assert not experts._wants_grad(t, None) and experts._wants_grad(t, t.clone().requires_grad_(True))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        assert experts._wants_grad(None, dual) and not experts._wants_grad(t, None)
        with torch.no_grad():
            assert experts._wants_grad(t, dual)
    assert not experts._wants_grad(t)


@pytest.mark.gpu
def test_forward_mode_is_refused(dev):
    from torch.autograd import forward_ad

    plan = experts.expert_plan(torch.zeros(4, 1, dtype=torch.int64, device=dev), 1)
    x, w, gates = torch.randn(4, 8, device=dev), torch.randn(1, 6, 8, device=dev), torch.rand(4, 1, device=dev)
    b = torch.randn(1, 6, device=dev)
    with forward_ad.dual_level():
        d = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: experts.expert_dispatch(d(x), plan), lambda: experts.expert_combine(d(x), gates, plan),
                     lambda: experts.expert_combine(x, d(gates), plan), lambda: experts.expert_combine(d(x), None, plan),
                     lambda: experts.expert_linear(d(x), w, None, plan), lambda: experts.expert_linear(x, d(w), b, plan),
                     lambda: experts.expert_linear(x, w, d(b), plan)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
                call()
        y = experts.expert_linear(x, w, b, plan)  # (no tangent: as ever)
        assert forward_ad.unpack_dual(y).tangent is None


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
def test_offsets_beyond_32_bits_are_bounded_before_they_are_narrowed():
    wide = torch.tensor([-2 ** 33, 0, 3, 2 ** 31, 2 ** 32 + 1, 2 ** 62])
    assert experts._offsets32(wide, 7).tolist() == [0, 0, 3, 7, 7, 7] and experts._offsets32(wide, 7).dtype == torch.int32
    narrow = torch.tensor([0, 3, 9, 9], dtype=torch.int32)
    assert experts._offsets32(narrow, 7) is narrow and experts._offsets32(narrow[::2], 7).is_contiguous()


@pytest.mark.gpu
def test_linear_of_the_first_rows_of_a_very_long_list(dev):
    x, w = torch.randn(50, 24, device=dev), torch.randn(3, 8, 24, device=dev)
    want = experts.expert_linear(x, w, None, torch.tensor([0, 20, 50, 50], device=dev))
    assert torch.equal(experts.expert_linear(x, w, None, torch.tensor([0, 20, 2 ** 32 + 5, 2 ** 33], device=dev)), want)


# ------------------------------------------------------------------------------------------------ crowded experts
def test_weight_gradients_of_many_experts_make_room_for_a_crowded_one():
    """sums of the weights' gradients are cut where one expert that had all rows would be summed in one run for long"""
    from presight_amd._lib import lib

    need = lambda M, E, n_in, n_out, code: lib().ps_expert_linear_workspace(2, 256, n_out, 256, n_in, M, E, n_in, n_out, code)  # noqa: E731
    for M, E, code in ((65536, 512, 0), (131072, 1024, 0), (131072, 1024, 1), (65536, 32, 2)):
        assert need(M, E, 64, 64, code) > 0
    # room for two pieces of 2048 rows, or of four times the even share, for every one that fits the rows; 64 more sums for the bias
    assert need(131072, 1024, 64, 64, 0) == 2 * 64 * (64 * 64 + 64) * 4
    assert need(65536, 32, 2048, 1024, 2) == 2 * 8 * (2048 * 1024 + 1024) * 4
    assert need(1 << 20, 512, 2048, 2048, 2) < 1 << 29  # (large weights: no more pieces than fill the chip)
    assert need(2048, 16, 64, 64, 0) == need(5000, 64, 512, 512, 2) == 0  # (short whoever has them)


@pytest.mark.gpu
@pytest.mark.parametrize("M,E", [(131072, 1024), (70000, 300)])
def test_a_crowded_experts_sums_are_cut(dev, M, E):
    """all rows to one expert: its first term is one and every other one 2^-28, which one run of fp32 additions loses; cut to 2048 rows it
    is off by 2048 + the pieces of additions at most"""
    x, dy = torch.full((M, 64), 2.0 ** -28, device=dev), torch.ones(M, 64, device=dev)
    x[0] = 1.0
    x.requires_grad_(True)
    w, b = torch.zeros(E, 64, 64, device=dev, requires_grad=True), torch.zeros(E, 64, device=dev, requires_grad=True)
    for at in (0, E // 2, E - 1):
        offsets = torch.where(torch.arange(E + 1, device=dev) > at, M, 0)
        dw, db = torch.autograd.grad(experts.expert_linear(x, w, b, offsets), [w, b], dy)
        ref = torch.full((64, 64), 1.0 + (M - 1) * 2.0 ** -28, dtype=torch.float64)
        within(dw[at], ref, 2048 + M // 2048 + 66, ref)
        assert (db[at] == M).all()  # (whole numbers below 2^24: exact)
        keep = torch.arange(E, device=dev) != at
        assert not dw[keep].any() and not db[keep].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,E,n_in,n_out,kind", [(70000, 300, 24, 40, "one"), (70000, 300, 24, 40, "ragged"), (66000, 5000, 16, 33, "one"),
                                                 (40000, 64, 136, 130, "one"), (30000, 64, 264, 300, "ragged"), (30011, 70, 265, 301, "one")])
def test_linear_of_crowded_experts(dev, M, E, n_in, n_out, kind, dtype):
    """some or all rows at one or a few of many experts, every tile, odd rows, with and without room for more than one piece"""
    check_linear(dev, M, E, n_in, n_out, dtype, kind, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("M,E", [(70000, 300), (66000, 5000)])
def test_crowded_offsets_that_do_not_ascend(dev, M, E):
    """ask for more pieces than there is room for: every access stays inside, what follows is right"""
    x, w = torch.ones(M, 24, device=dev, requires_grad=True), torch.ones(E, 40, 24, device=dev, requires_grad=True)
    for first, second in ((0, M), (M, 0), (M + 7, -9)):
        offsets = torch.tensor([first, second] * E, dtype=torch.int32, device=dev)[: E + 1]
        torch.autograd.grad(experts.expert_linear(x, w, None, offsets), [w], torch.ones(M, 40, device=dev))
    offsets = torch.tensor([0] * E + [M], device=dev)
    (dw,) = torch.autograd.grad(experts.expert_linear(x, w, None, offsets), [w], torch.ones(M, 40, device=dev))
    assert (dw[-1] == M).all() and not dw[:-1].any()


@pytest.mark.gpu
def test_crowded_experts_captured(dev):
    """one captured pass replayed for even, crowded and missing rows in turn: the eager bits"""
    M, E = 70000, 300
    g = torch.Generator().manual_seed(23)
    x, dy = torch.randn(M, 24, generator=g).to(dev), torch.randn(M, 40, generator=g).to(dev)
    w = torch.randn(E, 40, 24, generator=g).to(dev).requires_grad_(True)
    b = torch.randn(E, 40, generator=g).to(dev).requires_grad_(True)
    kinds = [lengths(M, E, kind, 5).to(torch.int32).to(dev) for kind in ("even", "one", "ragged", "nobody", "one")]
    offsets = kinds[0].clone()
    step = lambda: torch.autograd.grad(experts.expert_linear(x, w, b, offsets), [w, b], dy)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for o in kinds:
        offsets.copy_(o)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, r) for a, r in zip(kept, step()))
