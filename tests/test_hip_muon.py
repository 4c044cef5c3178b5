"""The orthogonalised update and its optimizer (presight_amd.optim.newton_schulz, HipMuon) against plain 64-bit restatements.

Tolerance.  Rounding errors of the iterates grow by up to the polynomial's steepest slope (about 4) per step in the small singular
directions and are damped in the others, so a bound from the formula alone is a thousand times too wide.  It is taken from the same
formula in plain fp32 instead: its distance from 64 bits in the Frobenius norm, per matrix.  The kernels hold 22 bits where fp32 holds 24
but sum the same fp32 way: each of a step's three stored results (S, a + b S + c S S, X) carries a rounding of 2^-23 in place of 2^-24, and
each of the three products a dropped term of 2^-24, so at most four times the unit that the plain form rounds with: 4 x its distance.  A
matrix for which that distance happens to be tiny gets 16 * 2^-24 of its norm instead.  The result's own rounding comes on top."""
import math
import os
import subprocess
import sys
import textwrap

import pytest
import torch

from presight_amd import optim

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ABC = optim.NS_COEFFICIENTS


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch.device("cuda:0")


def iterate(g, steps=5, abc=ABC, eps=1e-7):
    """the definition, in g's own precision, short side first"""
    a, b, c = abc
    x = g.transpose(-2, -1) if g.shape[-2] > g.shape[-1] else g
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + eps).to(x.dtype)
    for _ in range(steps):
        s = x @ x.transpose(-2, -1)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(-2, -1) if g.shape[-2] > g.shape[-1] else x


def norms(t):
    return t.double().flatten(-2).norm(dim=-1)


def check(got, g, steps=5, abc=ABC, eps=1e-7):
    g = g.detach().cpu()
    ref = iterate(g.double(), steps, abc, eps)
    plain = norms(iterate(g.float(), steps, abc, eps).double() - ref)
    f = torch.finfo(got.dtype)
    rounding = norms(ref) * f.eps / 2 + f.smallest_normal * f.eps * math.sqrt(g.shape[-1] * g.shape[-2])
    bound = torch.maximum(4 * plain, 16 * 2.0 ** -24 * norms(ref)) + (rounding if got.dtype != torch.float32 else 0)
    err = norms(got.detach().cpu().double() - ref)
    assert got.shape == g.shape and torch.isfinite(got).all()
    assert (err <= bound).all(), f"worst {float((err / bound.clamp_min(1e-300)).max()):.2f} x the bound, relative {float((err / norms(ref)).max()):.1e}"
    return ref


# ------------------------------------------------------------------------------------------------ refusals (no GPU needed)
def test_refuses_what_it_cannot_do():
    g = torch.zeros(4, 5)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        optim.newton_schulz(g)
    for kw in (dict(steps=0), dict(steps=65), dict(steps=2.5), dict(coefficients=(1.0, 2.0)), dict(coefficients=(3.0, 3.0, 3.0)),
               dict(coefficients=(float("nan"), 0.0, 0.0)), dict(eps=-1.0), dict(eps=float("inf"))):
        with pytest.raises(ValueError):
            optim.newton_schulz(g, **kw)
    with pytest.raises(RuntimeError, match="contiguous fp32 CUDA"):
        optim.HipMuon([torch.nn.Parameter(g)])


def test_bound_of_the_polynomial_holds_by_sampling():
    """what _ns_check lets through stays inside its bound on a fine grid; what leaves it is refused"""
    for abc in (ABC, (2.0, -1.5, 0.5), (1.5, -0.5, 0.0), (3.0, -16 / 5, 6 / 5), (1.0, 0.0, 0.0), (5.0, 0.0, 0.0), (1.0, 2.0, 0.0), (-2.0, 1.0, 3.0)):
        v = torch.linspace(0, 1, 20001, dtype=torch.float64)
        worst = 1.0
        for _ in range(3):
            worst = max(worst, float((abc[0] + abc[1] * v ** 2 + abc[2] * v ** 4).abs().max()), float((v * v).max()))
            v = (v * (abc[0] + abc[1] * v ** 2 + abc[2] * v ** 4)).abs()
            v = torch.linspace(0, float(v.max()), 20001, dtype=torch.float64)
            worst = max(worst, float(v.max()), float((v * v).max()))
        if worst > 15.001:
            with pytest.raises(ValueError):
                optim._ns_check(3, *abc)
        elif worst < 14.9:
            assert optim._ns_check(3, *abc) <= 16.0


def test_library_refuses_bad_sizes():
    from presight_amd._lib import lib

    h = lib()
    assert h.ps_newton_schulz_workspace(0, 80, 90) == 0 and h.ps_newton_schulz_workspace(1, 80, 90) > 0
    for rc in (h.ps_newton_schulz(None, 1, 8, 8, 0, 5, 1.0, 0.0, 0.0, 1.0, 0.0, None, None, None),
               h.ps_newton_schulz(None, 1, 8, 8, 0, 0, 1.0, 0.0, 0.0, 1.0, 0.0, None, None, None),
               h.ps_newton_schulz(None, 1, 20000, 20000, 0, 5, 1.0, 0.0, 0.0, 1.0, 0.0, None, None, None),
               h.ps_newton_schulz(None, 1 << 17, 8, 8, 0, 5, 1.0, 0.0, 0.0, 1.0, 0.0, None, None, None),
               h.ps_muon_step(1, None, None, None, None, None, None, None, 0.9, 1, 1.0, 5, 1.0, 0.0, 0.0, 1.0, 0.0, None, None)):
        assert rc != 0
    assert h.ps_newton_schulz(None, 0, 8, 8, 0, 5, 1.0, 0.0, 0.0, 1.0, 0.0, None, None, None) == 0


# ------------------------------------------------------------------------------------------------ values
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 1), (1, 70), (64, 64), (2, 2, 5, 7), (16, 64, 40), (5, 80, 64), (3, 385, 129), (7, 3, 64), (2, 65, 63),
                                   (1, 128, 128), (2, 129, 200), (4, 33, 900), (1, 640, 512), (1, 257, 1030), (130, 9, 4)])
def test_newton_schulz(dev, shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=g) * 3e-3).to(TYPES[dtype])
    check(optim.newton_schulz(x.to(dev)), x)


@pytest.mark.gpu
@pytest.mark.parametrize("steps,abc,eps", [(1, ABC, 1e-7), (2, (2.0, -1.5, 0.5), 0.0), (10, (1.5, -0.5, 0.0), 1e-3), (5, (1.0, 0.0, 0.0), 1e-7)])
def test_other_polynomials(dev, steps, abc, eps):
    x = torch.randn(3, 70, 50, generator=torch.Generator().manual_seed(1))
    check(optim.newton_schulz(x.to(dev), steps=steps, coefficients=abc, eps=eps), x, steps, abc, eps)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(64, 48), (300, 200)])
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1.0, 1e18, 3e37])
def test_any_scale(dev, shape, scale):
    """sums of squares that leave fp32's range; below eps the result shrinks with the input, as the definition has it"""
    x = torch.randn(shape, generator=torch.Generator().manual_seed(3)) * scale
    check(optim.newton_schulz(x.to(dev)), x)


@pytest.mark.gpu
@pytest.mark.parametrize("side", [40, 200])
def test_of_low_rank_and_of_zero(dev, side):
    g = torch.Generator().manual_seed(5)
    x = torch.stack([torch.randn(side, 1, generator=g) @ torch.randn(1, 2 * side, generator=g), torch.zeros(side, 2 * side),
                     torch.randn(side, 3, generator=g) @ torch.randn(3, 2 * side, generator=g)])
    y = optim.newton_schulz(x.to(dev))
    check(y, x)
    assert not y[1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("side", [40, 200])
def test_undefined_entries_stay_in_their_matrix(dev, side):
    x = torch.randn(4, side, side + 5, generator=torch.Generator().manual_seed(6))
    clean = optim.newton_schulz(x.to(dev))
    x[1, 3, 4], x[2, 0, 0] = float("nan"), float("inf")
    y = optim.newton_schulz(x.to(dev))
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()


@pytest.mark.gpu
def test_singular_values_move_to_one_and_vectors_stay(dev):
    g = torch.Generator().manual_seed(7)
    u, _, v = torch.linalg.svd(torch.randn(96, 160, generator=g, dtype=torch.float64), full_matrices=False)
    x = (u * torch.linspace(0.05, 1, 96, dtype=torch.float64)) @ v
    y = optim.newton_schulz(x.float().to(dev)).cpu().double()
    d = u.T @ y @ v.T
    s = d.diagonal()
    assert float(s.min()) > 0.6 and float(s.max()) < 1.3 and float((d - torch.diag(s)).abs().max()) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 64, 40), (2, 200, 136)])
def test_other_layouts_and_empty(dev, shape):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(8)).to(dev)
    want = optim.newton_schulz(x)
    assert torch.equal(optim.newton_schulz(x.transpose(1, 2).contiguous().transpose(1, 2)), want)
    wide = torch.zeros(shape[0], shape[1], shape[2] + 3, device=dev)
    wide[..., 1:-2] = x
    assert torch.equal(optim.newton_schulz(wide[..., 1:-2]), want)
    assert torch.equal(optim.newton_schulz(x[1]), want[1])  # (a matrix does not see the rest of its stack)
    assert optim.newton_schulz(x[:0]).shape == (0,) + shape[1:] and optim.newton_schulz(x[:, :0]).shape == (shape[0], 0, shape[2])


@pytest.mark.gpu
def test_a_large_matrix(dev):
    """1500 x 2300: against 64 bits on the GPU"""
    x = torch.randn(1500, 2300, generator=torch.Generator().manual_seed(9)).to(dev)
    ref, plain = iterate(x.double()), iterate(x)
    bound = max(4 * float((plain.double() - ref).norm()), 16 * 2.0 ** -24 * float(ref.norm()))
    assert float((optim.newton_schulz(x).double() - ref).norm()) <= bound


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(12, 600, 700), (12, 701, 603), (3, 700, 1100), (40, 130, 65)])
def test_every_tile(dev, shape, dtype):
    """stacks that take the largest tiles and others, wide and tall, odd rows; against 64 bits on the GPU, matrix by matrix"""
    x = (torch.randn(shape, generator=torch.Generator().manual_seed(14)) * 1e-2).to(TYPES[dtype]).to(dev)
    y = optim.newton_schulz(x)
    f = torch.finfo(y.dtype)
    for got, g in zip(y, x):
        ref, plain = iterate(g.double()), iterate(g.float())
        rounding = 0.0 if dtype == "f32" else float(ref.norm()) * f.eps / 2
        assert float((got.double() - ref).norm()) <= max(4 * float((plain.double() - ref).norm()), 16 * 2.0 ** -24 * float(ref.norm())) + rounding


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("shape", [(1, 8, 4096), (3, 70, 3000), (2, 4000, 100), (5, 30, 600), (64, 30, 600), (60, 128, 128), (1, 200, 5001)])
def test_long_and_many(dev, shape, dtype):
    """few rows and a long other side, whose sums over it are shared out; many matrices of few tiles"""
    x = (torch.randn(shape, generator=torch.Generator().manual_seed(16)) * 1e-2).to(TYPES[dtype])
    check(optim.newton_schulz(x.to(dev)), x)
    assert torch.equal(optim.newton_schulz(x.to(dev)), optim.newton_schulz(x.to(dev)))


# ------------------------------------------------------------------------------------------------ the optimizer
def muon_ref(p, g, buf, lr, mu, nesterov, wd, scale):
    buf = mu * buf + (1 - mu) * g
    u = mu * buf + (1 - mu) * g if nesterov else buf
    out, n_in = p.shape[-2:]
    rate = lr * (math.sqrt(max(1.0, out / n_in)) if scale == "spectral" else 0.2 * math.sqrt(max(out, n_in)))
    return (1 - lr * wd) * p - rate * iterate(u), buf, rate


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,scale", [(True, "spectral"), (False, "rms")])
@pytest.mark.parametrize("shapes", [[(16, 64, 40), (80, 64), (3, 64), (1, 64)], [(2, 300, 200), (64, 64), (260, 1000)]])
def test_muon_steps(dev, shapes, nesterov, scale):
    """three steps with fresh gradients, weight decay and a changed learning rate; a parameter whose gradient is missing in the second"""
    g = torch.Generator().manual_seed(10)
    start = [torch.randn(s, generator=g) for s in shapes]
    params = [torch.nn.Parameter(t.to(dev)) for t in start]
    opt = optim.HipMuon(params, lr=0.03, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=scale)
    ref = [(t.double(), torch.zeros(t.shape, dtype=torch.float64)) for t in start]
    size = [0.0] * len(shapes)
    for step in range(3):
        opt.lr = 0.03 / (1 + step)
        for i, p in enumerate(params):
            grad = torch.randn(p.shape, generator=g) * 10.0 ** (step - 2)
            p.grad = grad.to(dev)
            if step == 1 and i == 1:
                p.grad = None
                continue
            new, buf, rate = muon_ref(*[t for t in (ref[i][0], grad.double(), ref[i][1])], opt.lr, 0.9, nesterov, 0.1, scale)
            ref[i] = (new, buf)
            size[i] += rate
        opt.step()
    for i, (p, buf) in enumerate(zip(params, opt.momentum_buffers)):
        # updates: relative error below 1e-4 each (test_newton_schulz's bound at these sizes is smaller); parameters: three fp32 roundings of
        # values that the last one bounds within a factor of two
        many = math.prod(p.shape[:-2]) or 1
        bound = 1e-4 * size[i] * 1.3 * math.sqrt(many * min(p.shape[-2:])) + 6 * 2.0 ** -24 * 2 * float(ref[i][0].norm())
        assert float((p.detach().cpu().double() - ref[i][0]).norm()) <= bound
        torch.testing.assert_close(buf.cpu().double(), ref[i][1], rtol=0, atol=8 * 2.0 ** -24 * float(ref[i][1].abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(12, 600, 700), (12, 701, 603), (3, 704, 500), (2, 31, 33), (2, 50, 2000), (64, 16, 700)])
def test_muon_applies_the_orthogonalised_momentum(dev, shape):
    """the first step's u is the same bits computed outside (two products and a sum, each rounded), so its orthogonalised form is too; the
    parameter then carries two roundings of about its own size and one of the product's"""
    g = torch.Generator().manual_seed(15)
    p, grad = torch.randn(shape, generator=g).to(dev), torch.randn(shape, generator=g).to(dev)
    q = torch.nn.Parameter(p.clone())
    q.grad = grad
    opt = optim.HipMuon([q], lr=0.05, momentum=0.9, weight_decay=0.2)
    opt.step()
    buf = (1.0 - 0.9) * grad
    assert torch.equal(opt.momentum_buffers[0], buf)
    y = optim.newton_schulz(0.9 * buf + (1.0 - 0.9) * grad).double()
    rate = 0.05 * math.sqrt(max(1.0, shape[1] / shape[2]))
    ref = (1 - 0.05 * 0.2) * p.double() - rate * y
    bound = 3 * 2.0 ** -24 * (p.double().abs() + rate * y.abs()) + 2.0 ** -24 * (p.double().abs() + rate * y.abs())  # (and those of keep and rate)
    assert ((q.detach().double() - ref).abs() <= bound).all()


@pytest.mark.gpu
def test_muon_refuses_parameters_twice_and_changed(dev):
    p = torch.nn.Parameter(torch.randn(2, 40, 30, device=dev))
    with pytest.raises(ValueError, match="more than once"):
        optim.HipMuon([p, p])
    opt = optim.HipMuon([p])
    kept = p.detach().clone()
    for data in (p.data.double(), p.data.transpose(1, 2), p.data[:1]):
        q = p.data
        p.data = data
        p.grad = torch.ones_like(p)
        with pytest.raises(RuntimeError):
            opt.step()
        p.grad = None
        p.data = q
    assert torch.equal(p, kept) and not opt.momentum_buffers[0].any()


@pytest.mark.gpu
def test_muon_state_and_refusals(dev):
    g = torch.Generator().manual_seed(11)
    p = torch.nn.Parameter(torch.randn(6, 48, 32, generator=g).to(dev))
    q = torch.nn.Parameter(p.detach().clone())
    a, b = optim.HipMuon([p]), optim.HipMuon([q])
    for i in range(3):
        grad = torch.randn(p.shape, generator=g).to(dev)
        p.grad = grad
        a.step()
        if i == 1:
            b.load_state_dict(a.state_dict())
            q.data.copy_(p.data)
        if i == 2:
            q.grad = grad.clone()
            b.step()
    assert torch.equal(p, q) and torch.equal(a.momentum_buffers[0], b.momentum_buffers[0]) and b.step_count == 3
    for bad in (torch.zeros(4, device=dev), torch.zeros(4, 4, device=dev).half()):
        with pytest.raises((ValueError, RuntimeError)):
            optim.HipMuon([torch.nn.Parameter(bad)])
    with pytest.raises(ValueError):
        optim.HipMuon([p], momentum=1.0)
    with pytest.raises(ValueError):
        optim.HipMuon([p], scale="other")
    p.grad = None
    p._ps_group = 0
    p.grad = grad
    with pytest.raises(RuntimeError, match="decided on the device"):
        a.step()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 70, 3000), (12, 600, 700)])
def test_newton_schulz_captured(dev, shape):
    g = torch.Generator().manual_seed(17)
    x = torch.randn(shape, generator=g).to(dev)
    optim.newton_schulz(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = optim.newton_schulz(x)
    for _ in range(3):
        x.copy_(torch.randn(shape, generator=g))
        graph.replay()
        eager = optim.newton_schulz(x)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(16, 64, 40), (3, 64)], [(2, 200, 300)]])
def test_muon_captured(dev, shapes):
    """a captured step, replayed on new gradients with eager work in between, walks the eager path bit for bit"""
    g = torch.Generator().manual_seed(12)
    start = [torch.randn(s, generator=g).to(dev) for s in shapes]
    eager, graphed = ([torch.nn.Parameter(t.clone()) for t in start] for _ in range(2))
    a, b = optim.HipMuon(eager), optim.HipMuon(graphed)
    static = [torch.zeros_like(t) for t in start]
    for p, s in zip(graphed, static):
        p.grad = s
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (a step without gradients leaves nothing behind but the decay)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b.step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        for p, s in zip(eager, static):
            p.grad = torch.randn(p.shape, generator=g).to(dev)
            s.copy_(p.grad)
        graph.replay()
        a.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, graphed))
        assert all(torch.equal(p, q) for p, q in zip(a.momentum_buffers, b.momentum_buffers))


@pytest.mark.gpu
def test_experts_trained_by_muon(dev):
    """the operators as they are used together: rows to their experts, two layers, back with gates, gradients, the step on the stacked
    weights; against 64 bits"""
    from presight_amd import experts

    g = torch.Generator().manual_seed(13)
    N, k, E, D, H = 500, 2, 6, 40, 64
    ids = torch.randint(-1, E, (N, k), generator=g)
    x, gates, dy = torch.randn(N, D, generator=g), torch.rand(N, k, generator=g), torch.randn(N, D, generator=g)
    w1, w2 = torch.randn(E, H, D, generator=g) / D ** 0.5, torch.randn(E, D, H, generator=g) / H ** 0.5

    def forward64(w1, w2):
        y = torch.zeros(N, D, dtype=torch.float64)
        for j in range(k):
            for e in range(E):
                m = ids[:, j] == e
                h = torch.relu(x[m].double() @ w1[e].T)
                y = y.index_add(0, m.nonzero()[:, 0], gates[m, j].double()[:, None] * (h @ w2[e].T))
        return y

    refs = [w1.double().requires_grad_(True), w2.double().requires_grad_(True)]
    y64 = forward64(*refs)
    grads = torch.autograd.grad(y64, refs, dy.double())
    params = [torch.nn.Parameter(t.to(dev)) for t in (w1, w2)]
    opt = optim.HipMuon(params, lr=0.02, weight_decay=0.01)
    plan = experts.expert_plan(ids.to(dev), E)
    h = torch.relu(experts.expert_linear(experts.expert_dispatch(x.to(dev), plan), params[0], None, plan))
    y = experts.expert_combine(experts.expert_linear(h, params[1], None, plan), gates.to(dev), plan)
    torch.testing.assert_close(y.detach().cpu().double(), y64.detach(), rtol=0, atol=(D + H + 4) * 2.0 ** -23 * float(y64.abs().max()) * 4)
    y.backward(dy.to(dev))
    opt.step()
    for p, ref, grad in zip(params, refs, grads):
        new, _, rate = muon_ref(ref.detach(), grad, torch.zeros_like(grad), 0.02, 0.95, True, 0.01, "spectral")
        # the gradient's relative error (sums of about 170 rows of about 100 terms) grows by at most the polynomial's slope per step
        slack = rate * 4 ** 5 * (N + D + H) * 2.0 ** -23 * math.sqrt(E * 40) + 4 * 2.0 ** -24 * float(new.norm())
        assert float((p.detach().cpu().double() - new).norm()) <= slack


# ------------------------------------------------------------------------------------------------ gradients that live in a FlatGrads
def test_step_waits_for_gradients_written_on_side_streams(monkeypatch):
    """gradients of a FlatGrads are written in place, some of them on the proposal networks' side stream: it is joined before any is read"""
    from presight_amd.dist import FlatGrads

    joins = []
    monkeypatch.setattr(optim, "join_side_streams", lambda: joins.append(1))
    plain, held = torch.nn.Parameter(torch.zeros(4, 5)), [torch.nn.Parameter(torch.zeros(3, 4)) for _ in range(2)]
    plain.grad = torch.ones(4, 5)
    assert optim._with_gradients([plain]) == [0] and not joins
    fg = FlatGrads(held)
    held[1]._ps_touched = True
    assert optim._with_gradients([plain] + held) == [0, 2] and len(joins) == 1
    fg.zero_()
    assert optim._with_gradients(held) == []


@pytest.mark.gpu
def test_muon_of_gradients_written_on_a_side_stream(dev):
    from presight_amd import ops
    from presight_amd.dist import FlatGrads

    g = torch.Generator().manual_seed(18)
    start, grad = torch.randn(4, 96, 80, generator=g).to(dev), torch.randn(4, 96, 80, generator=g).to(dev)
    alone, held = torch.nn.Parameter(start.clone()), torch.nn.Parameter(start.clone())
    alone.grad = grad
    a, b = optim.HipMuon([alone]), optim.HipMuon([held])
    fg = FlatGrads([held])
    busy = torch.randn(4096, 4096, device=dev)
    side = ops.side_stream(dev)
    for _ in range(3):
        a.step()
        fg.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(20):  # (the write comes late)
                busy = busy @ busy * 1e-4
            held.grad.copy_(grad)
        ops.mark_touched([held])
        b.step()
        torch.cuda.synchronize()
        assert torch.equal(alone, held) and torch.equal(a.momentum_buffers[0], b.momentum_buffers[0])


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_HEAD = """
    import sys, torch, torch.distributed as dist
    sys.path.insert(0, {root!r})
    from presight_amd import optim
    from presight_amd.dist import FlatGrads, init_from_env
    rank, local, world = init_from_env("cpu")
    params = [torch.nn.Parameter(torch.zeros(4, 8)) for _ in range(3)]
"""
_TAIL = """
    dist.barrier(); dist.destroy_process_group()
    print("rank", rank, "ok")
"""
_SHARDED = """
    fg = FlatGrads(params, bucket_sizes=[1, 2], shard_world=world)
    assert optim._with_gradients(params) == []  # (nothing is exchanged yet)
    fg.enable_overlap([params[:1], params[1:]], mode="sharded")
    fg.zero_()
    sum(p.sum() * (rank + 1.0) for p in params).backward()
    fg.finish_exchange()
    try:
        optim._with_gradients(params)
        raise SystemExit("gradients that are averaged in shards must be refused")
    except RuntimeError as e:
        assert "sharded" in str(e)
    own = torch.nn.Parameter(torch.zeros(4, 8))
    own.grad = torch.ones(4, 8)
    assert optim._with_gradients([own]) == [0]
    fg = FlatGrads(params)  # a new buffer takes the gradients over
    fg.enable_overlap([params], mode="allreduce")
    fg.zero_()
    sum(p.sum() * (rank + 1.0) for p in params).backward()
    fg.finish_exchange()
    assert optim._with_gradients(params) == [0, 1, 2] and all(bool((p.grad == 1.5).all()) for p in params)
"""


def two_ranks(tmp_path, body, port):
    script = tmp_path / "worker.py"
    script.write_text("".join(textwrap.dedent(t) for t in (_HEAD, body, _TAIL)).format(root=ROOT))
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                        "--master-port", str(port), str(script)], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0 and r.stdout.count("ok") == 2, r.stdout[-2000:] + r.stderr[-2000:]


def test_gradients_averaged_in_shards_are_refused(tmp_path):
    two_ranks(tmp_path, _SHARDED, 29761)


_AGREED = """
    fg = FlatGrads(params)
    fg.flags_may_differ_across_ranks = True  # (routing left the middle one without samples on rank 1)
    fg.zero_()
    (params[0].sum() + (params[1].sum() * 4.0 if rank == 0 else 0.0)).backward()
    fg.finish_exchange()
    assert optim._with_gradients(params) == [0, 1] and bool((params[1].grad == 2.0).all())
    assert optim._with_gradients(params[1:]) == [0]
    fg.flags_may_differ_across_ranks = False  # (ranks are known to agree: nothing is asked)
    assert optim._with_gradients(params) == ([0, 1] if rank == 0 else [0])
"""


def test_ranks_agree_on_who_has_a_gradient(tmp_path):
    two_ranks(tmp_path, _AGREED, 29763)


# ------------------------------------------------------------------------------------------------ states of other parameters
def test_state_of_other_shapes_is_refused_whole():
    """a momentum that would broadcast into a stack, one that fits no buffer, and one too few: refused before anything is taken over"""
    opt = optim.HipMuon([])
    opt.momentum_buffers = [torch.zeros(3, 4, 5), torch.zeros(6, 7)]
    ok = torch.ones(3, 4, 5)
    for bad in ([torch.ones(4, 5), torch.ones(6, 7)], [torch.ones(1, 4, 5), torch.ones(6, 7)], [ok, torch.ones(7, 6)], [ok, torch.ones(7)], [ok]):
        with pytest.raises(ValueError, match="other parameters"):
            opt.load_state_dict({"step": 9, "lr": 0.5, "momentum_buffers": bad})
    assert opt.step_count == 0 and opt.lr == 0.02 and not any(b.any() for b in opt.momentum_buffers)
    opt.load_state_dict({"step": 9, "lr": 0.5, "momentum_buffers": [ok, torch.ones(6, 7)]})
    assert opt.step_count == 9 and opt.lr == 0.5 and all(b.all() for b in opt.momentum_buffers)


def test_a_refused_step_does_not_count():
    opt = optim.HipMuon([])
    p = torch.nn.Parameter(torch.zeros(4, 5))
    opt.params, opt.momentum_buffers = [p], [torch.zeros(4, 6)]
    p.grad = torch.zeros(4, 5)
    with pytest.raises(RuntimeError, match="has changed"):
        opt.step()
    assert opt.step_count == 0


# ------------------------------------------------------------------------------------------------ the polynomial's bound
@pytest.mark.parametrize("abc", [ABC, (2.0, -1.5, 0.5), (1.5, -0.5, 0.0), (3.0, -16 / 5, 6 / 5), (1.0, 0.0, 0.0), (3.9, -4.0, 0.0), (3.9, -4.0, 1e-17),
                                 (3.9, -4.0, -1e-17), (1.5, -0.5, 1e-20), (-3.0, 3.5, 1e-18), (0.0, 0.0, 1.0), (0.5, 0.0, 1.0), (1.0, 1.0, -0.25),
                                 (3.0, -3.0, 5e-324), (1e200, -1e200, 1e200)])
def test_bound_that_the_kernels_rely_on(abc):
    """what _ns_check returns is a power of two that the polynomial stays under, on a fine grid of every iterate's singular values; what
    leaves the range is refused, however small the leading coefficient"""
    a, b, c = abc
    v, most, polynomial = torch.linspace(0, 1, 100001, dtype=torch.float64), 0.0, 0.0
    for _ in range(3):
        p = (a + b * v ** 2 + c * v ** 4).abs()
        polynomial = max(polynomial, float(p.max()))
        top = float((v * p).max())
        most = max(most, polynomial, top * top)
        v = torch.linspace(0, top, 100001, dtype=torch.float64)
    if most > 15.0:
        with pytest.raises(ValueError):
            optim._ns_check(3, *abc)
    else:
        assert most < 14.9  # (no case sits on the border)
        grow = optim._ns_check(3, *abc)
        assert grow >= polynomial and math.log2(grow) % 1 == 0 and 1 <= grow <= 16


# ------------------------------------------------------------------------------------------------ stacks that no launch holds
def test_stacks_of_too_many_tiles_are_refused():
    """65535 rows of 20000 elements: 20.5 million tiles of 256 threads, more than 2^32; 16000 are the most"""
    from presight_amd._lib import check, lib

    h = lib()
    optim._matrices(torch.empty(65535, 1, 16000, device="meta"), "g")
    assert h.ps_newton_schulz_workspace(65535, 1, 16000) > 0
    for shape in ((65535, 1, 20000), (65535, 20000, 1), (65535, 1, 1 << 20), (16500, 64, 65536)):
        with pytest.raises(ValueError, match="tiles"):
            optim._matrices(torch.empty(shape, device="meta"), "g")
        assert h.ps_newton_schulz_workspace(*shape) == 0
        with pytest.raises(RuntimeError, match="sizes out of range"):
            check(h.ps_newton_schulz(256, *shape, 0, 5, 1.0, 0.0, 0.0, 1.0, 0.0, 256, 256, None), "ps_newton_schulz")


# ------------------------------------------------------------------------------------------------ entries of very different size
def uneven(m, n, kind, size, seed=19):
    """normal numbers, among them an entry, a row or a column `size` times the rest, or rows of every size between"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g)
    if kind == "entry":
        x[m // 3, n // 2] = size
    elif kind == "row":
        x[m // 2] *= size
    elif kind == "column":
        x[:, n // 3] *= size
    else:
        x *= size ** torch.rand(m, 1, generator=g)
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e3, 1e5, 1e6, 1e8, 1e10])
@pytest.mark.parametrize("m,n,kind", [(200, 300, "entry"), (200, 300, "row"), (200, 300, "column"), (300, 200, "rows"), (385, 1290, "entry"),
                                      (1290, 385, "row"), (64, 48, "entry"), (70, 3000, "entry")])
def test_outliers(dev, m, n, kind, size):
    """what is small beside the largest entries keeps its bits: the bound of evenly sized ones holds"""
    x = uneven(m, n, kind, size)
    check(optim.newton_schulz(x.to(dev)), x)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 8, 12])
def test_outliers_over_more_steps(dev, steps):
    """each step lifts the small directions further, and with them what rounding left there"""
    for kind, size in (("entry", 1e6), ("entry", 1e8), ("row", 1e5)):
        x = uneven(200, 300, kind, size)
        check(optim.newton_schulz(x.to(dev), steps=steps), x, steps)


@pytest.mark.gpu
def test_an_outlier_in_a_stack_of_large_tiles(dev):
    x = torch.stack([uneven(600, 700, k, s, seed=i) for i, (k, s) in enumerate([("entry", 1e6), ("row", 1e5), ("entry", 1.0), ("column", 1e8)] * 3)])
    y = optim.newton_schulz(x.to(dev)).cpu()
    for got, g in zip(y[:4], x[:4]):
        check(got, g)
    ref = iterate(x.to(dev).double()).cpu()
    for got, want in zip(y, ref):  # (the same four kinds again: 16 units of the norm or four times what plain fp32 is off by, 2e-6 of it)
        assert float((got.double() - want).norm()) <= 8e-6 * float(want.norm())


# ------------------------------------------------------------------------------------------------ a layer's gradients and the step on them
@pytest.mark.gpu
def test_a_layer_and_its_step_apart(dev):
    """the gradients of two expert layers against 64 bits, bounded by the sums of absolute values they are made of, and the step against the
    definition on those very gradients"""
    from presight_amd import experts

    g = torch.Generator().manual_seed(24)
    N, k, E, D, H = 700, 2, 5, 72, 96
    ids = torch.randint(-1, E, (N, k), generator=g)
    x, gates, dy = torch.randn(N, D, generator=g), torch.rand(N, k, generator=g), torch.randn(N, D, generator=g)
    start = [torch.randn(E, H, D, generator=g) / D ** 0.5, torch.randn(E, D, H, generator=g) / H ** 0.5]
    params = [torch.nn.Parameter(t.to(dev)) for t in start]
    opt = optim.HipMuon(params, lr=0.02, weight_decay=0.01)
    plan = experts.expert_plan(ids.to(dev), E)
    a = experts.expert_linear(experts.expert_dispatch(x.to(dev), plan), params[0], None, plan)
    h = torch.relu(a)
    experts.expert_combine(experts.expert_linear(h, params[1], None, plan), gates.to(dev), plan).backward(dy.to(dev))
    opt.step()
    # (which hidden values are cut off is taken from the rows as they came: next to zero a rounding decides it)
    open_ = (a.detach() > 0).cpu()
    place, off = plan.dst.cpu().long(), plan.offsets.tolist()
    src = plan.src.cpu().long()
    for size in (lambda t: t, torch.abs):  # the gradients, and the sums of their terms' absolute values
        xs, w1, w2 = size(x.double()), size(start[0].double()), size(start[1].double())
        grads = [torch.zeros_like(w1), torch.zeros_like(w2)]
        for e in range(E):
            rows = slice(off[e], off[e + 1])
            f = src[rows]
            d = size(dy.double())[f // k] * gates.double().reshape(-1)[f][:, None]
            hid = (xs[f // k] @ w1[e].T) * open_[rows]
            grads[1][e] = d.T @ hid
            grads[0][e] = ((d @ w2[e]) * open_[rows]).T @ xs[f // k]
        if size is torch.abs:
            sums = grads
        else:
            ref = grads
    terms = D + H + int(max(b - a for a, b in zip(off, off[1:]))) + 70
    for p, want, absum, w in zip(params, ref, sums, start):
        assert ((p.grad.cpu().double() - want).abs() <= terms * 2.0 ** -23 * absum).all()
        grad = p.grad.cpu()
        buf = (1 - 0.95) * grad
        u = 0.95 * buf + (1 - 0.95) * grad
        y = iterate(u.double())
        off_by = torch.maximum(4 * norms(iterate(u).double() - y), 16 * 2.0 ** -24 * norms(y))  # (of check(), per matrix)
        rate = 0.02 * math.sqrt(max(1.0, w.shape[1] / w.shape[2]))
        new = (1 - 0.02 * 0.01) * w.double() - rate * y
        # (u is the same bits here and there; the parameter carries the roundings of keep, of rate and of its two operations)
        slack = rate * off_by + 4 * 2.0 ** -24 * (norms(w) + rate * norms(y))
        assert (norms(p.detach().cpu().double() - new) <= slack).all()
    assert int((place >= 0).sum()) == off[-1]
