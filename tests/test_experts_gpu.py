"""Experts: the order of entries, rows there and back, products of all experts, against plain torch in float64.

Tolerances: those of ``test_dense_act_gpu`` for products; a weighted sum over S slots carries at most (S + 1) u of its terms' magnitudes, a dot product of
C values (C + 8) u, u half a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}


def _experts(tokens, slots, experts, none=0.0, seed=0, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed + tokens + 31 * experts)
    e = torch.randint(0, experts, (tokens, slots), generator=g) // torch.randint(1, 3, (tokens, slots), generator=g)     # low ones more often
    return e.masked_fill(torch.rand(tokens, slots, generator=g) < none, -1).to(dtype)


def _order(expert, experts):
    key = torch.where(expert.reshape(-1) < 0, experts, expert.reshape(-1)).long()
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel())
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    return position.view(expert.shape), torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])


PLANS = [(0, 1, 4), (1, 1, 1), (5, 2, 3), (192, 2, 8), (33, 1, 1024), (4096, 1, 1024), (4097, 1, 2), (5000, 3, 1), (20_011, 2, 89), (150_001, 4, 256)]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,slots,experts", PLANS)
def test_plan(tokens, slots, experts, dtype):
    from fasteq_b200.ops.experts import expert_device_status, expert_plan
    for none in (0.0, 0.3, 1.0):
        e = _experts(tokens, slots, experts, none, dtype=dtype)
        plan = expert_plan(e.cuda(), experts)
        position, offsets = _order(e, experts)
        assert plan.position.dtype == plan.offsets.dtype == torch.int32
        assert torch.equal(plan.position.cpu().long(), position) and torch.equal(plan.offsets.cpu().long(), offsets)
    assert expert_device_status() == 0


def test_plan_of_one_slot_strides_and_numbers_out_of_range():
    from fasteq_b200.ops.experts import expert_plan
    from fasteq_b200.status import device_status
    e = _experts(100, 2, 5, 0.2)
    assert torch.equal(expert_plan(e[:, 1].cuda(), 5).position, expert_plan(e[:, 1:].contiguous().cuda(), 5).position)
    assert torch.equal(expert_plan(e.cuda().t().contiguous().t(), 5).position.cpu().long(), _order(e, 5)[0])
    assert device_status() == {}
    bad = e.clone().long()
    bad[3, 0], bad[50, 1], bad[51, 0] = 5, 2 ** 40, -7
    plan = expert_plan(bad.cuda(), 5)
    assert device_status() == {"experts": 2} and device_status() == {}
    position, offsets = _order(torch.where(bad >= 5, -1, bad), 5)
    assert torch.equal(plan.position.cpu().long(), position) and torch.equal(plan.offsets.cpu().long(), offsets)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("tokens,slots,experts,shape", [(0, 2, 4, (8,)), (1, 1, 1, (1,)), (7, 3, 4, (3,)), (192, 2, 8, (128,)), (100, 1, 89, (33,)),
                                                        (100, 4, 5, (4, 3, 5)), (301, 2, 3, (512,)), (64, 2, 3, (2050,)), (3000, 2, 8, (20,)), (5, 2, 2, (0,)),
                                                        (5, 2, 2, ())])
def test_rows_there_and_back(tokens, slots, experts, shape, dtype):
    from fasteq_b200.ops.experts import expert_combine, expert_gather, expert_plan
    g = torch.Generator().manual_seed(tokens)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)
    e = _experts(tokens, slots, experts, 0.2)
    x, rows, weight, gy, gr = r(tokens, *shape), r(tokens * slots, *shape), r(tokens, slots), r(tokens, *shape), r(tokens * slots, *shape)
    position, offsets = _order(e, experts)
    live = (e >= 0).double()
    C = max(1, x[:1].numel())
    over = lambda t: t.view(*t.shape, *[1] * len(shape))

    plan = expert_plan(e.cuda(), experts)
    xd, rd, wd = (t.cuda().requires_grad_(True) for t in (x, rows, weight))
    there, back, summed = expert_gather(xd, plan), expert_combine(rd, plan, wd), expert_combine(rd, plan)
    want = torch.zeros(tokens * slots, *shape, dtype=dtype)
    want[position] = torch.where(over(e >= 0), x.unsqueeze(1), 0.0)
    assert torch.equal(there.cpu(), want)
    u, terms = U[dtype], over(weight.double() * live) * rows.double()[position]
    assert torch.all((back.detach().cpu().double() - terms.sum(1)).abs() <= (slots + 1) * u * terms.abs().sum(1))
    ones = over(live) * rows.double()[position]
    assert torch.all((summed.detach().cpu().double() - ones.sum(1)).abs() <= slots * u * ones.abs().sum(1))

    (gx,) = torch.autograd.grad(there, xd, gr.cuda())
    ones = over(live) * gr.double()[position]
    assert torch.all((gx.cpu().double() - ones.sum(1)).abs() <= slots * u * ones.abs().sum(1))
    grows, gweight = torch.autograd.grad(back, (rd, wd), gy.cuda())
    want = torch.zeros(tokens * slots, *shape, dtype=torch.float64)
    want[position] = over(weight.double() * live) * gy.double().unsqueeze(1)
    assert torch.all((grows.cpu().double() - want).abs() <= u * want.abs())
    prod = (rows.double()[position] * gy.double().unsqueeze(1)).reshape(tokens, slots, math.prod(shape)) * live.unsqueeze(2)
    assert torch.all((gweight.cpu().double() - prod.sum(2)).abs() <= (C + 8) * u * prod.abs().sum(2))
    (only,) = torch.autograd.grad(expert_combine(rd.detach(), plan, wd), wd, gy.cuda())
    assert torch.equal(only, gweight)


def test_what_is_not_finite_in_entries_of_no_expert_goes_nowhere():
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    e = torch.tensor([[0, 1], [-1, 1], [-1, -1], [2, -1]])
    plan = expert_plan(e.cuda(), 3)
    x = torch.ones(4, 8)
    x[2] = float("nan")
    rows = expert_gather(x.cuda(), plan)
    assert torch.isfinite(rows).all() and int(plan.offsets[-1]) == 4 and torch.all(rows[4:] == 0)
    rows = torch.ones(8, 8, device="cuda")
    rows[4:] = float("nan")
    rows.requires_grad_(True)
    weight = torch.ones(4, 2)
    weight[e < 0] = float("inf")
    weight = weight.cuda().requires_grad_(True)
    y = expert_combine(rows, plan, weight)
    assert torch.equal(y.detach().cpu()[:, 0], torch.tensor([2.0, 1.0, 0.0, 1.0]))
    gr, gw = torch.autograd.grad(y.sum(), (rows, weight))
    assert torch.all(gr[4:] == 0) and torch.all(gr[:4] == 1) and torch.equal(gw.cpu(), torch.where(e < 0, 0.0, 8.0))
    w, b = torch.ones(3, 5, 8, device="cuda", requires_grad=True), torch.ones(3, 5, device="cuda", requires_grad=True)
    out = expert_dense(rows, w, plan, b, "silu")
    assert torch.all(out[4:] == 0)
    cot = torch.ones_like(out)
    cot[4:] = float("nan")
    for t in torch.autograd.grad(out, (rows, w, b), cot):
        assert torch.isfinite(t).all()


def _dense_reference(rows, w, b, offsets, act, g, u):
    """Product of every expert in float64: value, gradients, and how far a result may be off."""
    from tests import test_dense_act_gpu as single
    X, N, K = w.shape
    inner = rows[0].numel() // K if rows.shape[0] else 1
    flat, gf = rows.reshape(-1, K), g.reshape(-1, N)
    parts = {n: [torch.zeros(flat.shape[0], c, dtype=torch.float64) for _ in range(2)] for n, c in (("y", N), ("x", K))}
    parts["w"] = [torch.zeros(X, N, K, dtype=torch.float64) for _ in range(2)]
    parts["b"] = [torch.zeros(X, N, dtype=torch.float64) for _ in range(2)]
    for e in range(X):
        a, z = int(offsets[e]) * inner, int(offsets[e + 1]) * inner
        one = single.reference(flat[a:z], w[e], None if b is None else b[e], None, gf[a:z], act, u)
        for n in ("y", "x"):
            for k in range(2):
                parts[n][k][a:z] = one[n][k]
        for n in ("w", "b"):
            for k in range(2):
                parts[n][k][e] = one[n][k]
    return {n: (v[0], v[1]) for n, v in parts.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("tokens,slots,experts,inner,K,N,act,bias", [
    (1, 1, 3, (), 16, 16, "silu", True), (40, 2, 5, (), 33, 7, "tanh", True), (192, 2, 8, (), 128, 256, "silu", True), (64, 1, 200, (), 8, 12, None, False),
    (300, 3, 4, (), 64, 64, None, True), (129, 1, 1, (), 100, 70, "sigmoid", True), (50, 2, 6, (4,), 64, 64, None, False), (20, 1, 3, (3, 3), 20, 24, "abs", True),
    (0, 2, 4, (), 8, 8, "silu", True), (700, 2, 89, (), 64, 128, "silu", False), (9, 2, 3, (0,), 8, 4, None, True)])
def test_experts_products(tokens, slots, experts, inner, K, N, act, bias, dtype):
    from fasteq_b200.ops.experts import expert_dense, expert_plan
    g = torch.Generator().manual_seed(tokens + K)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)
    e = _experts(tokens, slots, experts, 0.15)
    rows, w, b, go = r(tokens * slots, *inner, K), r(experts, N, K) / K ** 0.5, r(experts, N) if bias else None, r(tokens * slots, *inner, N)
    plan = expert_plan(e.cuda(), experts)
    leaves = [t.cuda().requires_grad_(True) for t in (rows, w, b) if t is not None]
    y = expert_dense(leaves[0], leaves[1], plan, leaves[2] if bias else None, act)
    grads = torch.autograd.grad(y, leaves, go.cuda())
    want = _dense_reference(rows, w, b, _order(e, experts)[1], act, go, U[dtype])
    assert y.shape == go.shape
    for n, v in zip(("y", "x", "w", "b"), (y.detach(), *grads)):
        ref, tol = want[n]
        off = (v.cpu().double().reshape(ref.shape) - ref).abs()
        assert torch.all(off <= tol), (n, float((off - tol).max()))


def _mlp(x, e, weight, w1, b1, w2, b2):
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    plan = expert_plan(e, w1.shape[0])
    rows = expert_gather(x, plan)
    rows = expert_dense(rows, w1, plan, b1, "silu")
    return expert_combine(expert_dense(rows, w2, plan, b2), plan, weight)


def _plain_mlp(x, e, weight, w1, b1, w2, b2):
    y = torch.zeros_like(x)
    for t in range(x.shape[0]):
        for s in range(e.shape[1]):
            k = int(e[t, s])
            if k >= 0:
                h = torch.nn.functional.silu(x[t] @ w1[k].t() + b1[k])
                y = y.index_add(0, torch.tensor([t]), (weight[t, s] * (h @ w2[k].t() + b2[k])).unsqueeze(0))
    return y


def _mlp_inputs(tokens, slots, experts, K, H, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)
    return (r(tokens, K), _experts(tokens, slots, experts, 0.1), torch.softmax(r(tokens, slots), 1), r(experts, H, K) / K ** 0.5, r(experts, H),
            r(experts, K, H) / H ** 0.5, r(experts, K))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_a_whole_step(dtype):
    """Order, rows there, two layers and the way back, with all gradients, against a loop over entries in float64."""
    data = _mlp_inputs(60, 2, 5, 24, 40, dtype)
    cot = torch.randn(60, 24, generator=torch.Generator().manual_seed(1), dtype=torch.float64)

    def run(f, dev, dt):
        args = [t.to(dev) if i == 1 else t.to(dt).to(dev).requires_grad_(True) for i, t in enumerate(data)]
        y = f(*args)
        grads = torch.autograd.grad(y, [t for i, t in enumerate(args) if i != 1], cot.to(dt).to(dev))
        return [t.detach().cpu().double() for t in (y, *grads)]
    # two layers, sums of 24, 40 and up to 60 terms each way: 5 sums of (60 + 8) u at most, relative to the largest value
    for a, e in zip(run(_mlp, "cuda", dtype), run(_plain_mlp, "cpu", torch.float64)):
        assert float((a - e).abs().max()) <= 5 * 68 * U[dtype] * float(e.abs().max())


def test_gradients_against_differences():
    data = _mlp_inputs(5, 2, 3, 3, 4, torch.float64, seed=2)
    args = [t.cuda() if i == 1 else t.cuda().requires_grad_(True) for i, t in enumerate(data)]
    assert torch.autograd.gradcheck(_mlp, args)
    assert torch.autograd.gradgradcheck(_mlp, args)


def test_same_bits_streams_and_graph():
    """The same inputs give the same bits, on another stream too; a captured step follows other experts and weights."""
    data = _mlp_inputs(300, 2, 7, 32, 64, torch.float32)
    args = [t.cuda() if i == 1 else t.cuda().requires_grad_(True) for i, t in enumerate(data)]
    leaves = [t for i, t in enumerate(args) if i != 1]

    def step():
        y = _mlp(*args)
        return (y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y)))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    args[1].copy_(torch.flip(args[1], (0,)))
    with torch.no_grad():
        args[3].mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    e = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for bad, n in ((e.float(), 3), (e, 0), (e, 1025), (e.view(2, 2, 2), 3), (e[:, :0], 3)):
        with pytest.raises(ValueError, match="expert_plan"):
            expert_plan(bad, n)
    with pytest.raises(RuntimeError, match="no CPU path"):
        expert_plan(e.cpu(), 3)
    plan = expert_plan(e, 3)
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    for f in (lambda: expert_gather(z(8, 4), plan), lambda: expert_gather(z(4, 4).half(), plan), lambda: expert_combine(z(4, 4), plan),
              lambda: expert_combine(z(8, 4), plan, z(4)), lambda: expert_combine(z(8, 4), plan, z(4, 2).double()),
              lambda: expert_dense(z(8, 4), z(2, 5, 4), plan), lambda: expert_dense(z(8, 4), z(3, 5, 3), plan), lambda: expert_dense(z(8), z(3, 5, 1), plan),
              lambda: expert_dense(z(8, 4), z(3, 5, 4), plan, z(5)), lambda: expert_dense(z(8, 4), z(3, 5, 4), plan, activation="relu"),
              lambda: expert_dense(z(4, 4), z(3, 5, 4), plan)):
        with pytest.raises(ValueError, match="expert_"):
            f()
    with pytest.raises(TypeError, match="ExpertPlan"):
        expert_gather(z(4, 4), e)
