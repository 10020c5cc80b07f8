"""Dense layers, experts and their order in calls at the edges of what they allow: values that are not finite, addresses that are not aligned, many experts,
padded batches, shared and broadcast operands, two streams, two graphs.  Tolerances are those of the dense layers' tests."""
import ctypes as C

import pytest
import torch

from tests import test_dense_act_gpu as single
from tests import test_experts_cpu as cabi
from tests import test_experts_gpu as experts_tests

pytestmark = pytest.mark.gpu

ACTS = {None: 0, "silu": 1, "tanh": 2, "sigmoid": 3, "abs": 4}


def _random(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("act", [None, "sigmoid"])
@pytest.mark.parametrize("M,K,N", [(200, 40, 72), (700, 64, 130), (3000, 33, 20)])
def test_weight_gradients_that_are_not_finite(M, K, N, act):
    """An infinity in x reaches its column of the weight gradient, a NaN in the cotangent its row; everything else is as without them."""
    from fasteq_b200.ops.dense_act import dense_act
    x, w, b, _, g = single._inputs(M, K, N, torch.float32)
    want = single.reference(x, w, b, None, g, act, single.U[torch.float32])
    z = x.double() @ w.double().t() + b.double()
    # the layer's own values keep to the clean x: what is not finite comes in through the operands of the gradient
    xg, wg, bg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
    y = dense_act(xg, wg, bg, act)
    g[M // 2, N - 1] = float("nan")
    g[M - 1, 0] = float("inf")
    gx, gw, gb = torch.autograd.grad(y, (xg, wg, bg), g.cuda())
    gz = g * single._slope(act, z).float()
    pattern = gz.t() @ x                                                  # FP32 on the CPU: where it is finite, and where not
    assert torch.equal(gw.cpu().isnan(), pattern.isnan()) and torch.equal(gw.cpu().isinf(), pattern.isinf())
    assert torch.equal(gw.cpu()[0].sign(), pattern[0].sign())
    assert torch.equal(gb.cpu().isfinite(), gz.sum(0).isfinite())
    ok = pattern.isfinite()
    ref, tol = want["w"]
    off = (gw.cpu().double() - ref).abs()
    assert int(ok.sum()) == (N - 2) * K and torch.all(off[ok] <= tol[ok])
    rows = [r for r in range(M) if r not in (M // 2, M - 1)]
    ref, tol = want["x"]
    assert torch.all((gx.cpu().double() - ref).abs()[rows] <= tol[rows])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("act", ["silu", "tanh", "sigmoid", "abs"])
def test_activations_over_the_whole_line(act, dtype):
    """Values and slopes of a layer of one channel and weight one, from the smallest arguments to infinity and NaN.  Within 8 half steps of the value (of one,
    for slopes, and of the exponential's argument: FP32 rounds z log2(e), which moves exp by |z| half steps), or of the smallest normal number."""
    from fasteq_b200.ops.dense_act import dense_act
    inf = float("inf")
    z = torch.cat([s * torch.logspace(-30, 2, 3001, dtype=torch.float64) for s in (1, -1)])
    z = torch.cat([z, torch.linspace(-20, 20, 4001, dtype=torch.float64), torch.tensor([0.0, 88.0, -88.0, 709.0, -709.0, 750.0, -750.0, 3e30, -3e30, inf, -inf, float("nan")])])
    z = z.to(dtype).unsqueeze(1)
    leaf = z.cuda().requires_grad_(True)
    y = dense_act(leaf, torch.ones(1, 1, dtype=dtype, device="cuda"), None, act)
    (d,) = torch.autograd.grad(y.sum(), leaf)
    want = z.double().requires_grad_(True)
    ref = single.F[act](want)
    (slope,) = torch.autograd.grad(ref.sum(), want)
    y, d, ref, z = y.detach().cpu().double(), d.cpu().double(), ref.detach(), z.double()
    assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y.isinf(), ref.isinf())
    u, least = single.U[dtype], torch.finfo(dtype).tiny * 1e8 if dtype == torch.float64 else torch.finfo(dtype).tiny
    ok = ref.isfinite() & z.isfinite()
    reach = z.abs().clamp(max=800)                                       # beyond, the exponential is 0 in both types
    off, may = (y - ref).abs(), (8 + 2 * reach) * u * ref.abs() + least * (1 + reach)
    assert torch.all(off[ok] <= may[ok]), float((off - may)[ok].max())
    # a slope is a sum of terms up to one and |z| exp(-|z|) <= 0.4, each off by what the sigmoid is, in FP32 by |z| half steps of it
    off, may = (d - slope).abs(), 9 * u * torch.ones_like(d) + 2 * reach * u * (slope.abs() + torch.exp(-reach)) + least * (1 + reach)
    assert torch.all(off[ok] <= may[ok]), float((off - may)[ok].max())


@pytest.mark.parametrize("act", ["silu", "tanh", None])
@pytest.mark.parametrize("M,K,N", [(300, 64, 96), (200, 33, 50), (150, 600, 40)])
def test_values_that_are_not_finite_with_a_residual(M, K, N, act):
    """Rows whose sums are not finite are formed again, with bias, activation, residual and slope; the others are as without them."""
    from fasteq_b200.ops.dense_act import dense_act
    x, w, b, r, g = single._inputs(M, K, N, torch.float32)
    clean = single.run(x, w, b, r, g, act)
    wild = [7, M // 2, M - 1]
    x[7], x[M // 2, 3], x[M - 1, K - 1] = 2.0 ** 115, float("inf"), float("nan")       # 2^115: finite, its sums are too
    leaf = x.cuda().requires_grad_(True)
    y = dense_act(leaf, w.cuda(), b.cuda(), act, r.cuda())
    (gx,) = torch.autograd.grad(y, leaf, g.cuda())
    z = x @ w.t() + b
    pattern = single.F[act](z) + r
    y, gx = y.detach().cpu(), gx.cpu()
    assert torch.equal(y.isnan(), pattern.isnan()) and torch.equal(y.isinf(), pattern.isinf())
    want = single.reference(x[7:8], w, b, r[7:8], g[7:8], act, single.U[torch.float32])
    for n, v in (("y", y), ("x", gx)):
        ref, tol = want[n]
        assert torch.all((v[7:8].double() - ref).abs() <= tol), n
    others = [i for i in range(M) if i not in wild]
    assert torch.equal(y[others], clean["y"].cpu()[others]) and torch.equal(gx[others], clean["x"].cpu()[others])
    assert gx[M - 1].isnan().all() or act is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("K,N", [(64, 64), (20, 33)])
def test_one_experts_infinities_stay_with_it(K, N, dtype):
    from fasteq_b200.ops.experts import expert_dense, expert_plan
    r, X, tokens = _random(3, dtype), 4, 150
    e = torch.arange(tokens, dtype=torch.int32) % X
    rows, w, b, g = r(tokens, K), r(X, N, K) / K ** 0.5, r(X, N), r(tokens, N)
    plan = expert_plan(e.cuda(), X)
    begin, end = int(plan.offsets[1]), int(plan.offsets[2])

    def run(rows, w, g):
        leaves = [t.cuda().requires_grad_(True) for t in (rows, w, b)]
        y = expert_dense(*leaves[:2], plan, leaves[2], "silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, g.cuda())]
    clean = run(rows, w, g)
    rows[begin + 3, 1], rows[end - 1, K - 1], w[1, 2, 3], g[begin] = float("inf"), float("nan"), 3e38, float("-inf")
    for i, (a, c) in enumerate(zip(run(rows, w, g), clean)):
        others = [j for j in range(tokens) if not begin <= j < end] if i < 2 else [0, 2, 3]
        assert torch.equal(a[others], c[others])
        assert not torch.isfinite(a[begin:end] if i < 2 else a[1]).all()


def _addressed(t, offset, fill=0.0):
    """A copy on the GPU whose address is `offset` elements behind an aligned one."""
    base = torch.full((t.numel() + 8,), fill, dtype=t.dtype, device="cuda")
    v = base[offset:offset + t.numel()].view(t.shape)
    v.copy_(t)
    return v, base


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("M,K,N,act", [(70, 64, 64, "silu"), (300, 33, 50, None), (600, 20, 68, "tanh"), (90, 640, 24, "abs")])
def test_addresses_through_the_c_interface(M, K, N, act, offset, dtype):
    """All operands and results one element off alignment, or none; nothing is written outside the results."""
    lib = cabi._core()
    x, w, b, res, g = single._inputs(M, K, N, dtype)
    want = single.reference(x, w, b, res, g, act, single.U[dtype])
    p = cabi.Problem(dtype=0 if dtype == torch.float32 else 1, k=K, n=N, experts=1, inner=1, act=ACTS[act], rows=M)
    keep = []

    def put(t):
        v, base = _addressed(t, offset, 77.0)
        keep.append((base, v))
        return v
    xd, wd, bd, rd, gd = (put(t) for t in (x, w, b, res, g))
    nan = float("nan")
    y, gx, gw, gb = (put(torch.full_like(t, nan)) for t in (g, x, w, b))
    slope = torch.full((M, (N + 3) // 4 * 4 if dtype == torch.float32 else N), nan, dtype=dtype, device="cuda")
    ptr = lambda t: C.c_void_p(t.data_ptr())
    scratch = []
    for backward in (0, 1):
        need = C.c_int64(0)
        assert lib.fasteq_product_scratch(C.byref(p), C.c_int32(backward), C.byref(need)) == 0
        scratch.append((torch.empty(need.value + 16, dtype=torch.uint8, device="cuda"), need))
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.fasteq_product_forward(C.byref(p), ptr(xd), ptr(wd), ptr(bd), ptr(rd), None, ptr(y), ptr(slope), ptr(scratch[0][0]), scratch[0][1], stream) == 0
    assert lib.fasteq_product_backward(C.byref(p), ptr(xd), ptr(wd), ptr(gd), ptr(slope) if act else None, None, ptr(gx), ptr(gw), ptr(gb), ptr(scratch[1][0]),
                                       scratch[1][1], stream) == 0
    single.check({"y": y, "x": gx, "w": gw, "b": gb}, want)
    for base, v in keep:
        assert torch.all(base[:offset] == 77.0) and torch.all(base[offset + v.numel():] == 77.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("tokens,experts,K,N", [(400, 150, 256, 24), (400, 400, 288, 40), (900, 1024, 16, 12), (300, 3, 640, 70), (200, 1000, 330, 8)])
def test_many_experts_and_long_rows(tokens, experts, K, N, dtype):
    from fasteq_b200.ops.experts import expert_dense, expert_plan
    r = _random(tokens + experts, dtype)
    e = experts_tests._experts(tokens, 1, experts, 0.1)
    rows, w, b, go = r(tokens, K), r(experts, N, K) / K ** 0.5, r(experts, N), r(tokens, N)
    plan = expert_plan(e.cuda(), experts)
    leaves = [t.cuda().requires_grad_(True) for t in (rows, w, b)]
    y = expert_dense(leaves[0], leaves[1], plan, leaves[2], "silu")
    grads = torch.autograd.grad(y, leaves, go.cuda())
    want = experts_tests._dense_reference(rows, w, b, experts_tests._order(e, experts)[1], "silu", go, single.U[dtype])
    for n, v in zip(("y", "x", "w", "b"), (y.detach(), *grads)):
        ref, tol = want[n]
        assert torch.all((v.cpu().double() - ref).abs() <= tol), n


def test_all_entries_to_one_expert_and_to_none():
    """One expert with every row (several chunks of its weight gradient), and no expert with any."""
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    x, w, b, _, g = single._inputs(5000, 32, 48, torch.float32)
    for number in (2, -1):
        plan = expert_plan(torch.full((5000,), number, dtype=torch.int64, device="cuda"), 4)
        leaves = [t.cuda().requires_grad_(True) for t in (x, torch.stack([w] * 4), torch.stack([b] * 4))]
        y = expert_combine(expert_dense(expert_gather(leaves[0], plan), leaves[1], plan, leaves[2], "silu"), plan)
        grads = torch.autograd.grad(y, leaves, g.cuda())
        if number < 0:
            assert not any(t.any() for t in (y, *grads))
            continue
        want = single.reference(x, w, b, None, g, "silu", single.U[torch.float32])
        single.check({"y": y.detach(), "x": grads[0], "w": grads[1][2], "b": grads[2][2]}, want)
        assert not grads[1][[0, 1, 3]].any() and not grads[2][[0, 1, 3]].any()


def test_a_padded_batch():
    """Padding given to no expert, NaN in its rows: values and gradients of the others are those of the batch without it, the padding's are zero."""
    data = experts_tests._mlp_inputs(70, 2, 5, 24, 40, torch.float32)
    x, e, weight = data[:3]

    def run(x, e, weight):
        args = [t.cuda() if i == 1 else t.cuda().requires_grad_(True) for i, t in enumerate((x, e, weight, *data[3:]))]
        y = experts_tests._mlp(*args)
        return [y.detach(), *torch.autograd.grad(y, [t for i, t in enumerate(args) if i != 1], torch.ones_like(y))]
    nan = float("nan")
    padded = run(torch.cat([x, torch.full((30, 24), nan)]), torch.cat([e, torch.full((30, 2), -1, dtype=e.dtype)]), torch.cat([weight, torch.full((30, 2), nan)]))
    for i, (a, c) in enumerate(zip(padded, run(x, e, weight))):
        assert torch.equal(a[:c.shape[0]], c) and (i > 2 or not a[c.shape[0]:].any())


def test_shared_and_broadcast_operands():
    """A bias and a residual that are expanded, a weight used twice, a single row."""
    from fasteq_b200.ops.dense_act import dense_act
    r = _random(8)
    x, w, c, row = r(50, 24), r(24, 24) / 5, r(1), r(1, 24)

    def both(f):
        out = []
        for dev, dt, layer in (("cuda", torch.float32, dense_act), ("cpu", torch.float64, lambda x, w, b=None, a=None, s=None: single.F[a](x @ w.t() + (0 if b is None else b)) + (0 if s is None else s))):
            leaves = [t.to(dt).to(dev).requires_grad_(True) for t in (x, w, c, row)]
            y = f(layer, *leaves)
            out.append([y.detach(), *torch.autograd.grad(y.square().sum(), leaves)])
        for a, e in zip(*out):
            # three layers of sums of 24 and a sum of 50 x 24 squares: 4 (1200 + 8) u at most, relative to the largest value
            assert float((a.cpu().double() - e).abs().max()) <= 4 * 1208 * 2.0 ** -24 * float(e.abs().max())
    both(lambda f, x, w, c, row: f(f(x, w, c.expand(24), "silu", row.expand(50, 24)), w, None, "tanh", x))
    both(lambda f, x, w, c, row: f(row[0], w.t(), c.expand(24), "silu") + x.mean() * 0)
    both(lambda f, x, w, c, row: f(row.expand(50, 24), w, None, None, x) * c)


def test_two_streams_at_once():
    """Calls on two streams at the same time have scratch of their own."""
    from fasteq_b200.ops.dense_act import dense_act
    sets = []
    for i in range(2):
        x, w, b, _, g = (t.cuda() if t is not None else None for t in single._inputs(20_000 + i, 100, 130, torch.float32, residual=True, seed=i))
        sets.append((x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True), g))

    def step(i):
        x, w, b, g = sets[i]
        y = dense_act(x, w, b, "silu")
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), g))
    want = [step(0), step(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, c) for run in got[i] for a, c in zip(run, want[i]))


def test_two_graphs_of_one_pool():
    """Two captured steps share a memory pool; each replay gives what the step gives, in either order."""
    data = [experts_tests._mlp_inputs(900 + 50 * i, 2, 6, 40, 72, torch.float32, seed=i) for i in range(2)]
    args = [[t.cuda() if i == 1 else t.cuda().requires_grad_(True) for i, t in enumerate(d)] for d in data]

    def step(a):
        y = experts_tests._mlp(*a)
        return [y.detach(), *torch.autograd.grad(y, [t for i, t in enumerate(a) if i != 1], torch.ones_like(y))]
    want = [[t.clone() for t in step(a)] for a in args]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if i else None):
            outs.append(step(args[i]))
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        assert all(torch.equal(a, c) for a, c in zip(outs[i], want[i]))


def test_extents_beyond_32_bits_are_refused():
    from fasteq_b200.ops.dense_act import dense_act
    from fasteq_b200.ops.experts import expert_combine, expert_gather, expert_plan
    one, big = torch.zeros(1, 1, device="cuda"), 2 ** 32 + 5
    with pytest.raises(ValueError, match="dense_act: channels"):
        dense_act(one, one.expand(big, 1))
    with pytest.raises(ValueError, match="dense_act: channels"):
        dense_act(one.expand(1, big), one.expand(1, big))
    plan = expert_plan(torch.zeros(1, dtype=torch.int64, device="cuda"), 1)
    with pytest.raises(ValueError, match="expert_gather: a row's values"):
        expert_gather(one.expand(1, big), plan)
    with pytest.raises(ValueError, match="expert_combine: a row's values"):
        expert_combine(one.expand(1, big), plan)


def test_dual_tensors_are_refused():
    """Forward-mode differentiation is not offered: a tangent is not dropped in silence."""
    import torch.autograd.forward_ad as forward_ad
    from fasteq_b200.ops.dense_act import dense_act
    from fasteq_b200.ops.experts import expert_combine, expert_gather, expert_plan
    plan = expert_plan(torch.tensor([0, 1, 0], device="cuda"), 2)
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(3, 4, device="cuda"), torch.ones(3, 4, device="cuda"))
        for call in (lambda: dense_act(x, torch.ones(2, 4, device="cuda")), lambda: expert_gather(x, plan), lambda: expert_combine(x, plan)):
            with pytest.raises(RuntimeError):
                call()
