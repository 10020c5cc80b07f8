"""Dense layer with bias, activation and residual, against torch in float64.

Tolerances, per element, with u half a step of the type (FP32 2^-24, FP64 2^-53): a sum of K products carries at most (K + 8) u of the sum
of their magnitudes, in any order (the tensor cores' truncating additions, one per 16 products and 2 u each, and the products their split leaves
out, 3 x 2^-27, are less); the activations' slopes are below 1.1 and the slopes' own below 0.8; what an activation itself rounds is below
8 u of its value, or of one for its slope."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F = {None: lambda z: z, "silu": torch.nn.functional.silu, "tanh": torch.tanh, "sigmoid": torch.sigmoid, "abs": torch.abs}
U = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}


def _inputs(M, K, N, dtype, bias=True, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * M + 5 * K + N)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)
    return r(M, K), r(N, K) / max(K, 1) ** 0.5, 0.3 * r(N) if bias else None, r(M, N) if residual else None, r(M, N)


def _slope(act, z):
    z = z.detach().requires_grad_(True)
    return torch.autograd.grad(F[act](z).sum(), z)[0] if act else torch.ones_like(z)


def reference(x, w, b, r, g, act, u):
    """Values and gradients in float64, and how far a result may be from them."""
    x, w, b, r, g = (None if t is None else t.double() for t in (x, w, b, r, g))
    M, K, N = *x.shape, w.shape[0]
    z = x @ w.t() + (0 if b is None else b)
    ez = (K + 8) * u * (x.abs() @ w.abs().t() + (0 if b is None else b.abs()))
    y, d = F[act](z), _slope(act, z)
    ey = 1.1 * ez + 8 * u * y.abs() + u * (y.abs() + (0 if r is None else r.abs() + y.abs()))
    y = y if r is None else y + r
    gz, egz = g * d, g.abs() * (0.8 * ez + 9 * u if act else 0 * ez)
    out = {"y": (y, ey)}
    out["x"] = (gz @ w, (N + 8) * u * (gz.abs() @ w.abs()) + 2 * egz @ w.abs())
    out["w"] = (gz.t() @ x, (M + 8) * u * (gz.abs().t() @ x.abs()) + 2 * egz.t() @ x.abs())
    out["b"] = (gz.sum(0), (M + 8) * u * gz.abs().sum(0) + 2 * egz.sum(0))
    out["r"] = (g, 0 * g)
    return out


def run(x, w, b, r, g, act):
    from fasteq_b200.ops.dense_act import dense_act
    leaves = {n: t.cuda().requires_grad_(True) for n, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    y = dense_act(leaves["x"], leaves["w"], leaves.get("b"), act, leaves.get("r"))
    grads = torch.autograd.grad(y, list(leaves.values()), g.cuda())
    with torch.no_grad():
        alone = dense_act(leaves["x"], leaves["w"], leaves.get("b"), act, leaves.get("r"))
    assert torch.equal(y, alone)
    return {"y": y.detach(), **dict(zip(leaves, grads))}


def check(got, want):
    for n, v in got.items():
        ref, tol = want[n]
        assert v.shape == ref.shape, n
        off = (v.cpu().double() - ref).abs()
        assert torch.all(off <= tol), (n, float((off - tol).max()), float(off.max()))


SIZES = [(0, 8, 8), (1, 1, 1), (1, 128, 128), (5, 7, 3), (3, 33, 99), (64, 64, 64), (129, 64, 65), (192, 128, 128), (127, 20, 260), (257, 512, 40),
         (300, 100, 512), (1000, 130, 66), (40, 1664, 64), (70, 40, 1280), (5000, 32, 16)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_values_and_gradients(M, K, N, dtype):
    act = [None, "silu", "tanh", "sigmoid", "abs"][(M + N) % 5]
    data = _inputs(M, K, N, dtype, bias=(M + K) % 4 != 0, residual=K % 3 != 0)
    check(run(*data, act), reference(*data, act, U[dtype]))


@pytest.mark.parametrize("act", list(F))
def test_every_activation(act):
    for dtype in U:
        data = _inputs(200, 64, 72, dtype, seed=3)
        check(run(*data, act), reference(*data, act, U[dtype]))


@pytest.mark.parametrize("M,K,N", [(148 * 128 + 5, 64, 64), (40_000, 33, 20), (20_000, 128, 256)])
def test_many_rows(M, K, N):
    data = _inputs(M, K, N, torch.float32, seed=1)
    check(run(*data, "silu"), reference(*data, "silu", U[torch.float32]))


def test_no_less_precise_than_torch():
    """2-norm against float64: at most 1.5 times the error of torch's own FP32 evaluation, or 1e-6."""
    from fasteq_b200.ops.dense_act import dense_act
    g = torch.Generator(device="cuda").manual_seed(0)
    for M, K, N in ((20_000, 64, 64), (6_000, 512, 256), (4_000, 1664, 64)):
        x, w, b, go = (torch.randn(*s, generator=g, device="cuda") for s in ((M, K), (N, K), (N,), (M, N)))

        def all_of(f, dt):
            leaves = [t.to(dt).requires_grad_(True) for t in (x, w / K ** 0.5, b)]
            y = f(*leaves)
            return [t.detach().double() for t in (y, *torch.autograd.grad(y, leaves, go.to(dt)))]
        torch_form = lambda x, w, b: torch.nn.functional.silu(x @ w.t() + b)
        want, plain = all_of(torch_form, torch.float64), all_of(torch_form, torch.float32)
        got = all_of(lambda x, w, b: dense_act(x, w, b, "silu"), torch.float32)
        for ours, theirs, ref in zip(got, plain, want):
            e, t = float((ours - ref).norm() / ref.norm()), float((theirs - ref).norm() / ref.norm())
            assert e <= max(1e-6, 1.5 * t), (M, K, N, e, t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_strides_alignment_and_leading_dimensions(dtype):
    from fasteq_b200.ops.dense_act import dense_act
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype).cuda()
    u = U[dtype]

    def same(x, w, b, res):
        x2, r2 = x.reshape(-1, x.shape[-1]).cpu(), None if res is None else res.reshape(-1, w.shape[0]).cpu()
        want, tol = reference(x2, w.cpu(), None if b is None else b.cpu(), r2, torch.zeros(x2.shape[0], w.shape[0]), "silu", u)["y"]
        got = dense_act(x, w, b, "silu", res)
        assert got.shape == (*x.shape[:-1], w.shape[0])
        assert torch.all((got.reshape(want.shape).cpu().double() - want).abs() <= tol)

    w, b = r(64, 32), r(64)
    same(r(5, 31, 32), w, b, r(5, 31, 64))
    same(r(32), w, b, r(64))
    same(r(32, 150).t(), w, b, None)                                    # transposed rows
    same(r(150, 96)[:, 32:64], w, b, r(150, 128)[:, ::2])               # columns of wider rows, every other column
    same(r(150, 32), r(32, 64).t(), b, r(1, 64).expand(150, 64))        # transposed weight, broadcast residual
    flat = r(150 * 32 + 1)[1:].view(150, 32)                            # not 16-byte aligned
    same(flat, r(64 * 32 + 1)[1:].view(64, 32), r(65)[1:], r(150 * 64 + 1)[1:].view(150, 64))
    same(r(0, 32), w, b, r(0, 64))
    same(r(3, 0, 32), w, b, None)


def test_no_channels():
    from fasteq_b200.ops.dense_act import dense_act
    b = torch.randn(6, device="cuda")
    x, w = torch.zeros(3, 0, device="cuda", requires_grad=True), torch.zeros(6, 0, device="cuda", requires_grad=True)
    y = dense_act(x, w, b, "tanh")
    assert torch.allclose(y, torch.tanh(b).expand(3, 6), rtol=1e-6)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == (3, 0) and gw.shape == (6, 0)
    assert dense_act(torch.ones(3, 4, device="cuda"), torch.ones(0, 4, device="cuda")).shape == (3, 0)


def test_infinities_and_nan_stay_in_their_rows():
    """Values that are not finite, or whose sums are not, come out as torch's products give them; other rows and columns are untouched."""
    from fasteq_b200.ops.dense_act import dense_act
    x, w, b, _, _ = _inputs(300, 64, 96, torch.float32, seed=9)
    clean = dense_act(x.cuda(), w.cuda(), b.cuda()).cpu()
    x[7, 3], x[200, 60], x[201, 0], x[5] = float("inf"), float("nan"), -float("inf"), 3e38
    w[10, 3] = 0.0                                                       # inf * 0
    w[50] = 1.0
    got = dense_act(x.cuda(), w.cuda(), b.cuda()).cpu().double()
    want = (x @ w.t() + b).double()                                      # FP32, on the CPU
    for i in (7, 200, 201, 5):
        assert torch.equal(got[i].isnan(), want[i].isnan()) and torch.equal(got[i] == float("inf"), want[i] == float("inf"))
        assert torch.equal(got[i] == -float("inf"), want[i] == -float("inf"))
    rows = [i for i in range(300) if i not in (7, 200, 201, 5)]
    cols = [j for j in range(96) if j not in (10, 50)]
    assert torch.equal(got[rows][:, cols].float(), clean[rows][:, cols])


@pytest.mark.parametrize("big,small", [(1e30, 1e-30), (3e37, 1e-38), (1e-20, 1e-15)])
def test_the_whole_range_of_fp32(big, small):
    from fasteq_b200.ops.dense_act import dense_act
    x, w, _, _, _ = _inputs(200, 48, 40, torch.float32, seed=2)
    x, w = x * big, w * small
    want = x.double() @ w.double().t()
    off = (dense_act(x.cuda(), w.cuda()).cpu().double() - want).abs()
    # 2^-149: the spacing of FP32's smallest numbers, to which each of 48 products may be rounded
    assert torch.all(off <= 56 * 2.0 ** -24 * (x.double().abs() @ w.double().abs().t()) + 48 * 2.0 ** -149)


def test_gradients_against_differences():
    from fasteq_b200.ops.dense_act import dense_act
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).cuda().requires_grad_(True)
    for act in (None, "silu", "tanh", "sigmoid"):
        args = (r(5, 4), r(3, 4), r(3), r(5, 3))
        f = lambda x, w, b, res: dense_act(x, w, b, act, res)
        assert torch.autograd.gradcheck(f, args)
        assert torch.autograd.gradgradcheck(f, args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_higher_orders(dtype):
    """A force loss: the gradient of a scalar through the layer, differentiated with respect to weights and bias, and once more."""
    from fasteq_b200.ops.dense_act import dense_act
    x, w, b, _, v = _inputs(40, 24, 16, dtype, seed=6)

    def orders(f, dev, dt):
        xt, wt, bt = (t.to(dt).to(dev).requires_grad_(True) for t in (x, w, b))
        (gx,) = torch.autograd.grad((f(xt, wt, bt) * v.to(dt).to(dev)).sum(), xt, create_graph=True)
        second = torch.autograd.grad(gx.square().sum(), (wt, bt, xt), create_graph=True)
        third = torch.autograd.grad(sum(t.square().sum() for t in second), (wt, bt))
        return [t.detach().cpu().double() for t in (gx, *second, *third)]

    want = orders(lambda x, w, b: torch.nn.functional.silu(x @ w.t() + b), "cpu", torch.float64)
    got = orders(lambda x, w, b: dense_act(x, w, b, "silu"), "cuda", dtype)
    # sums of 24 to 40 products in a chain of a dozen operations, relative to the largest value
    for a, e in zip(got, want):
        assert float((a - e).abs().max()) <= 12 * 48 * U[dtype] * float(e.abs().max())


def test_only_the_gradients_asked_for():
    from fasteq_b200.ops.dense_act import dense_act
    x, w, b, r, g = (t.cuda() for t in _inputs(50, 16, 24, torch.float32))
    want = reference(x.cpu(), w.cpu(), b.cpu(), r.cpu(), g.cpu(), "tanh", U[torch.float32])
    for n, k in (("x", 0), ("w", 1), ("b", 2), ("r", 3)):
        leaves = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b, r))]
        (got,) = torch.autograd.grad(dense_act(leaves[0], leaves[1], leaves[2], "tanh", leaves[3]), leaves[k], g)
        check({n: got}, want)


def test_one_tensor_in_two_places_and_the_same_bits():
    from fasteq_b200.ops.dense_act import dense_act
    x = torch.randn(90, 48, device="cuda", requires_grad=True)
    w = torch.randn(48, 48, device="cuda") / 7
    f = lambda: torch.autograd.grad(dense_act(x, w, None, "silu", x).sum(), x)[0]      # x is the residual too
    xd = x.detach().double().requires_grad_(True)
    (want,) = torch.autograd.grad((torch.nn.functional.silu(xd @ w.double().t()) + xd).sum(), xd)
    a = f()
    assert torch.equal(a, f()) and float((a.double() - want).abs().max()) <= 120 * U[torch.float32] * 20
    y = torch.randn(5000, 48, device="cuda")
    assert torch.equal(dense_act(y, w, None, "silu"), dense_act(y, w, None, "silu"))


def test_side_stream_and_graph():
    """Launches go to the current stream; forward and backward are captured and replayed with other inputs."""
    from fasteq_b200.ops.dense_act import dense_act
    x, w, b, r, g = (t.cuda() for t in _inputs(500, 64, 96, torch.float32))
    x.requires_grad_(True), w.requires_grad_(True)

    def step():
        y = dense_act(x, w, b, "silu", r)
        return (y.detach(), *torch.autograd.grad(y, (x, w), g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(step(), eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x)), w.mul_(0.5), r.add_(1.0)
    graph.replay()
    assert all(torch.equal(a, e) for a, e in zip(out, step()))


def test_refusals():
    from fasteq_b200.ops.dense_act import dense_act
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    for kw in (dict(activation="gelu"), dict(bias=torch.zeros(5, device="cuda")), dict(bias=torch.zeros(6, 1, device="cuda")),
               dict(residual=torch.zeros(6, device="cuda")), dict(residual=torch.zeros(4, 6, device="cuda", dtype=torch.float64))):
        with pytest.raises(ValueError, match="dense_act"):
            dense_act(x, w, **kw)
    for a, c in ((x, torch.zeros(6, 7, device="cuda")), (x, w[0]), (x.half(), w.half()), (x, w.double()), (x.to(torch.int32), w)):
        with pytest.raises(ValueError, match="dense_act"):
            dense_act(a, c)
    with pytest.raises(RuntimeError, match="no CPU path"):
        dense_act(x, w.cpu())
