"""Dense layers and experts where the result is known bit for bit, or to a step of the type: selections, whole numbers, single rows.

FP32 goes through three bf16 parts per operand.  Where a sum has one term, or terms that are whole numbers whose sums stay below 2^24, nothing is rounded or
truncated on the way, so the results have to be equal; a product that stands alone is off by what the split leaves out (3 x 2^-27), by the small parts' own sums
(2^-28) and by one rounding, together less than 2 u, u = 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _random(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)


def _whole(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randint(-3, 4, s, generator=g).to(dtype)


def _grads(y, leaves, g):
    return [t.cpu() for t in torch.autograd.grad(y, leaves, g.cuda())]


@pytest.mark.parametrize("K,N", [(16, 64), (64, 64), (128, 40), (256, 96), (512, 64), (640, 33), (1664, 20), (99, 130)])
def test_one_hot_rows_select_the_weights(K, N):
    """A species embedding through a dense layer: every value is a weight; a one-hot cotangent selects rows of the weight for grad_x."""
    from fasteq_b200.ops.dense_act import dense_act
    r, M = _random(K), 300
    w, x = r(N, K), torch.zeros(M, K)
    pick = torch.arange(M) * 7 % K
    scale = torch.tensor([1.0, -4.0, 0.125])[torch.arange(M) % 3]
    x[torch.arange(M), pick] = scale
    assert torch.equal(dense_act(x.cuda(), w.cuda()).cpu(), scale[:, None] * w[:, pick].t())
    leaf = r(M, K).cuda().requires_grad_(True)
    g, to = torch.zeros(M, N), torch.arange(M) * 11 % N
    g[torch.arange(M), to] = scale
    (gx,) = _grads(dense_act(leaf, w.cuda()), [leaf], g)
    assert torch.equal(gx, scale[:, None] * w[to])


@pytest.mark.parametrize("K", [32, 64, 256, 512, 67])
def test_identity_and_permutation_weights_return_the_rows(K):
    from fasteq_b200.ops.dense_act import dense_act
    x, order = _random(K)(500, K), torch.randperm(K, generator=torch.Generator().manual_seed(K))
    assert torch.equal(dense_act(x.cuda(), torch.eye(K, device="cuda")).cpu(), x)
    leaf = x.cuda().requires_grad_(True)
    y = dense_act(leaf, torch.eye(K)[order].cuda())
    assert torch.equal(y.detach().cpu(), x[:, order])
    g = _random(K + 1)(500, K)
    (gx,) = _grads(y, [leaf], g)
    assert torch.equal(gx[:, order], g)


# rows at the ends of 32-row blocks, of chunks of 64 and 288 rows, of the tensor
@pytest.mark.parametrize("M,K,N", [(200, 64, 64), (257, 128, 96), (1000, 33, 20), (5000, 256, 130), (40_000, 33, 20)])
def test_one_row_of_the_cotangent(M, K, N):
    """The weight gradient is that row's outer product, whatever the number of rows around it; the bias gradient the row itself."""
    from fasteq_b200.ops.dense_act import dense_act
    r = _random(M + K)
    x, w, b, row = r(M, K), r(N, K), r(N), r(N)
    leaves = [t.cuda().requires_grad_(True) for t in (w, b)]
    y = dense_act(x.cuda(), leaves[0], leaves[1])
    for at in sorted({0, 31, 32, 63, 64, 127, 255, 256, 287, 288, M // 2, M - 33, M - 32, M - 1}):
        if not 0 <= at < M:
            continue
        g = torch.zeros(M, N)
        g[at] = row
        gw, gb = torch.autograd.grad(y, leaves, g.cuda(), retain_graph=True)
        want = row.double()[:, None] * x[at].double()
        assert torch.all((gw.cpu().double() - want).abs() <= 2 * U * want.abs()), at
        assert torch.equal(gb.cpu(), row), at


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("M,K,N", [(1, 8, 8), (129, 64, 65), (1000, 130, 66), (5000, 300, 48), (148 * 128 + 5, 64, 64), (40_000, 33, 20), (20_011, 128, 256)])
def test_whole_numbers(M, K, N, dtype):
    """Sums of up to 40,000 products of numbers up to 3: a row, a block or a chunk that were lost or counted twice would show."""
    from fasteq_b200.ops.dense_act import dense_act
    r = _whole(M + K, dtype)
    x, w, b, s, g = r(M, K), r(N, K), r(N), r(M, N), r(M, N)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b, s)]
    y = dense_act(leaves[0], leaves[1], leaves[2], None, leaves[3])
    got = [y.detach().cpu(), *_grads(y, leaves, g)]
    x, w, b, s, g = (t.double() for t in (x, w, b, s, g))
    for a, e in zip(got, (x @ w.t() + b + s, g @ w, g.t() @ x, g.sum(0), g)):
        assert torch.equal(a.double(), e)


@pytest.mark.parametrize("N", [1, 7, 8, 9, 16, 17, 31, 32, 33])
@pytest.mark.parametrize("K", [1, 8, 15, 16, 17, 32, 100])
def test_whole_numbers_of_few_channels(K, N):
    """FP64 has narrow tiles for these, of 8, 16 and 32 columns; one matrix and several."""
    from fasteq_b200.ops.dense_act import dense_act
    from fasteq_b200.ops.experts import expert_dense, expert_plan
    r, M, X = _whole(K + 50 * N, torch.float64), 777, 5
    x, w, b, s, g = r(M, K), r(X, N, K), r(X, N), r(M, N), r(M, N)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w[0], b[0], s)]
    y = dense_act(leaves[0], leaves[1], leaves[2], "abs", leaves[3])
    z = x @ w[0].t() + b[0]
    gz = g * z.sign()
    for a, e in zip((y.detach().cpu(), *_grads(y, leaves, g)), (z.abs() + s, gz @ w[0], gz.t() @ x, gz.sum(0), g)):
        assert torch.equal(a, e)
    e = torch.arange(M) * 13 % (X + 1) - 1
    plan = expert_plan(e.cuda(), X)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = expert_dense(leaves[0], leaves[1], plan, leaves[2])
    got = [y.detach().cpu(), *_grads(y, leaves, g)]
    ends = plan.offsets.tolist()
    want = [torch.zeros_like(t) for t in (g, x, w, b)]
    for k in range(X):
        rows = slice(ends[k], ends[k + 1])
        want[0][rows], want[1][rows], want[2][k], want[3][k] = x[rows] @ w[k].t() + b[k], g[rows] @ w[k], g[rows].t() @ x[rows], g[rows].sum(0)
    for a, c in zip(got, want):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("tokens,slots,experts,K,N", [(40, 2, 5, 33, 7), (3000, 2, 8, 64, 128), (20_011, 1, 89, 64, 64), (900, 1, 600, 300, 12), (9000, 3, 2, 40, 72)])
def test_whole_numbers_through_experts(tokens, slots, experts, K, N, dtype):
    """The order, the rows there, every expert's product and the weighted way back, with all gradients."""
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    r = _whole(tokens + K, dtype)
    e = torch.randint(-1, experts, (tokens, slots), generator=torch.Generator().manual_seed(tokens))
    x, w, b, weight, g = r(tokens, K), r(experts, N, K), r(experts, N), r(tokens, slots), r(tokens, N)

    def framework(x, w, b, weight):
        plan = expert_plan(e.cuda(), experts)
        return expert_combine(expert_dense(expert_gather(x, plan), w, plan, b), plan, weight)

    def definition(x, w, b, weight):
        y = torch.zeros(tokens, N, dtype=torch.float64)
        for k in range(experts):
            t, s = (e == k).nonzero(as_tuple=True)
            y = y.index_add(0, t, weight[t, s, None] * (x[t] @ w[k].t() + b[k]))
        return y
    out = []
    for f, to in ((framework, lambda t: t.cuda()), (definition, lambda t: t.double())):
        leaves = [to(t).requires_grad_(True) for t in (x, w, b, weight)]
        y = f(*leaves)
        out.append([t.detach().cpu().double() for t in (y, *torch.autograd.grad(y, leaves, to(g)))])
    for a, c in zip(*out):
        assert torch.equal(a, c)
