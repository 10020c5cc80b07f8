"""Activations of the dense layers, through a layer of one channel and weight one, where their argument is exact."""
import numpy as np
import pytest
import torch

from tests import test_dense_act_gpu as single

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}
INF = float("inf")


def _line(dtype, top):
    """Arguments from the smallest to `top` on both sides of zero, and dense ones between."""
    z = torch.cat([torch.logspace(-30, np.log10(top), 4001, dtype=torch.float64), torch.linspace(0, top, 20_001, dtype=torch.float64)])
    return torch.cat([z, -z]).to(dtype).unsqueeze(1)


def _run(z, act):
    from fasteq_b200.ops.dense_act import dense_act
    leaf = z.cuda().requires_grad_(True)
    y = dense_act(leaf, torch.ones(1, 1, dtype=z.dtype, device="cuda"), None, act)
    (d,) = torch.autograd.grad(y.sum(), leaf)
    return y.detach().cpu(), d.cpu()


@pytest.mark.parametrize("dtype", list(U))
def test_tanh_stays_within_one(dtype):
    """tanh is nowhere above one, so that its slope 1 - tanh^2 is nowhere negative; from |z| = 20 on it is one."""
    z = torch.cat([_line(dtype, 25.0), _line(dtype, 1e4), torch.tensor([[20.0], [-20.0], [3e30], [-3e30], [INF], [-INF]], dtype=dtype)])
    y, d = _run(z, "tanh")
    assert torch.all(y.abs() <= 1) and torch.all(d >= 0) and torch.all(d <= 1)
    far = z.abs() >= 20
    assert torch.equal(y[far], z[far].sign()) and not d[far].any()
    assert _run(torch.full((1, 1), float("nan"), dtype=dtype), "tanh")[0].isnan().all()


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_sigmoid_and_silu_keep_their_digits(act, dtype):
    """Relative accuracy over the whole line, into the subnormal numbers.  With e = exp(-|z|) within 5 u in FP32 (its exponential 2 units of the last place, 4 u, and a
    rounding; FP64: a reduced argument, a polynomial and their roundings, below that too), 1 / (1 + e) is within 2.5 u for e, u for the sum and 2 u for the reciprocal, e / (1 + e) within
    5 + 1 + 2 + 1 = 9 u, times z 10 u; sigmoid's slope e / (1 + e)^2 within 9 + 5.5 + 1 u, SiLU's terms s and z s (1 - s) within 9 and 9 + 5.5 + 4.  Results below the smallest
    normal number are off by steps of the smallest number there is, times what multiplies them."""
    u, tiny, least = U[dtype], torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    z = torch.cat([_line(dtype, 95.0 if dtype == torch.float32 else 740.0), _line(dtype, 10.0)])
    y, d = _run(z, act)
    x = z.flatten().numpy().astype(np.longdouble)
    s, rest = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
    ref, slope, terms = (s, s * rest, s * rest) if act == "sigmoid" else (x * s, s * (1 + x * rest), s + np.abs(x) * s * rest)
    off, may = np.abs(y.flatten().numpy().astype(np.longdouble) - ref), (9 if act == "sigmoid" else 10) * u * np.abs(ref) + 2 * least * (1 + np.abs(x))
    assert np.all(off <= may), (float(np.max(off / (np.abs(ref) + tiny))) / u, float(x[np.argmax(off - may)]))
    off, may = np.abs(d.flatten().numpy().astype(np.longdouble) - slope), 20 * u * terms + 2 * least * (1 + np.abs(x))
    assert np.all(off <= may), (float(np.max(off / (terms + tiny))) / u, float(x[np.argmax(off - may)]))
    assert torch.all(y[z < -1] < 0 if act == "silu" else y[z > -80] > 0) and torch.all(y[z == 0] == (0.5 if act == "sigmoid" else 0))


@pytest.mark.parametrize("act", ["silu", "sigmoid", "tanh"])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("M,K,N", [(300, 64, 96), (200, 33, 50), (150, 600, 40)])
def test_large_arguments_beside_small_ones(M, K, N, residual, act):
    """Rows whose arguments reach some hundreds between rows whose arguments are of order one: values and gradients, and the small rows' bits do not change."""
    x, w, b, r, g = single._inputs(M, K, N, torch.float32, residual=residual, seed=11)
    clean = single.run(x, w, b, r, g, act)
    large = [3, 40, M // 2, M - 1]
    x[large] *= 200
    got = single.run(x, w, b, r, g, act)
    want = single.reference(x, w, b, r, g, act, U[torch.float32])
    assert float((x.double() @ w.double().t()).abs().max()) > 300
    single.check(got, want)
    others = [i for i in range(M) if i not in large]
    assert torch.equal(got["y"][others], clean["y"][others]) and torch.equal(got["x"][others], clean["x"][others])
