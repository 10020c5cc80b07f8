"""Activations of the dense layers, through a layer of one channel and weight one, where their argument is exact."""
import numpy as np
import pytest
import torch

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
