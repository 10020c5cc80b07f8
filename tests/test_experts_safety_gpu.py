"""Dense layers with an epilogue and experts: outputs that are not asked for, tangents, plans made by several threads, plans that were changed, status words."""
import ctypes as C
import threading

import pytest
import torch

from tests import test_dense_act_gpu as single
from tests import test_experts_cpu as cabi
from tests import test_experts_gpu as experts_tests

pytestmark = pytest.mark.gpu


def _ptr(t):
    return C.c_void_p(t.data_ptr())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("M,K,N,offset", [(70, 64, 64, 0), (70, 64, 64, 1), (300, 33, 50, 0), (90, 0, 24, 0)])
def test_slopes_of_the_identity_are_not_touched(M, K, N, offset, dtype):
    """Whichever kernel a call takes: aligned, unaligned, without channels to sum over."""
    lib = cabi._core()
    x, w, b, _, _ = single._inputs(M, K, N, dtype, residual=False)
    p = cabi.Problem(dtype=0 if dtype == torch.float32 else 1, k=K, n=N, experts=1, inner=1, act=0, rows=M)
    base = torch.zeros(M * K + 8, dtype=dtype, device="cuda")
    xd = base[offset:offset + M * K].view(M, K)
    xd.copy_(x)
    wd, bd, y = w.cuda(), b.cuda(), torch.empty(M, N, dtype=dtype, device="cuda")
    slope = torch.full((M, (N + 3) // 4 * 4), 77.0, dtype=dtype, device="cuda")
    need = C.c_int64(0)
    assert lib.fasteq_product_scratch(C.byref(p), C.c_int32(0), C.byref(need)) == 0
    scratch = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    assert lib.fasteq_product_forward(C.byref(p), _ptr(xd), _ptr(wd), _ptr(bd), None, None, _ptr(y), _ptr(slope), _ptr(scratch), need, _stream()) == 0
    single.check({"y": y}, single.reference(x, w, b, None, torch.zeros(M, N), None, single.U[dtype]))
    assert torch.all(slope == 77.0)
