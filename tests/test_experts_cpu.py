"""Refusals of the dense layers with an epilogue and of the experts, without a GPU: through Python, and status codes at the C interface."""
import ctypes as C

import pytest
import torch


def test_cpu_tensors_and_unknown_activations_are_refused():
    from fasteq_b200.ops.dense_act import dense_act
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        dense_act(x, w)
    with pytest.raises(ValueError, match="activation"):
        dense_act(x, w, activation="swish")
    with pytest.raises(RuntimeError, match="no CPU path"):
        expert_plan(torch.zeros(4, dtype=torch.int64), 2)
    for call in (lambda: expert_gather(x, None), lambda: expert_combine(x, None), lambda: expert_dense(x, w.unsqueeze(0), None)):
        with pytest.raises(TypeError, match="ExpertPlan"):
            call()


class Problem(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("k", C.c_int32), ("n", C.c_int32), ("experts", C.c_int32), ("inner", C.c_int32), ("act", C.c_int32), ("rows", C.c_int64)]


OK, UNSUPPORTED, INVALID = 0, 1, 2
GOOD = dict(dtype=0, k=8, n=8, experts=1, inner=1, act=1, rows=4)
P, I32, I64 = C.c_void_p, C.c_int32, C.c_int64


def _core():
    from fasteq_b200 import _cabi
    return _cabi.core()


@pytest.mark.parametrize("change,status", [(dict(dtype=2), INVALID), (dict(k=-1), INVALID), (dict(n=-1), INVALID), (dict(rows=-1), INVALID), (dict(act=5), INVALID),
                                           (dict(act=-1), INVALID), (dict(inner=0), INVALID), (dict(experts=0), INVALID), (dict(experts=2), INVALID),
                                           (dict(rows=2 ** 31), UNSUPPORTED), (dict(rows=2 ** 45), UNSUPPORTED), (dict(n=2 ** 30), UNSUPPORTED),
                                           (dict(rows=0), OK), (dict(n=0), OK), ({}, INVALID)])
def test_forward_problems(change, status):
    lib = _core()
    p = Problem(**{**GOOD, **change})
    assert lib.fasteq_product_forward(C.byref(p), None, None, None, None, None, None, None, None, I64(0), None) == status


def test_other_entries_refuse_null_pointers_and_sizes():
    lib = _core()
    p, one = Problem(**GOOD), C.c_int64(0)
    assert lib.fasteq_product_forward(None, None, None, None, None, None, None, None, None, I64(0), None) == INVALID
    none = (None,) * 8
    assert lib.fasteq_product_backward(C.byref(p), *none, None, I64(0), None) == OK              # no gradient is asked for
    some = C.create_string_buffer(64)
    assert lib.fasteq_product_backward(C.byref(p), None, None, None, None, None, some, None, None, None, I64(0), None) == INVALID
    assert lib.fasteq_product_backward(C.byref(p), some, some, some, None, None, None, None, some, None, I64(0), None) == INVALID      # bias without weights
    assert lib.fasteq_product_scratch(C.byref(p), I32(0), None) == INVALID
    for change, backward, there in ((dict(), 0, False), (dict(), 1, False), (dict(k=2048), 0, True), (dict(k=7), 0, True), (dict(n=7), 0, False), (dict(n=7), 1, True),
                                    (dict(rows=100_000), 1, True), (dict(rows=100_000, dtype=1), 0, False), (dict(rows=0, k=7), 1, False)):
        q = Problem(**{**GOOD, **change})
        assert lib.fasteq_product_scratch(C.byref(q), I32(backward), C.byref(one)) == OK and (one.value > 0) == there, change
    long = Problem(**{**GOOD, "k": 2048})
    assert lib.fasteq_product_forward(C.byref(long), some, some, None, None, None, some, None, some, I64(16), None) == INVALID
    buffer = C.create_string_buffer(1 << 20)
    need = C.c_int64(0)
    assert lib.fasteq_product_scratch(C.byref(long), I32(0), C.byref(need)) == OK and need.value + 16 <= len(buffer)
    odd = C.c_void_p(C.addressof(buffer) // 16 * 16 + 20)                                       # scratch that is not 16-byte aligned
    assert lib.fasteq_product_forward(C.byref(long), some, some, None, None, None, some, None, odd, need, None) == INVALID
    many = Problem(**{**GOOD, "experts": 1025})
    assert lib.fasteq_product_scratch(C.byref(many), I32(1), C.byref(one)) == UNSUPPORTED
    assert lib.fasteq_expert_plan_scratch(I64(-1), I32(3), C.byref(one)) == INVALID
    assert lib.fasteq_expert_plan_scratch(I64(5), I32(1025), C.byref(one)) == UNSUPPORTED
    assert lib.fasteq_expert_plan_scratch(I64(2 ** 31), I32(3), C.byref(one)) == UNSUPPORTED
    assert lib.fasteq_expert_plan_scratch(I64(100), I32(3), C.byref(one)) == OK and one.value == 0
    some = C.c_int32(0)
    assert lib.fasteq_expert_plan(None, I32(4), I64(5), I32(3), None, C.byref(some), None, None) == INVALID
    assert lib.fasteq_expert_plan(C.byref(some), I32(2), I64(1), I32(3), C.byref(some), C.byref(some), None, None) == INVALID
    assert lib.fasteq_expert_gather(I32(0), None, None, None, I32(3), I64(4), I32(1), I32(8), None, None) == INVALID
    assert lib.fasteq_expert_gather(I32(0), None, None, None, I32(3), I64(0), I32(1), I32(8), None, None) == OK
    assert lib.fasteq_expert_gather(I32(2), None, None, None, I32(3), I64(0), I32(1), I32(8), None, None) == INVALID
    assert lib.fasteq_expert_combine(I32(0), None, None, None, None, I32(3), I64(4), I32(0), I32(8), None, None) == INVALID
    assert lib.fasteq_expert_combine(I32(1), None, None, None, None, I32(3), I64(4), I32(1), I32(8), None, None) == INVALID
    assert lib.fasteq_expert_combine_backward(I32(0), None, None, None, None, None, I32(3), I64(4), I32(1), I32(8), C.byref(some), None, None) == INVALID
    assert lib.fasteq_expert_combine_backward(I32(0), None, None, None, None, None, I32(3), I64(4), I32(1), I32(8), None, None, None) == OK
    assert lib.fasteq_expert_device_status(None) == INVALID
