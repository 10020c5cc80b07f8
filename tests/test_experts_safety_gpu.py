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


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused_whatever_the_grad_mode(grad):
    """Forward-mode differentiation is not offered; no_grad does not switch it off, so a tangent is refused there too, of whichever operand."""
    import torch.autograd.forward_ad as forward_ad
    from fasteq_b200.ops.dense_act import dense_act
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    z = lambda *s: torch.ones(*s, device="cuda")
    plan = expert_plan(torch.tensor([[0, 1], [1, 0], [0, 0]], device="cuda"), 2)
    calls = [(lambda x, w, b, r: dense_act(x, w, b, "silu", r), (z(3, 4), z(5, 4), z(5), z(3, 5))), (lambda x: expert_gather(x, plan), (z(3, 4),)),
             (lambda rows, weight: expert_combine(rows, plan, weight), (z(6, 4), z(3, 2))),
             (lambda rows, w, b: expert_dense(rows, w, plan, b, "tanh"), (z(6, 4), z(2, 5, 4), z(2, 5)))]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for f, args in calls:
            for i in range(len(args)):
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError):
                    f(*dual)
            f(*args)


def test_tangents_of_cotangents_are_refused():
    """The gradients are linear in the cotangent: its tangent would have to come out as theirs."""
    import torch.autograd.forward_ad as forward_ad
    from fasteq_b200.ops.dense_act import dense_act
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    leaf = lambda *s: torch.ones(*s, device="cuda", requires_grad=True)
    plan = expert_plan(torch.tensor([[0, 1], [1, 0], [0, 0]], device="cuda"), 2)
    x, rows, w, weight = leaf(3, 4), leaf(6, 4), leaf(2, 5, 4), leaf(3, 2)
    outputs = [(dense_act(x, w[0], None, "silu"), x), (expert_gather(x, plan), x), (expert_combine(rows, plan, weight), weight), (expert_combine(rows, plan), rows),
               (expert_dense(rows, w, plan), rows)]
    with forward_ad.dual_level():
        for y, to in outputs:
            g = torch.ones_like(y)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(y, to, forward_ad.make_dual(g, g.clone()), retain_graph=True)
            torch.autograd.grad(y, to, g)


def test_plans_of_several_threads():
    """Threads that plan for different numbers of experts through the C interface, which takes no lock of Python's: no call takes shared memory from another's launch."""
    lib = cabi._core()
    threads, bad = [], []
    start = threading.Barrier(4)

    def work(i):
        experts, n = (1024, 400, 800, 600)[i], 200 + i
        g = torch.Generator().manual_seed(i)
        e = torch.randint(0, experts, (n,), generator=g, dtype=torch.int32)
        position, offsets = experts_tests._order(e.view(-1, 1), experts)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            ed, pd = e.cuda(), torch.empty(n, dtype=torch.int32, device="cuda")
            od = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
        args = (_ptr(ed), C.c_int32(4), C.c_int64(n), C.c_int32(experts), _ptr(pd), _ptr(od), None, C.c_void_p(stream.cuda_stream))
        start.wait()
        for _ in range(3000):
            rc = lib.fasteq_expert_plan(*args)
            if rc != 0:
                bad.append((experts, rc))
        stream.synchronize()
        if not (torch.equal(pd.cpu().long(), position.flatten()) and torch.equal(od.cpu().long(), offsets)):
            bad.append((experts, "order"))
    torch.cuda.synchronize()
    for i in range(4):
        threads.append(threading.Thread(target=work, args=(i,)))
        threads[-1].start()
    for t in threads:
        t.join()
    assert not bad, (len(bad), bad[:5])


def test_first_calls_of_several_threads():
    """A fresh process whose first dense layers come from eight threads at once: what a call needs to know of the device is asked for once, and every result is right."""
    import os
    import subprocess
    import sys
    code = """
import threading, torch
from fasteq_b200.ops.dense_act import dense_act
x, w = torch.arange(64 * 48, device="cuda").remainder(7).float().view(64, 48), torch.arange(40 * 48, device="cuda").remainder(5).float().view(40, 48)
torch.cuda.synchronize()
out, start = [None] * 8, threading.Barrier(8)
def work(i):
    start.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        out[i] = dense_act(x, w)
        torch.cuda.current_stream().synchronize()
threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
want = x.cpu().double() @ w.cpu().double().t()
assert all(o is not None and torch.equal(o.cpu().double(), want) for o in out)
print("right")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=150, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "right" in r.stdout, r.stderr[-2000:]


def test_a_plan_changed_in_place_is_refused():
    """By every call, and by the gradients of calls made before the change; in inference mode too, and resized or exchanged storage as well."""
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    e = torch.tensor([[0, 1], [1, 0], [2, -1]], device="cuda")
    z = lambda *s: torch.randn(*s, device="cuda", requires_grad=True)
    x, rows, w, weight = z(3, 4), z(6, 4), z(3, 5, 4), z(3, 2)
    calls = [lambda p: expert_gather(x, p), lambda p: expert_combine(rows, p, weight), lambda p: expert_combine(rows, p), lambda p: expert_dense(rows, w, p, None, "silu")]
    for change in (lambda p: p.position.add_(1), lambda p: p.offsets.zero_(), lambda p: p.position[0].fill_(2 ** 30)):
        for inference in (False, True):
            with torch.inference_mode(inference):
                plan = expert_plan(e, 3)
                before = [f(plan) for f in calls]
                change(plan)
                for f in calls:
                    with pytest.raises(RuntimeError, match="changed in place"):
                        f(plan)
            for y, f in zip(before, calls) if not inference else ():
                leaves = [t for t in (x, rows, w, weight) if any(n is t for n in _leaves(y))]
                if f is calls[3] and torch.equal(plan.offsets.cpu(), torch.tensor([0, 2, 4, 5], dtype=torch.int32)):
                    continue                                            # its gradients need the offsets alone
                with pytest.raises(RuntimeError, match="changed in place|modified by an inplace operation"):
                    torch.autograd.grad(y, leaves, torch.ones_like(y))
    for change in (lambda p: p.position.set_(), lambda p: p.offsets.set_()):
        plan = expert_plan(e, 3)
        change(plan)
        for f in calls:
            with pytest.raises(RuntimeError, match="changed in place"):
                f(plan)


def _leaves(y):
    out, todo = [], [y.grad_fn]
    while todo:
        for f, _ in todo.pop().next_functions:
            if f is not None:
                todo.append(f)
                if hasattr(f, "variable"):
                    out.append(f.variable)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("width", [5, 64])
def test_positions_out_of_range_are_reported_and_left_alone(width, dtype):
    """Through the C interface, where positions are the caller's memory: nothing is read or written at them, the other entries are as ever."""
    from fasteq_b200.ops.experts import expert_device_status
    lib = cabi._core()
    tokens, slots, experts = 50, 2, 4
    e = experts_tests._experts(tokens, slots, experts, 0.1)
    position, offsets = experts_tests._order(e, experts)
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(width), dtype=torch.float64).to(dtype)
    bad = {(3, 0): -1, (10, 1): tokens * slots, (20, 0): 2 ** 31 - 1, (21, 1): -2 ** 31, (49, 1): tokens * slots + 7}
    wrong = position.clone()
    for at, p in bad.items():
        wrong[at] = p
    x, rows, weight, g = r(tokens, width), r(tokens * slots, width), r(tokens, slots), r(tokens, width)
    xd, rd, wd, gd, pd, od = (t.cuda() for t in (x, rows, weight, g, wrong.int(), offsets.int()))
    nan = lambda *s: torch.full(s, float("nan"), dtype=dtype, device="cuda")
    there, y, gr, gw = nan(tokens * slots, width), nan(tokens, width), nan(tokens * slots, width), nan(tokens, slots)
    dt, sizes = C.c_int32(0 if dtype == torch.float32 else 1), (C.c_int32(experts), C.c_int64(tokens), C.c_int32(slots), C.c_int32(width))
    assert expert_device_status() == 0
    for call in (lambda: lib.fasteq_expert_gather(dt, _ptr(xd), _ptr(pd), _ptr(od), *sizes, _ptr(there), _stream()),
                 lambda: lib.fasteq_expert_combine(dt, _ptr(rd), _ptr(wd), _ptr(pd), _ptr(od), *sizes, _ptr(y), _stream()),
                 lambda: lib.fasteq_expert_combine_backward(dt, _ptr(rd), _ptr(wd), _ptr(gd), _ptr(pd), _ptr(od), *sizes, _ptr(gr), _ptr(gw), _stream())):
        assert call() == 0
        torch.cuda.synchronize()
        assert expert_device_status() == 2 and expert_device_status() == 0
    left_out = torch.zeros(tokens, slots, dtype=torch.bool)
    for at in bad:
        left_out[at] = True
    live = ((e >= 0) & ~left_out).double()
    untouched = position[left_out]
    for t in (there, gr):
        assert t[untouched.cuda()].isnan().all() and t.isnan().any(1).sum() == len(bad)
    u, terms = single.U[dtype], (weight.double() * live)[:, :, None] * rows.double()[position]
    assert torch.all((y.cpu().double() - terms.sum(1)).abs() <= 3 * u * terms.abs().sum(1))
    prod = rows.double()[position] * g.double()[:, None] * live[:, :, None]
    assert torch.all((gw.cpu().double() - prod.sum(2)).abs() <= (width + 8) * u * prod.abs().sum(2))
    keep = (e >= 0) & ~left_out
    assert torch.equal(there.cpu()[position[keep]], x[:, None].expand(-1, slots, -1)[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("offsets", [[0, 300, 2 ** 30, 2 ** 31 - 1], [-5, 300, 700, 700], [0, 700, 300, 700], [700, 300, 100, 0], [500, -2 ** 31, 900, 20]])
def test_offsets_of_no_plan_stay_within_the_rows(offsets, shift, dtype):
    """Through the C interface, where offsets are the caller's memory: nothing is written beside the results, and offsets beyond the rows end with them."""
    lib = cabi._core()
    X, M, K, N, pad = 3, 700, 40, 72, 64
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(M), dtype=torch.float64).to(dtype)
    x, w, b, g = r(M, K), r(X, N, K) / K ** 0.5, r(X, N), r(M, N)
    p = cabi.Problem(dtype=0 if dtype == torch.float32 else 1, k=K, n=N, experts=X, inner=1, act=2, rows=M)
    bases = []

    def put(t):                          # between guards, `shift` values off alignment
        base = torch.full((t.numel() + 2 * pad + 8,), 77.0, dtype=dtype, device="cuda")
        v = base[pad + shift:pad + shift + t.numel()].view(t.shape)
        v.copy_(t)
        bases.append((base, v))
        return v
    xd, wd, bd, gd = (put(t) for t in (x, w, b, g))
    y, gx, gw, gb = (put(torch.zeros_like(t)) for t in (g, x, w, b))
    slope = torch.zeros(M + pad, N, dtype=dtype, device="cuda")
    od = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    scratch = []
    for backward in (0, 1):
        need = C.c_int64(0)
        assert lib.fasteq_product_scratch(C.byref(p), C.c_int32(backward), C.byref(need)) == 0
        scratch.append((torch.full((need.value + 256,), 77, dtype=torch.uint8, device="cuda"), need))
    assert lib.fasteq_product_forward(C.byref(p), _ptr(xd), _ptr(wd), _ptr(bd), None, _ptr(od), _ptr(y), _ptr(slope), _ptr(scratch[0][0]), scratch[0][1], _stream()) == 0
    assert lib.fasteq_product_backward(C.byref(p), _ptr(xd), _ptr(wd), _ptr(gd), _ptr(slope), _ptr(od), _ptr(gx), _ptr(gw), _ptr(gb), _ptr(scratch[1][0]), scratch[1][1],
                                       _stream()) == 0
    torch.cuda.synchronize()
    for base, v in bases:
        assert torch.all(base[:pad + shift] == 77.0) and torch.all(base[pad + shift + v.numel():] == 77.0)
    for buffer, need in scratch:
        assert torch.all(buffer[need.value:] == 77)
    assert not slope[M:].any()
    ends = [min(max(o, 0), M) for o in offsets]
    if ends == sorted(ends) and ends[0] == 0:
        want = experts_tests._dense_reference(x, w, b, ends, "tanh", g, single.U[dtype])
        for n, v in (("y", y), ("x", gx), ("w", gw), ("b", gb)):
            ref, tol = want[n]
            assert torch.all((v.cpu().double() - ref).abs() <= tol), n


def test_status_words_wait_for_every_stream():
    """A plan on a side stream, behind work that takes a while: its report is read, not overlooked, by either way of reading it."""
    from fasteq_b200.ops.experts import expert_device_status, expert_plan
    from fasteq_b200.status import device_status
    side, e = torch.cuda.Stream(), torch.tensor([0, 7, 1], device="cuda")
    torch.cuda.synchronize()
    for read, want, nothing in ((expert_device_status, 2, 0), (device_status, {"experts": 2}, {})):
        assert read() == nothing
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)
            expert_plan(e, 3)
        assert read() == want
        assert read() == nothing


def test_the_widest_layers_and_one_channel_more():
    """4,194,240 channels are the most: with all gradients; one more is refused by name before anything runs."""
    from fasteq_b200.ops.dense_act import dense_act
    from fasteq_b200.ops.experts import expert_dense, expert_plan
    most = 64 * 65535
    one = torch.zeros(1, 1, device="cuda")
    plan = expert_plan(torch.zeros(1, dtype=torch.int64, device="cuda"), 1)
    for call in (lambda: dense_act(one, one.expand(most + 1, 1)), lambda: dense_act(one.expand(1, most + 1), one.expand(1, most + 1)),
                 lambda: expert_dense(one, one.expand(1, most + 1, 1), plan)):
        with pytest.raises(ValueError, match="channels"):
            call()
    for dtype, K in ((torch.float64, 65), (torch.float32, 9)):
        x, w = torch.randint(-3, 4, (3, K), device="cuda").to(dtype), torch.randint(-3, 4, (most, K), device="cuda").to(dtype)
        g = torch.randint(-3, 4, (3, most), device="cuda").to(dtype)
        x.requires_grad_(True), w.requires_grad_(True)
        y = dense_act(x, w)
        gx, gw = torch.autograd.grad(y, (x, w), g)
        xd, wd, gd = x.detach().double(), w.detach().double(), g.double()
        assert torch.equal(y.detach().double(), xd @ wd.t()) and torch.equal(gw.double(), gd.t() @ xd)
        assert torch.equal(gx.double(), gd @ wd) or dtype == torch.float32       # FP32 sums beyond 2^24 round
        assert float((gx.double() - gd @ wd).abs().max()) <= (most + 8) * 2.0 ** -24 * float((gd.abs() @ wd.abs()).max())
        del x, w, g, y, gx, gw, xd, wd, gd
