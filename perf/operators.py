"""Dense layers with an epilogue, and experts: what is measured of them.

Three kinds of work, as a user of the framework has them next to its message passing:

* ``dense``    one layer ``act(x W^T + b) + residual`` of a node or edge network, alone or with every gradient;
* ``route``    node features brought into the order of the experts (species, say) that the nodes are given to, the experts' outputs
               brought back and added with weights; alone or with every gradient;
* ``experts``  the whole step: the order, the features in it, one product per expert (``mix``: the components of one irrep share their
               expert's matrix) or two with bias and activation (``mlp``), and the weighted way back; alone or with every gradient.

With ``own`` false the passes are elementary torch operations, with ``own`` true calls of the framework.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPE = {"f32": torch.float32, "f64": torch.float64}


def listed():
    return [
        # a residual node update on one periodic cell of 192 atoms, 128 channels: launch latency
        dict(name="dense_one_cell", kind="dense", dtype="f32", rows=192, k=128, n=128, act="silu", bias=True, residual=True, grad=False),
        # a hidden layer of the radial network over the edges of a 64-structure batch: memory traffic
        dict(name="dense_edges", kind="dense", dtype="f32", rows=644_552, k=64, n=64, act="silu", bias=True, residual=False, grad=False),
        # a widening node layer of that batch (12,288 atoms) with every gradient
        dict(name="dense_batch_gradients", kind="dense", dtype="f32", rows=12_288, k=128, n=512, act="silu", bias=True, residual=False, grad=True),
        # odd extents: 33 channels, 80,533 edges, residual, every gradient
        dict(name="dense_odd_gradients", kind="dense", dtype="f32", rows=80_533, k=33, n=99, act="tanh", bias=True, residual=True, grad=True),
        # the wide FP64 model: 12,288 atoms, 256 channels, every gradient
        dict(name="dense_f64_gradients", kind="dense", dtype="f64", rows=12_288, k=256, n=256, act="silu", bias=True, residual=True, grad=True),
        # one cell of 192 atoms, two of eight experts each, a tenth of the nodes given to none (padding): launch latency
        dict(name="route_one_cell", kind="route", dtype="f32", tokens=192, slots=2, experts=8, width=128, unrouted=0.1, grad=False),
        # 128 x (0e + 1o) features of 1024 structures (150,873 atoms), two of 32 experts each, every gradient: memory traffic
        dict(name="route_large_gradients", kind="route", dtype="f32", tokens=150_873, slots=2, experts=32, width=512, unrouted=0.0, grad=True),
        # FP64 features by species (89 of them), one expert a node, every gradient
        dict(name="route_species_f64_gradients", kind="route", dtype="f64", tokens=12_288, slots=1, experts=89, width=1024, unrouted=0.0, grad=True),
        # experts on one cell: latency of the whole step
        dict(name="experts_one_cell", kind="experts", form="mlp", dtype="f32", tokens=192, slots=2, experts=8, rows=1, k=128, hidden=256,
             unrouted=0.0, grad=False),
        # a batch of 12,288 atoms, two of eight experts each, training
        dict(name="experts_batch_gradients", kind="experts", form="mlp", dtype="f32", tokens=12_288, slots=2, experts=8, rows=1, k=128, hidden=256,
             unrouted=0.0, grad=True),
        # a matrix per species (89 of them, few atoms to most) for the four components of 64 x (0e + 1o), an odd number of atoms, some given to none
        dict(name="experts_species_gradients", kind="experts", form="mix", dtype="f32", tokens=20_011, slots=1, experts=89, rows=4, k=64, hidden=64,
             unrouted=0.05, grad=True),
        # FP64 experts of a batch of eight structures
        dict(name="experts_f64_gradients", kind="experts", form="mlp", dtype="f64", tokens=1_536, slots=2, experts=10, rows=1, k=128, hidden=128,
             unrouted=0.0, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _extent(rng, lo, hi):
    """Channel counts: multiples of 32 and of 4 as models have them, and any."""
    v = _log_int(rng, lo, hi)
    step = rng.choice([32, 32, 4, 1])
    return max(lo, v // step * step)


def _seconds(case):
    """A measure of a case's cost, to keep drawn cases below the largest listed one."""
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / (50e12 if case["dtype"] == "f32" else 25e12)


def draw(rng):
    kind = rng.choice(["dense", "dense", "route", "experts", "experts"])
    dtype = "f64" if rng.random() < 0.2 else "f32"
    grad = rng.random() < 0.6
    if kind == "dense":
        case = dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, 644_552), k=_extent(rng, 8, 512), n=_extent(rng, 8, 512),
                    act=rng.choice(["identity", "silu", "silu", "tanh", "sigmoid"]), bias=rng.random() < 0.8, residual=rng.random() < 0.5, grad=grad)
        size = "rows"
    elif kind == "route":
        case = dict(kind=kind, dtype=dtype, tokens=_log_int(rng, 1, 150_873), slots=rng.randint(1, 4), experts=_log_int(rng, 2, 256),
                    width=_extent(rng, 8, 1024), unrouted=rng.choice([0.0, 0.0, 0.2]), grad=grad)
        size = "tokens"
    else:
        form = rng.choice(["mlp", "mlp", "mix"])
        case = dict(kind=kind, form=form, dtype=dtype, tokens=_log_int(rng, 1, 20_011), slots=rng.randint(1, 4), experts=_log_int(rng, 2, 89),
                    rows=rng.choice([1, 3, 4, 9]) if form == "mix" else 1, k=_extent(rng, 16, 256), hidden=_extent(rng, 16, 512),
                    unrouted=rng.choice([0.0, 0.0, 0.2]), grad=grad)
        size = "tokens"
    if "slots" in case:
        case["slots"] = min(case["slots"], case["experts"])
    most = max(_seconds(c) for c in listed() if c["kind"] == kind and c["dtype"] == ("f32" if kind != "dense" else dtype))
    while _seconds(case) > most:
        case[size] = max(1, case[size] * 2 // 3)
        if case[size] == 1:
            break
    return case


# ------------------------------------------------------------------------------------------------ inputs

def _randn(g, dtype, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _choices(case, g):
    """Experts of every node and their weights: the best of random scores, some experts liked better than others; -1: given to none."""
    scores = torch.randn((case["tokens"], case["experts"]), generator=g, device=DEV)
    scores = scores + torch.randn((case["experts"],), generator=g, device=DEV)
    expert = scores.topk(case["slots"], dim=1).indices
    weight = torch.softmax(scores, dim=1).gather(1, expert).to(DTYPE[case["dtype"]])
    if case["unrouted"] > 0:
        expert = expert.masked_fill(torch.rand((case["tokens"], 1), generator=g, device=DEV) < case["unrouted"], -1)
    return expert.to(torch.int32), weight


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, grad = DTYPE[case["dtype"]], case["grad"]
    s = dict(case=dict(case))
    if case["kind"] == "dense":
        M, K, N = case["rows"], case["k"], case["n"]
        s["x"], s["w"] = _randn(g, dt, M, K), _randn(g, dt, N, K) / math.sqrt(K)
        s["b"] = 0.1 * _randn(g, dt, N) if case["bias"] else None
        s["r"] = _randn(g, dt, M, N) if case["residual"] else None
        s["g"] = _randn(g, dt, M, N) if grad else None
        leaves = ("x", "w", "b", "r")
    elif case["kind"] == "route":
        T, S, C = case["tokens"], case["slots"], case["width"]
        s["expert"], s["weight"] = _choices(case, g)
        s["x"], s["y"] = _randn(g, dt, T, C), _randn(g, dt, T * S, C)
        s["g"] = _randn(g, dt, T, C) if grad else None
        s["grows"] = _randn(g, dt, T * S, C) if grad else None
        leaves = ("x", "y", "weight")
    else:
        T, X, I, K, H = case["tokens"], case["experts"], case["rows"], case["k"], case["hidden"]
        s["expert"], s["weight"] = _choices(case, g)
        if case["form"] == "mix":
            s["x"], s["w1"] = _randn(g, dt, T, I, K), _randn(g, dt, X, H, K) / math.sqrt(K)
            s["g"] = _randn(g, dt, T, I, H) if grad else None
            leaves = ("x", "w1", "weight")
        else:
            s["x"], s["w1"], s["b1"] = _randn(g, dt, T, K), _randn(g, dt, X, H, K) / math.sqrt(K), 0.1 * _randn(g, dt, X, H)
            s["w2"], s["b2"] = _randn(g, dt, X, K, H) / math.sqrt(H), 0.1 * _randn(g, dt, X, K)
            s["g"] = _randn(g, dt, T, K) if grad else None
            leaves = ("x", "w1", "b1", "w2", "b2", "weight")
    s["leaves"] = [n for n in leaves if s.get(n) is not None]
    if grad:
        for n in s["leaves"]:
            s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    kind, grad = s["case"]["kind"], s["case"]["grad"]
    if own:
        with torch.set_grad_enabled(grad):
            return _own_dense(s) if kind == "dense" else _own_route(s) if kind == "route" else _own_experts(s)
    with torch.no_grad():
        return _plain_dense(s) if kind == "dense" else _plain_route(s) if kind == "route" else _plain_experts(s)


def _own_dense(s):
    from fasteq_b200.ops.dense_act import dense_act
    out = {"y": dense_act(s["x"], s["w"], bias=s["b"], activation=s["case"]["act"], residual=s["r"])}
    if s["case"]["grad"]:
        grads = torch.autograd.grad(out["y"], [s[n] for n in s["leaves"]], s["g"])
        out.update(zip(("g" + n for n in s["leaves"]), grads))
        out["y"] = out["y"].detach()
    return out


def _own_route(s):
    from fasteq_b200.ops.experts import expert_combine, expert_gather, expert_plan
    plan = expert_plan(s["expert"], s["case"]["experts"])
    rows = expert_gather(s["x"], plan)
    y = expert_combine(s["y"], plan, s["weight"])
    out = dict(offsets=plan.offsets, position=plan.position.reshape(-1), rows=rows.detach(), out=y.detach())
    if s["case"]["grad"]:
        grads = torch.autograd.grad([rows, y], [s[n] for n in s["leaves"]], [s["grows"], s["g"]])
        out.update(zip(("g" + n for n in s["leaves"]), grads))
    return out


def _own_experts(s):
    from fasteq_b200.ops.experts import expert_combine, expert_dense, expert_gather, expert_plan
    plan = expert_plan(s["expert"], s["case"]["experts"])
    rows = expert_gather(s["x"], plan)
    if s["case"]["form"] == "mix":
        rows = expert_dense(rows, s["w1"], plan)
    else:
        rows = expert_dense(rows, s["w1"], plan, bias=s["b1"], activation="silu")
        rows = expert_dense(rows, s["w2"], plan, bias=s["b2"])
    y = expert_combine(rows, plan, s["weight"])
    out = dict(y=y.detach())
    if s["case"]["grad"]:
        grads = torch.autograd.grad(y, [s[n] for n in s["leaves"]], s["g"])
        out.update(zip(("g" + n for n in s["leaves"]), grads))
    return out


def _act(name, z):
    """An activation and its derivative."""
    if name == "silu":
        t = 1 / (1 + torch.exp(-z))
        return z * t, t * (1 + z * (1 - t))
    if name == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if name == "sigmoid":
        t = 1 / (1 + torch.exp(-z))
        return t, t * (1 - t)
    return z, torch.ones_like(z)


def _plain_dense(s):
    z = s["x"] @ s["w"].t()
    if s["b"] is not None:
        z = z + s["b"]
    y, d = _act(s["case"]["act"], z) if s["case"]["act"] != "identity" else (z, None)
    if s["r"] is not None:
        y = y + s["r"]
    out = {"y": y}
    if s["case"]["grad"]:
        gz = s["g"] if d is None else s["g"] * d
        out["gx"], out["gw"] = gz @ s["w"], gz.t() @ s["x"]
        if s["b"] is not None:
            out["gb"] = gz.sum(dim=0)
        if s["r"] is not None:
            out["gr"] = s["g"]
    return out


def _sorted(expert, experts):
    """Stable order of the (node, slot) pairs by expert, those of none last: (expert of each pair, order, position, offsets)."""
    e = expert.reshape(-1).long()
    e = torch.where(e < 0, experts, e)
    order = torch.argsort(e, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(e.numel(), device=e.device)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=e.device)
    offsets[1:] = torch.bincount(e, minlength=experts + 1)[:experts].cumsum(0)
    return e, order, position, offsets


def _there(x, order, e, experts, slots):
    """Rows of the nodes in the experts' order, zero for pairs of no expert."""
    return x[order // slots] * (e[order] < experts).view(-1, *[1] * (x.dim() - 1)).to(x.dtype)


def _back(rows, position, e, experts, slots, weight=None):
    keep = (e < experts).view(-1, slots)
    weight = keep.to(rows.dtype) if weight is None else torch.where(keep, weight, 0.0)
    v = rows[position].view(-1, slots, *rows.shape[1:])
    return (v * weight.view(*weight.shape, *[1] * (rows.dim() - 1))).sum(dim=1)


def _back_gradients(rows, g, order, position, e, experts, slots, weight):
    """Gradients of the weighted way back: of the rows and of the weights."""
    keep = (e < experts).view(-1, slots)
    grows = _there(g, order, e, experts, slots) * weight.reshape(-1)[order].view(-1, *[1] * (g.dim() - 1))
    prod = rows[position].view(-1, slots, *rows.shape[1:]) * g.unsqueeze(1)
    return grows, torch.where(keep, prod.flatten(2).sum(dim=2), 0.0)


def _plain_route(s):
    X, S = s["case"]["experts"], s["case"]["slots"]
    e, order, position, offsets = _sorted(s["expert"], X)
    out = dict(offsets=offsets.to(torch.int32), position=position.to(torch.int32))
    out["rows"] = _there(s["x"], order, e, X, S)
    out["out"] = _back(s["y"], position, e, X, S, s["weight"])
    if s["case"]["grad"]:
        out["gx"] = _back(s["grows"], position, e, X, S)
        out["gy"], out["gweight"] = _back_gradients(s["y"], s["g"], order, position, e, X, S, s["weight"])
    return out


def _plain_experts(s):
    """Products of all experts as one batched product over rows padded to the longest expert."""
    X, S = s["case"]["experts"], s["case"]["slots"]
    e, order, position, offsets = _sorted(s["expert"], X)
    counts = offsets[1:] - offsets[:-1]
    longest, routed = max(1, int(counts.max())), int(offsets[-1])
    es = e[order[:routed]]
    slot = es * longest + torch.arange(routed, device=e.device) - offsets[es]

    def pad(rows):                       # [R, ..., C] -> [experts, longest * ..., C]
        buf = rows.new_zeros((X * longest, *rows.shape[1:]))
        buf[slot] = rows[:routed]
        return buf.view(X, -1, rows.shape[-1])

    def unpad(buf, rows):                # and back, zero rows for pairs of no expert
        out = rows.new_zeros((*rows.shape[:-1], buf.shape[-1]))
        out[:routed] = buf.view(X * longest, *rows.shape[1:-1], buf.shape[-1])[slot]
        return out

    rows = _there(s["x"], order, e, X, S)
    p0 = pad(rows)
    p1 = torch.bmm(p0, s["w1"].transpose(1, 2))
    if s["case"]["form"] == "mix":
        last = unpad(p1, rows)
    else:
        h, d = _act("silu", p1 + s["b1"].unsqueeze(1))
        last = unpad(torch.bmm(h, s["w2"].transpose(1, 2)) + s["b2"].unsqueeze(1), rows)
    out = dict(y=_back(last, position, e, X, S, s["weight"]))
    if s["case"]["grad"]:
        glast, out["gweight"] = _back_gradients(last, s["g"], order, position, e, X, S, s["weight"])
        gp = pad(glast)
        if s["case"]["form"] == "mlp":
            out["gw2"], out["gb2"] = torch.bmm(gp.transpose(1, 2), h), gp.sum(dim=1)
            gp = torch.bmm(gp, s["w2"]) * d
            out["gb1"] = gp.sum(dim=1)
        out["gw1"] = torch.bmm(gp.transpose(1, 2), p0)
        out["gx"] = _back(unpad(torch.bmm(gp, s["w1"]), rows), position, e, X, S)
    return out


# ------------------------------------------------------------------------------------------------ definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    v = {n: s[n].detach().double().requires_grad_(True) for n in s["leaves"]}
    cot = {n: s[n].double() for n in ("g", "grows") if s.get(n) is not None}
    f = {"identity": lambda z: z, "silu": torch.nn.functional.silu, "tanh": torch.tanh, "sigmoid": torch.sigmoid}
    with torch.enable_grad():
        if case["kind"] == "dense":
            z = torch.einsum("mk,nk->mn", v["x"], v["w"])
            z = z + v["b"] if "b" in v else z
            y = f[case["act"]](z)
            y = y + v["r"] if "r" in v else y
            out, ys, gs = {"y": y.detach()}, [y], [cot.get("g")]
        elif case["kind"] == "route":
            pairs = [(x, t, j) for t, row in enumerate(s["expert"].tolist()) for j, x in enumerate(row)]
            ordered = sorted(range(len(pairs)), key=lambda i: (pairs[i][0] if pairs[i][0] >= 0 else case["experts"], i))
            token = torch.tensor([pairs[i][1] for i in ordered], device=DEV)
            slot = torch.tensor([pairs[i][2] for i in ordered], device=DEV)
            live = torch.tensor([float(pairs[i][0] >= 0) for i in ordered], device=DEV, dtype=torch.float64).unsqueeze(1)
            rows = v["x"].index_select(0, token) * live
            y = torch.zeros_like(s["x"], dtype=torch.float64).index_add(0, token, v["y"] * live * v["weight"][token, slot].unsqueeze(1))
            out = dict(offsets=None, position=None, rows=rows.detach(), out=y.detach())
            ys, gs = [rows, y], [cot.get("grows"), cot.get("g")]
        else:
            shape = (*s["x"].shape[:-1], case["hidden"] if case["form"] == "mix" else case["k"])
            y = torch.zeros(shape, dtype=torch.float64, device=DEV)
            for x in range(case["experts"]):
                token, slot = (s["expert"] == x).nonzero(as_tuple=True)
                h = v["x"][token] @ v["w1"][x].t()
                if case["form"] == "mlp":
                    h = torch.nn.functional.silu(h + v["b1"][x]) @ v["w2"][x].t() + v["b2"][x]
                y = y.index_add(0, token, h * v["weight"][token, slot].view(-1, *[1] * (h.dim() - 1)))
            out, ys, gs = {"y": y.detach()}, [y], [cot.get("g")]
        if case["grad"]:
            grads = torch.autograd.grad(ys, [v[n] for n in s["leaves"]], gs)
            out.update(zip(("g" + n for n in s["leaves"]), grads))
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size, grad = 4 if case["dtype"] == "f32" else 8, case["grad"]
    if case["kind"] == "dense":
        M, K, N = case["rows"], case["k"], case["n"]
        small = N * K + (N if case["bias"] else 0)
        values = M * K + small + M * N * (2 if case["residual"] else 1)
        flops = 2 * M * K * N
        if grad:
            values += M * N + M * K + small                       # the gradient that comes in; those of x, W and b
            flops *= 3
        return dict(bytes=size * values, flops=flops)
    T, S, X = case["tokens"], case["slots"], case["experts"]
    pairs, routed = T * S, T * S * (1 - case["unrouted"])
    if case["kind"] == "route":
        C = case["width"]
        values = T * C + pairs * C + pairs * C + T * C + pairs    # x, rows, y, out, weights
        flops = 2 * pairs * C
        if grad:
            values += pairs * C + T * C + T * C + pairs * C + pairs      # gradients of rows and out; of x, y and the weights
            flops += 4 * pairs * C
        return dict(bytes=size * values + 4 * (2 * pairs + X + 1), flops=flops)
    I, K, H = case["rows"], case["k"], case["hidden"]
    mlp = case["form"] == "mlp"
    weights = X * (H * K * 2 + H + K) if mlp else X * H * K
    values = T * I * K + weights + T * I * (K if mlp else H) + pairs
    flops = 2 * routed * I * K * H * (2 if mlp else 1)
    if grad:
        values += T * I * (K if mlp else H) + T * I * K + weights + pairs
        flops *= 3
    return dict(bytes=size * values + 4 * pairs, flops=flops)
