"""Workloads of the routed-row operators: tokens sorted by expert, rows brought back to
their tokens, and the experts' linear layers between the two.

Every case is one pass of one operator, as a training step or a serving step calls it:

* ``sort``: ``sort_tokens`` -- the dispatch plan of the routing indices and the tokens'
  rows in expert order, with the gate weights applied where ``weights`` is true; with
  ``grad`` also the gradients of x (and of the weights);
* ``unsort``: ``unsort_tokens`` -- the expert rows summed per token with the gate weights,
  plus a residual; with ``grad`` also the gradients of rows, weights and residual;
* ``linear``: ``grouped_linear`` -- activation(A W_g^T + bias_g) + residual for the rows of
  every expert g; with ``grad`` also the gradients of A, W, bias and residual.

``own`` False computes the plain forms with elementary torch operations in fp32 (one
rounding at the end); ``own`` True calls the framework.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step, two of eight experts: latency of plan + row copy
        dict(name="sort_one_token", op="sort", T=1, d=4096, E=8, k=2, dtype="bf16", weights=False, capacity=0,
             align=1, pad=0, grad=False),
        # the routed rows of a 16384-token training step, and their gradient back to x
        dict(name="sort_train", op="sort", T=16384, d=4096, E=8, k=2, dtype="bf16", weights=False, capacity=0,
             align=1, pad=0, grad=True),
        # fine-grained experts (128 of them, top-8), weights applied before the experts
        dict(name="sort_fine_weighted", op="sort", T=32768, d=2048, E=128, k=8, dtype="fp16", weights=True,
             capacity=0, align=1, pad=0, grad=True),
        # odd row length, padded tokens without an expert, capacity cut, groups rounded up
        dict(name="sort_ragged", op="sort", T=1537, d=1027, E=13, k=3, dtype="fp32", weights=True, capacity=300,
             align=8, pad=101, grad=True),
        # eight tokens of a decode step: back to token order on top of the residual stream
        dict(name="unsort_decode", op="unsort", T=8, d=4096, E=8, k=2, dtype="bf16", weights=True, capacity=0,
             align=1, pad=0, residual=True, grad=False),
        # the same 16384-token training step on the way back, with its gradients
        dict(name="unsort_train", op="unsort", T=16384, d=4096, E=8, k=2, dtype="bf16", weights=True, capacity=0,
             align=1, pad=0, residual=True, grad=True),
        # top-8 of 128 experts with a capacity of 1.25 times the mean load
        dict(name="unsort_fine_capacity", op="unsort", T=32768, d=2048, E=128, k=8, dtype="fp16", weights=True,
             capacity=2560, align=1, pad=0, residual=False, grad=True),
        # odd row length, unweighted sum (weights were applied before the experts)
        dict(name="unsort_ragged", op="unsort", T=1537, d=1027, E=13, k=3, dtype="fp32", weights=False, capacity=300,
             align=8, pad=101, residual=True, grad=True),
        # one decode token: two rows against two of eight experts, bound by the weights
        dict(name="linear_one_token", op="linear", R=2, G=8, K=4096, N=14336, dtype="bf16", act="gelu", bias=True,
             residual=False, skew=0.0, tail=0, grad=False),
        # a decode batch of 128 tokens through the experts' second layer
        dict(name="linear_decode_batch", op="linear", R=256, G=8, K=14336, N=4096, dtype="bf16", act="none", bias=True,
             residual=True, skew=0.3, tail=0, grad=False),
        # an 8192-token training step of GELU experts with biases, forward and backward
        dict(name="linear_train", op="linear", R=16384, G=8, K=4096, N=14336, dtype="bf16", act="gelu", bias=True,
             residual=False, skew=0.3, tail=0, grad=True),
        # many small experts, odd sizes, empty groups, rows behind the last group
        dict(name="linear_ragged", op="linear", R=5003, G=64, K=1000, N=520, dtype="fp16", act="silu", bias=True,
             residual=True, skew=1.0, tail=37, grad=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("sort", "unsort", "linear"))
    if op == "linear":
        while True:
            c = dict(op=op, R=_log_int(rng, 1, 32768), G=_log_int(rng, 1, 128), K=8 * _log_int(rng, 8, 1792),
                     N=8 * _log_int(rng, 8, 1792), dtype=rng.choice(("bf16", "fp16")), act=rng.choice(ACTIVATIONS),
                     bias=rng.random() < 0.75, residual=rng.random() < 0.5, skew=rng.choice((0.0, 0.3, 1.0)),
                     tail=rng.choice((0, 0, 1, 77)), grad=rng.random() < 0.5)
            if c["G"] * c["N"] * c["K"] <= 8 * 14336 * 4096 and c["R"] * c["N"] * c["K"] <= 16384 * 14336 * 4096:
                return c
    while True:
        E = _log_int(rng, 1, 128)
        c = dict(op=op, T=_log_int(rng, 1, 32768), d=_log_int(rng, 64, 8192), E=E, k=rng.randint(1, min(8, E)),
                 dtype=rng.choice(("bf16", "fp16", "fp32")), weights=rng.random() < 0.6, capacity=0,
                 align=rng.choice((1, 1, 8, 64)), pad=0, grad=rng.random() < 0.6)
        if rng.random() < 0.7:
            c["d"] = 8 * max(1, c["d"] // 8)
        if rng.random() < 0.4:
            c["capacity"] = max(1, int(rng.uniform(0.7, 1.5) * c["T"] * c["k"] / E))
        if rng.random() < 0.4:
            c["pad"] = rng.randint(0, c["T"] // 3)
        if op == "unsort":
            c["residual"] = rng.random() < 0.5
        size = 4 if c["dtype"] == "fp32" else 2
        if c["T"] * c["k"] * c["d"] * size <= 32768 * 8 * 2048 * 2 and E * c["align"] * c["d"] * size <= 1 << 28:
            return c


def work(case):
    c = case
    es = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "linear":
        R, G, K, N = c["R"], c["G"], c["K"], c["N"]
        weights = min(G, R) * N * K * es
        nbytes = R * K * es + weights + (R + c["tail"]) * N * es
        nbytes += min(G, R) * N * es if c["bias"] else 0
        nbytes += R * N * es if c["residual"] else 0
        flops = 2.0 * R * N * K
        if c["grad"]:   # dA and dW; dout and A read, the gradients written
            flops *= 3
            nbytes += (R + c["tail"]) * (N + K) * es + G * N * K * es + weights + R * K * es
            nbytes += G * N * es if c["bias"] else 0
        return {"bytes": nbytes, "flops": flops}
    slots = c["T"] * c["k"]
    kept = (c["T"] - c["pad"]) * c["k"]
    if c["capacity"]:
        kept = min(kept, c["capacity"] * c["E"])
    cap = _rows_cap(c["T"], c["k"], c["E"], c["capacity"], c["align"])
    row = c["d"] * es
    wb = 4 * slots if c["weights"] else 0
    if c["op"] == "sort":
        nbytes = 4 * slots + c["T"] * row + wb + cap * row + 4 * slots + 8 * c["E"]
        flops = kept * c["d"] if c["weights"] else 0
        if c["grad"]:
            nbytes += kept * row + c["T"] * row + wb
            flops += kept * c["d"]
            if c["weights"]:
                nbytes += c["T"] * row + wb
                flops += 3 * kept * c["d"]
    else:
        res = c["T"] * row if c["residual"] else 0
        nbytes = 4 * slots + wb + kept * row + res + c["T"] * row
        flops = 2 * kept * c["d"]
        if c["grad"]:
            nbytes += c["T"] * row + wb + cap * row + 4 * slots
            flops += kept * c["d"]
            if c["weights"]:
                nbytes += kept * row + wb
                flops += 2 * kept * c["d"]
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------ inputs
def _rows_cap(T, k, E, capacity, align):
    kept = min(T * k, capacity * E) if capacity else T * k
    return kept + E * (align - 1)


def _group_sizes(case, seed):
    """Rows of each group: G - 1 sorted cuts of a skewed split of R (empty groups occur)."""
    rng = random.Random(seed * 1000003 + case["R"])
    p = [math.exp(case["skew"] * rng.gauss(0, 1)) for _ in range(case["G"])]
    total, run, cuts = sum(p), 0.0, [0]
    if case["R"] < 4 * case["G"]:   # a few rows on random groups
        n = [0] * case["G"]
        for g in rng.choices(range(case["G"]), weights=p, k=case["R"]):
            n[g] += 1
        return n
    for q in p:
        run += q
        cuts.append(round(case["R"] * run / total))
    return [b - a for a, b in zip(cuts[:-1], cuts[1:])]


def _linear_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    R, G, K, N = case["R"] + case["tail"], case["G"], case["K"], case["N"]

    def normal(shape, std):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dt)

    sizes = _group_sizes(case, seed)
    s = dict(case=case, a=normal((R, K), 1.0), w=torch.empty((G, N, K), device="cuda", dtype=dt))
    for i in range(G):
        s["w"][i] = normal((N, K), K ** -0.5)
    s["bias"] = normal((G, N), 0.5) if case["bias"] else None
    s["residual"] = normal((R, N), 1.0) if case["residual"] else None
    s["dout"] = normal((R, N), 1.0) if case["grad"] else None
    offs = [0]
    for n in sizes:
        offs.append(offs[-1] + n)
    s["offsets"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
    s["most"] = max(sizes)
    return s


def _routing(case, g):
    T, E, k = case["T"], case["E"], case["k"]
    logits = torch.randn((T, E), generator=g, device="cuda") + 0.5 * torch.randn((E,), generator=g, device="cuda")
    v, idx = torch.topk(logits, k, dim=1)
    idx = idx.to(torch.int32)
    if case["pad"]:
        idx[T - case["pad"]:] = -1
    return idx.contiguous(), torch.softmax(v, 1).contiguous()


def _row_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    T, d = case["T"], case["d"]

    def normal(rows):
        return torch.randn((rows, d), generator=g, device="cuda", dtype=torch.float32).to(dt)

    idx, w = _routing(case, g)
    cap = _rows_cap(T, case["k"], case["E"], case["capacity"], case["align"])
    s = dict(case=case, idx=idx, w=w if case["weights"] else None, cap=cap)
    if case["op"] == "sort":
        s["x"] = normal(T)
        s["drows"] = normal(max(cap, 1)) if case["grad"] else None
    else:
        s["rows"] = normal(max(cap, 1))
        s["residual"] = normal(T) if case["residual"] else None
        s["dout"] = normal(T) if case["grad"] else None
    return s


def prepare(case, seed):
    if case["op"] == "linear":
        s = _linear_inputs(case, seed)
        leaves = ("a", "w", "bias", "residual")
    else:
        s = _row_inputs(case, seed)
        leaves = ("x", "w") if case["op"] == "sort" else ("rows", "w", "residual")
        if case["op"] == "unsort":   # the plan that sorted the tokens is at hand on the way back
            s["plan"] = _plan(s["idx"], case["E"], case["capacity"], case["align"])
    if case["grad"]:
        for n in leaves:
            if s[n] is not None:
                s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------ plain forms
def _plan(idx, E, capacity, align):
    """Rows of the (token, slot) pairs grouped by expert, in (token, slot) order."""
    T, k = idx.shape
    flat = idx.reshape(-1).long()
    key = torch.where(flat >= 0, flat, E)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=E + 1)[:E]
    kept = counts.clamp(max=capacity) if capacity else counts
    offsets = torch.zeros(E + 1, dtype=torch.int64, device=idx.device)
    offsets[1:] = torch.cumsum((kept + align - 1) // align * align, 0)
    first = torch.zeros(E + 1, dtype=torch.int64, device=idx.device)
    first[1:] = torch.cumsum(counts, 0)
    sk = key[order]
    pos = torch.arange(T * k, device=idx.device) - first[sk]
    live = sk < E
    if capacity:
        live = live & (pos < capacity)
    slot_row = torch.empty_like(flat)
    slot_row[order] = torch.where(live, offsets[sk.clamp(max=E - 1)] + pos, -1)
    cap = max(_rows_cap(T, k, E, capacity, align), 1)
    row_token = torch.full((cap + 1,), -1, dtype=torch.int64, device=idx.device)
    row_token[torch.where(slot_row >= 0, slot_row, cap)] = torch.arange(T * k, device=idx.device) // k
    i32 = torch.int32
    return dict(counts=counts.to(i32), offsets=offsets.to(i32), slot_row=slot_row.to(i32),
                row_token=row_token[:cap].to(i32), rows_cap=_rows_cap(T, k, E, capacity, align), T=T, k=k)


def _spread(x, slot_row, w, k, cap):
    """rows[slot_row[t, j]] = w[t, j] * x[t] in fp32; rows that no slot fills are zero."""
    rows = torch.zeros((cap + 1, x.shape[1]), dtype=torch.float32, device=x.device)
    v = x.float().repeat_interleave(k, 0)
    if w is not None:
        v = v * w.reshape(-1, 1)
    rows[torch.where(slot_row >= 0, slot_row, cap).long()] = v
    return rows[:cap]


def _gathered(rows, slot_row):
    """rows[slot_row] in fp32, zeros for the dropped slots."""
    live = (slot_row >= 0).unsqueeze(1)
    return torch.where(live, rows[slot_row.clamp(min=0).long()].float(), 0.0)


def _plain_sort(s):
    c = s["case"]
    T, k, d, dt = c["T"], c["k"], c["d"], s["x"].dtype
    p = _plan(s["idx"], c["E"], c["capacity"], c["align"])
    cap = max(s["cap"], 1)
    out = dict(rows=_spread(s["x"], p["slot_row"], s["w"], k, cap).to(dt), offsets=p["offsets"], counts=p["counts"],
               slot_row=p["slot_row"])
    if c["grad"]:
        g = _gathered(s["drows"], p["slot_row"]).view(T, k, d)
        if s["w"] is not None:
            out["dw"] = (g * s["x"].float().unsqueeze(1)).sum(2)
            g = g * s["w"].unsqueeze(2)
        out["dx"] = g.sum(1).to(dt)
    return out


def _plain_unsort(s):
    c = s["case"]
    T, k, d, dt = c["T"], c["k"], c["d"], s["rows"].dtype
    sr = s["plan"]["slot_row"]
    v = _gathered(s["rows"], sr).view(T, k, d)
    y = (v * s["w"].unsqueeze(2)).sum(1) if s["w"] is not None else v.sum(1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = dict(out=y.to(dt))
    if c["grad"]:
        out["drows"] = _spread(s["dout"], sr, s["w"], k, s["rows"].shape[0]).to(dt)
        if s["w"] is not None:
            out["dw"] = (v * s["dout"].float().unsqueeze(1)).sum(2)
        if s["residual"] is not None:
            out["dresidual"] = s["dout"]
    return out


def _act(z, name):
    """activation(z) and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    c = s["case"]
    a, w, dt = s["a"], s["w"], s["a"].dtype
    off = s["offsets"].long()
    # the groups as one batch of equal length (rows past a group's end are masked)
    place = torch.arange(s["most"], device=a.device).unsqueeze(0) + off[:-1].unsqueeze(1)
    live = place < off[1:].unsqueeze(1)
    R = a.shape[0]
    place = torch.where(live, place, R)

    def batch(t):
        return torch.where(live.unsqueeze(2), t[place.clamp(max=R - 1)].float(), 0.0)

    def rows(t):
        flat = torch.zeros((R + 1, t.shape[2]), dtype=torch.float32, device=a.device)
        flat[place.reshape(-1)] = t.reshape(-1, t.shape[2])
        return flat[:R]

    ab, wf = batch(a), w.float()
    z = torch.matmul(ab, wf.transpose(1, 2))
    if s["bias"] is not None:
        z = z + s["bias"].float().unsqueeze(1)
    y, slope = _act(z, c["act"])
    y = rows(y)
    if s["residual"] is not None:   # rows behind the last group are the residual alone
        y = y + s["residual"].float()
    out = dict(out=y.to(dt))
    if c["grad"]:
        dz = batch(s["dout"]) * slope
        out["da"] = rows(torch.matmul(dz, wf)).to(dt)
        out["dw"] = torch.matmul(dz.transpose(1, 2), ab).to(dt)
        if s["bias"] is not None:
            out["dbias"] = dz.sum(1).to(dt)
        if s["residual"] is not None:
            out["dresidual"] = s["dout"]
    return out


# ------------------------------------------------------------------------------ the framework's calls
def _own_sort(s):
    import swiftmoe_b200 as S
    c = s["case"]
    rows, plan = S.sort_tokens(s["x"], s["idx"], c["E"], weights=s["w"], capacity=c["capacity"], row_align=c["align"])
    out = dict(rows=rows, offsets=plan["offsets"], counts=plan["counts"], slot_row=plan["slot_row"])
    if c["grad"]:
        leaves = [s["x"]] + ([s["w"]] if s["w"] is not None else [])
        g = torch.autograd.grad(rows, leaves, s["drows"])
        out["dx"] = g[0]
        if s["w"] is not None:
            out["dw"] = g[1]
    return out


def _own_unsort(s):
    import swiftmoe_b200 as S
    y = S.unsort_tokens(s["rows"], s["plan"], weights=s["w"], residual=s["residual"])
    out = dict(out=y)
    if s["case"]["grad"]:
        names = ["rows"] + [n for n in ("w", "residual") if s[n] is not None]
        g = torch.autograd.grad(y, [s[n] for n in names], s["dout"])
        out.update({"d" + n: v for n, v in zip(names, g)})
    return out


def _own_linear(s):
    import swiftmoe_b200 as S
    c = s["case"]
    y = S.grouped_linear(s["a"], s["w"], s["offsets"], bias=s["bias"], activation=c["act"], residual=s["residual"])
    out = dict(out=y)
    if c["grad"]:
        names = ["a", "w"] + [n for n in ("bias", "residual") if s[n] is not None]
        g = torch.autograd.grad(y, [s[n] for n in names], s["dout"])
        out.update({"d" + n: v for n, v in zip(names, g)})
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"sort": _own_sort, "unsort": _own_unsort, "linear": _own_linear}[op](state)
    with torch.no_grad():
        return {"sort": _plain_sort, "unsort": _plain_unsort, "linear": _plain_linear}[op](state)


# ------------------------------------------------------------------------------ 64 bits
def _exact_rows(case, seed):
    """Row by row from the definition: expert e's rows are its (token, slot) pairs in
    order, at most `capacity` of them, its first row a multiple of `align`."""
    s = _row_inputs(case, seed)
    T, k, E, d = case["T"], case["k"], case["E"], case["d"]
    flat = s["idx"].reshape(-1).cpu()
    slot_row = torch.full((T * k,), -1, dtype=torch.int32)
    counts = torch.zeros(E, dtype=torch.int32)
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    for e in range(E):
        mine = torch.nonzero(flat == e).reshape(-1)
        counts[e] = mine.numel()
        if case["capacity"]:
            mine = mine[:case["capacity"]]
        slot_row[mine] = int(offsets[e]) + torch.arange(mine.numel(), dtype=torch.int32)
        offsets[e + 1] = int(offsets[e]) + -(-mine.numel() // case["align"]) * case["align"]
    live = torch.nonzero(slot_row >= 0).reshape(-1).cuda()   # slots, ascending
    dst = slot_row.cuda()[live].long()
    tok = live // k
    wt = s["w"].detach().double().reshape(-1)[live] if s["w"] is not None else torch.ones(live.numel(), dtype=torch.float64, device="cuda")
    wt = wt.unsqueeze(1)
    cap = max(s["cap"], 1)
    f64 = dict(dtype=torch.float64, device="cuda")
    if case["op"] == "sort":
        rows = torch.zeros((cap, d), **f64)
        rows[dst] = s["x"].double()[tok] * wt
        out = dict(rows=rows, offsets=offsets, counts=counts, slot_row=slot_row)
        if case["grad"]:
            g = s["drows"].double()[dst]
            out["dx"] = torch.zeros((T, d), **f64).index_add_(0, tok, g * wt)
            if s["w"] is not None:
                out["dw"] = torch.zeros(T * k, **f64).index_put_((live,), (g * s["x"].double()[tok]).sum(1)).view(T, k)
        return out
    y = s["residual"].double().clone() if s["residual"] is not None else torch.zeros((T, d), **f64)
    v = s["rows"].double()[dst]
    out = dict(out=y.index_add_(0, tok, v * wt))
    if case["grad"]:
        do = s["dout"].double()[tok]
        out["drows"] = torch.zeros((cap, d), **f64).index_put_((dst,), do * wt)
        if s["w"] is not None:
            out["dw"] = torch.zeros(T * k, **f64).index_put_((live,), (v * do).sum(1)).view(T, k)
        if s["residual"] is not None:
            out["dresidual"] = s["dout"].double()
    return out


def _exact_linear(case, seed):
    s = _linear_inputs(case, seed)
    R, G, K, N = case["R"] + case["tail"], case["G"], case["K"], case["N"]
    f64 = dict(dtype=torch.float64, device="cuda")
    off = s["offsets"].tolist()
    out = dict(out=torch.zeros((R, N), **f64))
    if case["grad"]:
        out.update(da=torch.zeros((R, K), **f64), dw=torch.zeros((G, N, K), **f64))
        if s["bias"] is not None:
            out["dbias"] = torch.zeros((G, N), **f64)
        if s["residual"] is not None:
            out["dresidual"] = s["dout"].double()
    for g in range(G):
        lo, hi = off[g], off[g + 1]
        if lo == hi:
            continue
        a, w = s["a"][lo:hi].double(), s["w"][g].double()
        z = a @ w.T
        if s["bias"] is not None:
            z += s["bias"][g].double()
        z.requires_grad_(case["grad"])
        with torch.enable_grad():
            if case["act"] == "gelu":
                y = 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
            elif case["act"] == "gelu_tanh":
                u = math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)
                y = z / (1 + torch.exp(-2 * u))
            elif case["act"] == "silu":
                y = z / (1 + torch.exp(-z))
            elif case["act"] == "relu":
                y = torch.where(z > 0, z, 0.0)
            else:
                y = z * 1.0
        if case["grad"]:
            do = s["dout"][lo:hi].double()
            (dz,) = torch.autograd.grad(y, z, do)
            out["da"][lo:hi] = dz @ w
            out["dw"][g] = dz.T @ a
            if s["bias"] is not None:
                out["dbias"][g] = dz.sum(0)
        out["out"][lo:hi] = y.detach()
    if s["residual"] is not None:
        out["out"] += s["residual"].double()
    return out


def exact(case, seed):
    if case["op"] == "linear":
        return _exact_linear(case, seed)
    with torch.no_grad():
        return _exact_rows(case, seed)
