"""sort_tokens, unsort_tokens and grouped_linear (kernels and autograd) against plain 64-bit
forms.  Tolerances are element-wise bounds: half a step of the output type on the result
(finfo.eps / 2), plus the fp32 arithmetic before it, plus -- in the gradients of an
activation -- the half step that rounding the kept pre-activations costs."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.autograd]

DT = [torch.bfloat16, torch.float16, torch.float32]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(scope="module")
def S():
    import swiftmoe_b200
    return swiftmoe_b200


@pytest.fixture(scope="module")
def K():
    from swiftmoe_b200 import kernels
    return kernels


def half_step(ref, dtype):
    """One rounding of ref to dtype (subnormals: half the smallest one)."""
    f = torch.finfo(dtype)
    return f.eps / 2 * ref.abs() + f.smallest_normal * f.eps / 2


def close(got, ref, bound):
    assert got.shape == ref.shape
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off; worst error / bound "
                           f"{float((err / bound.clamp(min=1e-300)).max()):.3f}")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def routing(T, E, k, seed, pad=0):
    g = gen(seed)
    idx = torch.stack([torch.randperm(E, generator=g, device="cuda")[:k] for _ in range(max(T, 1))])[:T].to(torch.int32)
    if pad:
        idx[T - pad:] = -1
        idx[::3, 0] = -1
    w = torch.rand((T, k), generator=g, device="cuda") + 0.05
    return idx.contiguous(), w


def plain_rows(idx, E, capacity, align):
    """slot -> row in (token, slot) order per expert (python loop), and the row total."""
    T, k = idx.shape
    flat = idx.reshape(-1).tolist()
    lists = [[s for s, e in enumerate(flat) if e == x] for x in range(E)]
    sr = [-1] * (T * k)
    start = 0
    for x in range(E):
        kept = lists[x][:capacity] if capacity else lists[x]
        for i, s in enumerate(kept):
            sr[s] = start + i
        start += -(-len(kept) // align) * align
    return torch.tensor(sr, device="cuda", dtype=torch.int64).view(T, k), start


ROWS = [  # T, d, E, k, capacity, align, pad
    (1, 4096, 8, 2, 0, 1, 0),
    (1, 8, 1, 1, 0, 1, 0),
    (5, 24, 4, 3, 0, 8, 2),        # 16-bit rows of 48 bytes
    (37, 1030, 13, 3, 7, 1, 5),    # even, not a multiple of 8; capacity
    (2000, 1034, 5, 2, 0, 8, 30),  # the same, one warp per token, several full steps
    (64, 129, 8, 8, 0, 64, 0),     # odd length, every expert of every token
    (33, 72, 40, 32, 3, 4, 9),     # k = 32
    (700, 264, 6, 2, 100, 1, 100),  # one warp per token
    (1500, 16, 3, 1, 0, 16, 0),
    (1900, 2064, 10, 9, 0, 1, 3),   # one warp per token, several full steps and a rest; k > 8
    (9, 64, 5, 2, 0, 1, 9),        # no token has an expert
]


@pytest.mark.parametrize("n,k,E,cap,align", [
    (2049, 1, 3, 0, 1),         # just past one block
    (20000, 4, 600, 0, 8),      # eight warps per block, several steps each, more than 512 experts
    (33000, 8, 128, 1500, 1),   # 32 warps per block
    (60011, 1, 4096, 3, 2),     # more experts than threads
    (300000, 2, 2, 0, 1024)])
def test_plan_of_many_slots(K, n, k, E, cap, align):
    g = gen(n)
    idx = torch.randint(-1, E, (n, k), generator=g, device="cuda", dtype=torch.int32)
    plan = K.dispatch_plan(idx, E, cap, align)
    flat = idx.reshape(-1).long()
    key = torch.where(flat >= 0, flat, E)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=E + 1)[:E]
    kept = counts.clamp(max=cap) if cap else counts
    start = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    start[1:] = torch.cumsum((kept + align - 1) // align * align, 0)
    first = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    first[1:] = torch.cumsum(counts, 0)
    sk = key[order]
    pos = torch.arange(n * k, device="cuda") - first[sk]
    live = (sk < E) & (pos < (cap or n * k))
    sr = torch.empty_like(flat)
    sr[order] = torch.where(live, start[sk.clamp(max=E - 1)] + pos, -1)
    assert torch.equal(plan["counts"].long(), counts) and torch.equal(plan["offsets"].long(), start)
    assert torch.equal(plan["slot_row"].long(), sr)
    total = int(start[E])
    tokens = torch.full((total,), -1, dtype=torch.int64, device="cuda")
    tokens[sr[sr >= 0]] = torch.nonzero(sr >= 0).reshape(-1) // k
    assert torch.equal(plan["row_token"][:total].long(), tokens)
    assert K.read_device_error("cuda") == 0


def same_rows(rows, sr, x, w, dtype):
    """rows[sr] = w x with one rounding, every other row exactly zero."""
    ref = torch.zeros(rows.shape, dtype=torch.float64, device="cuda")
    v = x.double().unsqueeze(1) * (w.double().unsqueeze(2) if w is not None else 1.0)
    v = v.expand(sr.shape[0], sr.shape[1], x.shape[1])
    live = sr >= 0
    ref[sr[live]] = v[live]
    if w is None:
        assert torch.equal(rows.double(), ref)
    else:   # the fp32 product is rounded before the type's own rounding
        close(rows, ref, half_step(ref, dtype) * (1 + 2.0 ** -10) + 2.0 ** -24 * ref.abs())


def same_sum(out, sr, y, w, residual, dtype):
    g = torch.where((sr >= 0).unsqueeze(2), y.double()[sr.clamp(min=0)], 0.0)
    t = g * (w.double().unsqueeze(2) if w is not None else 1.0)
    ref, mag = t.sum(1), t.abs().sum(1)
    if residual is not None:
        ref, mag = ref + residual.double(), mag + residual.double().abs()
    close(out, ref, half_step(ref, dtype) * (1 + 2.0 ** -10) + (2 * sr.shape[1] + 1) * 2.0 ** -24 * mag)


def same_dots(dw, sr, y, x):
    g = torch.where((sr >= 0).unsqueeze(2), y.double()[sr.clamp(min=0)], 0.0) * x.double().unsqueeze(1)
    # a lane adds its own terms one by one, then the lanes' and warps' sums
    n = x.shape[1] / 32 + 16
    close(dw, g.sum(2), n * 2.0 ** -24 * g.abs().sum(2) + 1e-37)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,d,E,k,cap,align,pad", ROWS)
@pytest.mark.parametrize("weighted", [False, True])
def test_sort_forward_and_gradients(S, dtype, T, d, E, k, cap, align, pad, weighted):
    idx, w = routing(T, E, k, T + d, pad)
    g = gen(7 * T + d)
    x = torch.randn((T, d), generator=g, device="cuda").to(dtype).requires_grad_()
    w = w.requires_grad_() if weighted else None
    rows, plan = S.sort_tokens(x, idx, E, weights=w, capacity=cap, row_align=align)
    sr, total = plain_rows(idx, E, cap, align)
    assert torch.equal(plan["slot_row"].view(T, k).long(), sr) and int(plan["offsets"][E]) == total
    assert rows.shape == (plan["rows_cap"], d)
    same_rows(rows.detach(), sr, x.detach(), w, dtype)
    drows = torch.randn(rows.shape, generator=g, device="cuda").to(dtype)
    drows[total:] = float("nan")          # rows of no slot have no influence
    grads = torch.autograd.grad(rows, [x] + ([w] if weighted else []), drows)
    same_sum(grads[0], sr, drows, w, None, dtype)
    if weighted:
        same_dots(grads[1], sr, drows, x.detach())
        (only_x,) = torch.autograd.grad(S.sort_tokens(x, idx, E, weights=w.detach(), capacity=cap, row_align=align)[0],
                                        [x], drows)
        assert torch.equal(only_x, grads[0])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,d,E,k,cap,align,pad", ROWS)
@pytest.mark.parametrize("weighted,res", [(False, True), (True, False), (True, True)])
def test_unsort_forward_and_gradients(S, K, dtype, T, d, E, k, cap, align, pad, weighted, res):
    idx, w = routing(T, E, k, T + d, pad)
    g = gen(11 * T + d)
    plan = K.dispatch_plan(idx, E, cap, align)
    sr, total = plain_rows(idx, E, cap, align)
    rows = torch.randn((plan["rows_cap"] + 3, d), generator=g, device="cuda").to(dtype)
    rows[total:] = float("inf")
    rows.requires_grad_()
    w = w.requires_grad_() if weighted else None
    r = torch.randn((T, d), generator=g, device="cuda").to(dtype).requires_grad_() if res else None
    out = S.unsort_tokens(rows, plan, weights=w, residual=r)
    same_sum(out.detach(), sr, rows.detach(), w, r, dtype)
    dout = torch.randn((T, d), generator=g, device="cuda").to(dtype)
    leaves = [rows] + [t for t in (w, r) if t is not None]
    grads = dict(zip(["rows"] + [n for n, t in (("w", w), ("r", r)) if t is not None],
                     torch.autograd.grad(out, leaves, dout)))
    same_rows(grads["rows"], sr, dout, w, dtype)
    if weighted:
        same_dots(grads["w"], sr, rows.detach(), dout)
        if not res:   # the same sums as the layer's combine, bit for bit
            assert torch.equal(out, K.combine(rows.detach(), plan["slot_row"], w.detach(), T, k))
    if res:
        assert torch.equal(grads["r"], dout)


def test_rows_gradients_against_differences(S, K):
    """Both operators are linear in each argument: central differences with any step are the
    directional derivative up to the fp32 rounding of the two outputs."""
    T, d, E, k = 50, 36, 7, 3
    idx, w = routing(T, E, k, 3, pad=4)
    g = gen(5)
    x, vx = torch.randn((T, d), generator=g, device="cuda"), torch.randn((T, d), generator=g, device="cuda")
    vw = torch.randn((T, k), generator=g, device="cuda")
    x.requires_grad_()
    w.requires_grad_()
    rows, plan = S.sort_tokens(x, idx, E, weights=w, capacity=15)
    c = torch.randn(rows.shape, generator=g, device="cuda")
    gx, gw = torch.autograd.grad(rows, [x, w], c)
    h = 0.5

    def f(a, b):
        return K.sort_rows(a, plan, b).double()

    for got, (p, m) in ((gx.double() * vx, (f(x + h * vx, w), f(x - h * vx, w))),
                        (gw.double() * vw, (f(x, w + h * vw), f(x, w - h * vw)))):
        noise = (c.double().abs() * (p.abs() + m.abs()) * 2.0 ** -22).sum() / (2 * h)
        assert abs(float(got.sum() - (c.double() * (p - m)).sum() / (2 * h))) <= float(noise)
    y, vy = torch.randn_like(rows), torch.randn(rows.shape, generator=g, device="cuda")
    y.requires_grad_()
    out = S.unsort_tokens(y, plan, weights=w)
    co = torch.randn(out.shape, generator=g, device="cuda")
    gy, gw = torch.autograd.grad(out, [y, w], co)

    def q(a, b):
        return K.unsort_rows(a, plan, b).double()

    mag = q(y.detach().abs() + h * vy.abs(), w.detach() + h * vw.abs())
    for got, (p, m) in ((gy.double() * vy, (q(y + h * vy, w), q(y - h * vy, w))),
                        (gw.double() * vw, (q(y, w + h * vw), q(y, w - h * vw)))):
        noise = (co.double().abs() * mag * 8 * 2.0 ** -22).sum() / (2 * h)
        assert abs(float(got.sum() - (co.double() * (p - m)).sum() / (2 * h))) <= float(noise)


# ------------------------------------------------------------------------ grouped linear
def act64(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z.clone()


def slope64(z, name):
    z = z.clone().requires_grad_()
    with torch.enable_grad():
        (s,) = torch.autograd.grad(act64(z, name).sum(), z)
    return s


def acc(K_):
    """fp32 accumulation on the tensor cores: up to a step of the running sum per 16-deep
    product, and the sums inside one."""
    return (K_ / 16 + 16) * 2.0 ** -23


def group_case(sizes, K_, N, dtype, seed, head=0, tail=0, bias="same", residual=True):
    g = gen(seed)
    R = head + sum(sizes) + tail
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    off = [head]
    for s in sizes:
        off.append(off[-1] + s)
    c = dict(a=n(R, K_).to(dtype), w=(n(len(sizes), N, K_) * K_ ** -0.5).to(dtype),
             b=None if bias is None else n(len(sizes), N).to(dtype if bias == "same" else torch.float32),
             r=n(R, N).to(dtype) if residual else None, dout=n(R, N).to(dtype),
             off=torch.tensor(off, dtype=torch.int32, device="cuda"), offs=off)
    return c


def ref_forward(c):
    """z, its accumulated magnitude, per row; NaN-free rows of groups only."""
    R, N = c["dout"].shape
    z = torch.zeros((R, N), dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(z)
    for g in range(c["w"].shape[0]):
        lo, hi = c["offs"][g], c["offs"][g + 1]
        a, w = c["a"][lo:hi].double(), c["w"][g].double()
        z[lo:hi], mag[lo:hi] = a @ w.T, a.abs() @ w.abs().T
        if c["b"] is not None:
            z[lo:hi] += c["b"][g].double()
            mag[lo:hi] += c["b"][g].double().abs()
    return z, mag


GROUPS = [  # sizes, K, N, rows before the first group, rows behind the last
    ([1], 8, 8, 0, 0),
    ([1], 4096, 24, 0, 0),               # single token: one group
    ([0, 1, 0, 1], 520, 264, 0, 0),      # one token's two experts
    ([2], 8200, 16, 0, 0),               # long rows, two warps per column
    ([0, 0, 1], 64, 40, 0, 1),           # one row in all, one row of no group
    ([3], 2048, 256, 0, 0),              # few tiles: K split
    ([40, 0, 9], 1536, 520, 2, 0),       # K split, two groups, rows before the first
    ([0, 300, 0, 77], 128, 256, 0, 5),
    ([129, 255, 3], 72, 200, 1, 130),    # sizes off every tile
    ([513, 64, 200], 256, 512, 0, 0),
    ([37] * 16 + [0] * 48, 136, 8, 0, 0),
    ([20, 0, 1500], 80, 72, 0, 0),       # weight gradient split along the rows, slices without any
    ([300, 5, 0, 200, 17] * 4, 64, 1056, 0, 3),   # several tiles per block, narrow last column tile
    ([0, 0, 0], 64, 64, 0, 7),           # no rows at all
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,K_,N,head,tail", GROUPS)
@pytest.mark.parametrize("act", ACTS)
def test_grouped_linear_forward(S, K, dtype, sizes, K_, N, head, tail, act):
    c = group_case(sizes, K_, N, dtype, K_ + N, head, tail, bias="fp32" if act == "silu" else "same",
                   residual=act != "gelu")
    z, mag = ref_forward(c)
    out = S.grouped_linear(c["a"], c["w"], c["off"], bias=c["b"], activation=act, residual=c["r"])
    ref = act64(z, act)
    # slopes of the activations stay below 1.13; their own evaluation to 2^-19
    err = 1.13 * acc(K_) * mag + 2.0 ** -19 * (1 + z.abs())
    if c["r"] is not None:
        ref, err = ref + c["r"].double(), err + 2.0 ** -23 * c["r"].double().abs()
    close(out, ref, half_step(ref, dtype) + err * (1 + torch.finfo(dtype).eps))
    # the rows of no group: the residual alone, or zeros
    lo, hi = c["offs"][0], c["offs"][-1]
    other = torch.cat([out[:lo], out[hi:]])
    want = torch.cat([c["r"][:lo], c["r"][hi:]]) if c["r"] is not None else torch.zeros_like(other)
    assert torch.equal(other, want)
    # a caller's buffer keeps them
    mine = torch.full_like(out, 7.0)
    K.grouped_linear(c["a"], c["w"], c["off"], c["b"], act, c["r"], out=mine)
    assert torch.equal(mine[lo:hi], out[lo:hi])
    assert (mine[:lo] == 7).all() and (mine[hi:] == 7).all()
    assert K.read_device_error("cuda") == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,K_,N,head,tail", GROUPS)
@pytest.mark.parametrize("act", ACTS)
def test_grouped_linear_gradients(S, K, dtype, sizes, K_, N, head, tail, act):
    c = group_case(sizes, K_, N, dtype, 3 * K_ + N, head, tail, bias="fp32" if act == "relu" else "same")
    lo, hi = c["offs"][0], c["offs"][-1]
    for t in (c["a"], c["dout"]):   # rows of no group must not reach any gradient
        t[:lo] = float("nan")
        t[hi:] = float("inf")
    leaves = [c["a"].requires_grad_(), c["w"].requires_grad_(), c["b"].requires_grad_(), c["r"].requires_grad_()]
    out = S.grouped_linear(c["a"], c["w"], c["off"], bias=c["b"], activation=act, residual=c["r"])
    da, dw, db, dr = torch.autograd.grad(out, leaves, c["dout"])
    with torch.no_grad():
        z, mag = ref_forward(c)
        eps = torch.finfo(dtype).eps
        slope = slope64(z, act)
        dout = c["dout"].double().clone()
        dout[:lo] = 0
        dout[hi:] = 0
        dz = dout * slope
        # z is kept rounded (half a step) after its accumulation error; |act''| < 1.2, and
        # relu's slope jumps where z is within its error of 0
        zerr = acc(K_) * mag + half_step(z, dtype)
        serr = (z.abs() <= zerr).double() if act == "relu" else (1.2 * zerr + 2.0 ** -18) * (act != "none")
        e32 = dout.abs() * serr + 2.0 ** -23 * dz.abs()
        e16 = e32 + (half_step(dz, dtype) * (1 + eps) if act != "none" else 0)
        for g in range(len(sizes)):
            a0, a1 = c["offs"][g], c["offs"][g + 1]
            a, w = c["a"][a0:a1].double(), c["w"][g].double()
            ref = dz[a0:a1] @ w
            close(da[a0:a1], ref, half_step(ref, dtype) + (1 + eps) * (
                e16[a0:a1] @ w.abs() + acc(N) * (dz[a0:a1].abs() @ w.abs())))
            n = a1 - a0
            ref = dz[a0:a1].T @ a
            close(dw[g], ref, half_step(ref, dtype) + (1 + eps) * (
                e16[a0:a1].T @ a.abs() + acc(n) * (dz[a0:a1].abs().T @ a.abs())))
            ref = dz[a0:a1].sum(0)
            close(db[g], ref, half_step(ref, db.dtype) + (1 + eps) * (
                e32[a0:a1].sum(0) + (n + 8) * 2.0 ** -24 * dz[a0:a1].abs().sum(0)))
        assert (da[:lo] == 0).all() and (da[hi:] == 0).all()
        assert dr.dtype == dtype and torch.equal(dr.isnan(), c["dout"].isnan())
        assert torch.equal(dr[lo:hi], c["dout"][lo:hi])
        # fp32 weight gradients: the same products without the last rounding
        z16 = torch.empty_like(c["dout"])
        K.grouped_linear(c["a"], c["w"], c["off"], c["b"], act, None, preact=z16)
        dz16, none = K.linear_act_bwd(c["dout"], c["off"], act, z16)
        w32 = K.linear_wgrad(dz16, c["a"], c["off"], out_dtype=torch.float32)
        assert none is None and torch.equal(w32.to(dtype), dw)
    assert K.read_device_error("cuda") == 0


def test_gradients_asked_for_one_at_a_time(S):
    c = group_case([70, 0, 33], 64, 72, torch.bfloat16, 1, 1, 2)
    full = [c[n].clone().requires_grad_() for n in "awbr"]
    want = torch.autograd.grad(S.grouped_linear(full[0], full[1], c["off"], full[2], "gelu", full[3]), full, c["dout"])
    for i in range(4):
        one = [c[n].clone().requires_grad_(j == i) for j, n in enumerate("awbr")]
        (got,) = torch.autograd.grad(S.grouped_linear(one[0], one[1], c["off"], one[2], "gelu", one[3]), [one[i]], c["dout"])
        assert torch.equal(got, want[i])
    # a gradient that is a broadcast view
    out = S.grouped_linear(full[0], full[1], c["off"], full[2], "silu", full[3])
    a = torch.autograd.grad(out.sum(), full, retain_graph=True)
    b = torch.autograd.grad(out, full, torch.ones_like(out))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_grouped_linear_gradient_against_differences(S, act):
    """Directional derivative by central differences of the operator itself (fp16): its
    roundings are independent half steps at most (six standard deviations of a uniform
    error), the step's curvature term h^2 / 6 |f'''| with |act'''| < 2.2."""
    c = group_case([40, 0, 25], 64, 48, torch.float16, 9, residual=False)
    v = (torch.randn(c["a"].shape, generator=gen(4), device="cuda") * 0.5).half()
    h = 2.0 ** -3
    a = c["a"].requires_grad_()
    out = S.grouped_linear(a, c["w"], c["off"], bias=c["b"], activation=act)
    (da,) = torch.autograd.grad(out, [a], c["dout"])
    with torch.no_grad():
        hi, lo = (a.double() + h * v.double()).half(), (a.double() - h * v.double()).half()
        p, m = (S.grouped_linear(t, c["w"], c["off"], bias=c["b"], activation=act).double() for t in (hi, lo))
        step = (hi.double() - lo.double()) / (2 * h)     # the direction after fp16's rounding
        dout = c["dout"].double()
        want, got = (dout * (p - m)).sum() / (2 * h), (da.double() * step).sum()
        eps = torch.finfo(torch.float16).eps
        var = (dout * eps / 2 * (p.abs() + m.abs())).square().sum() / 3 / (2 * h) ** 2
        var = var + (half_step(da.double(), torch.float16) * step).square().sum()
        dz = torch.zeros_like(dout)
        for g in range(3):
            s = slice(c["offs"][g], c["offs"][g + 1])
            dz[s] = step[s] @ c["w"][g].double().T
        curve = (dout.abs() * 2.2 * dz.abs() ** 3).sum() * h * h / 6
        # the kept z and dz roundings reach da once each
        var = var + (dout * dz * eps * 1.2).square().sum()
        assert abs(float(want - got)) <= 6 * math.sqrt(float(var)) + float(curve)


def test_gradient_that_starts_off_a_16_byte_boundary(S):
    c = group_case([70, 0, 33], 64, 72, torch.bfloat16, 1, 1, 2)
    leaves = [c[n].clone().requires_grad_() for n in "awbr"]
    want = torch.autograd.grad(S.grouped_linear(leaves[0], leaves[1], c["off"], leaves[2], "gelu", leaves[3]), leaves, c["dout"])
    buf = torch.empty(c["dout"].numel() + 1, dtype=torch.bfloat16, device="cuda")
    dout = buf[1:].view(c["dout"].shape).copy_(c["dout"])
    got = torch.autograd.grad(S.grouped_linear(leaves[0], leaves[1], c["off"], leaves[2], "gelu", leaves[3]), leaves, dout)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("sizes", [[1, 0, 1], [70, 0, 33], [300, 500, 200]])
def test_residual_in_place(S, K, sizes):
    """out may be the residual: rows of two decode kernels, a split and a whole launch."""
    c = group_case(sizes, 1024, 72, torch.bfloat16, 1, 1 if sum(sizes) > 2 else 0, 0)
    want = S.grouped_linear(c["a"], c["w"], c["off"], c["b"], "silu", c["r"])
    out = c["r"].clone()
    assert K.grouped_linear(c["a"], c["w"], c["off"], c["b"], "silu", out, out=out) is out
    assert torch.equal(out, want)


def test_relu_passes_the_gradient_at_nan(S):
    c = group_case([40], 64, 24, torch.bfloat16, 3, 0, 0, residual=False)
    a, b, ones = c["a"].clone(), c["b"].clone().requires_grad_(), torch.ones_like(c["dout"])
    rest = ones.clone()
    rest[7] = 0
    others, = torch.autograd.grad(S.grouped_linear(a, c["w"], c["off"], b, "relu"), [b], rest)
    a[7] = float("nan")
    every, = torch.autograd.grad(S.grouped_linear(a, c["w"], c["off"], b, "relu"), [b], ones)
    assert torch.equal(every, others + 1)   # counts of rows, exact in bf16


def test_infinities_and_nan_stay_in_their_rows(S):
    """A NaN or infinity in a group's rows reaches that row's outputs and that group's weight
    gradient only, whatever tile it shares."""
    c = group_case([70, 30, 28], 64, 40, torch.bfloat16, 2, 0, 3, residual=False)
    clean = [c[n].clone().requires_grad_() for n in "awb"]
    bad = [c[n].clone() for n in "awb"]
    bad[0][75] = float("inf")
    bad[0][80, 3] = float("nan")
    bad = [t.requires_grad_() for t in bad]
    o1 = S.grouped_linear(clean[0], clean[1], c["off"], bias=clean[2], activation="relu")
    o2 = S.grouped_linear(bad[0], bad[1], c["off"], bias=bad[2], activation="relu")
    keep = [r for r in range(131) if r not in (75, 80)]
    assert torch.equal(o1[keep], o2[keep]) and o2[80].isnan().all()
    g1 = torch.autograd.grad(o1, clean, c["dout"])
    g2 = torch.autograd.grad(o2, bad, c["dout"])
    assert torch.equal(g1[1][[0, 2]], g2[1][[0, 2]]) and not g2[1][1].isfinite().all()
    assert torch.equal(g1[0][keep], g2[0][keep])


def routed_mlp(S, x, idx, w, p, E, act="gelu", capacity=0):
    rows, plan = S.sort_tokens(x, idx, E, capacity=capacity)
    h = S.grouped_linear(rows, p["w1"], plan["offsets"], bias=p["b1"], activation=act)
    y = S.grouped_linear(h, p["w2"], plan["offsets"], bias=p["b2"])
    return S.unsort_tokens(y, plan, weights=w, residual=x)


def mlp_params(E, d, F, dtype, seed):
    g = gen(seed)
    n = lambda *s, std: (torch.randn(s, generator=g, device="cuda") * std).to(dtype)  # noqa: E731
    return dict(w1=n(E, F, d, std=d ** -0.5), b1=n(E, F, std=0.3), w2=n(E, d, F, std=F ** -0.5), b2=n(E, d, std=0.3))


@pytest.mark.parametrize("capacity", [0, 40])
def test_routed_mlp_trains_as_its_64_bit_form(S, K, capacity):
    """The operators together: router, sort, two linear layers with biases, unsort with the
    gate weights and the residual; loss gradients of everything."""
    T, d, E, F, k, dtype = 150, 96, 5, 136, 2, torch.bfloat16
    g = gen(1)
    p = mlp_params(E, d, F, dtype, 2)
    x = torch.randn((T, d), generator=g, device="cuda").to(dtype)
    idx, w = K.router(x, torch.randn((E, d), generator=g, device="cuda").to(dtype), k)
    dout = torch.randn((T, d), generator=g, device="cuda").to(dtype)
    leaves = [t.requires_grad_() for t in (x, w, *p.values())]
    out = routed_mlp(S, x, idx, w, p, E, capacity=capacity)
    got = torch.autograd.grad(out, leaves, dout)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    x64, w64, (w1, b1, w2, b2) = ref[0], ref[1], ref[2:]
    o = x64.clone()
    flat = idx.reshape(-1)
    for e in range(E):
        s = torch.nonzero(flat == e).reshape(-1)[:capacity or None]
        t = s // k
        y = act64(x64[t] @ w1[e].T + b1[e], "gelu") @ w2[e].T + b2[e]
        o = o.index_add(0, t, y * w64.reshape(-1)[s].unsqueeze(1))
    want = torch.autograd.grad(o, ref, dout.double())
    # three stored 16-bit intermediates on the way (h, y and the rows' gradients): relative to
    # the tensor's size, each costs about half a step
    for a, b in zip([out, *got], [o, *want]):
        assert float(((a.double() - b).norm() / b.norm()).detach()) <= 4 * torch.finfo(dtype).eps / 2


def test_same_results_every_time(S, K):
    idx, w = routing(3000, 16, 4, 8)
    p = mlp_params(16, 128, 256, torch.bfloat16, 3)
    x = torch.randn((3000, 128), generator=gen(2), device="cuda").bfloat16()
    dout = torch.randn((3000, 128), generator=gen(3), device="cuda").bfloat16()
    first = None
    for _ in range(3):
        leaves = [t.detach().clone().requires_grad_() for t in (x, w, *p.values())]
        q = dict(zip(p, leaves[2:]))
        out = routed_mlp(S, leaves[0], idx, leaves[1], q, 16)
        res = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
        first = first or res
        assert all(torch.equal(a, b) for a, b in zip(first, res))


def test_captured_and_replayed(S, K):
    """Forward and backward captured into a CUDA graph, replayed on other inputs and routing;
    two such graphs of split launches replayed on two streams at once."""
    T, E, d, F, k = 24, 4, 512, 256, 2
    p = mlp_params(E, d, F, torch.bfloat16, 5)
    leaves = [t.requires_grad_() for t in p.values()]

    def inputs(seed):
        idx, w = routing(T, E, k, seed)
        g = gen(seed)
        return [torch.randn((T, d), generator=g, device="cuda").bfloat16(), idx, w,
                torch.randn((T, d), generator=g, device="cuda").bfloat16()]

    def step(x, idx, w, dout):
        out = routed_mlp(S, x, idx, w, p, E)
        return [out.detach(), *torch.autograd.grad(out, [x, w, *leaves], dout)]

    def eager(seed):
        x, idx, w, dout = inputs(seed)
        return [t.clone() for t in step(x.requires_grad_(), idx, w.requires_grad_(), dout)]

    want = {s: eager(s) for s in range(4)}
    graphs = []
    for s in range(2):
        static = inputs(s)
        static[0].requires_grad_()
        static[2].requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(*static)
        graphs.append((graph, static, res))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(2):
        with torch.no_grad():
            for s, (_, static, _) in enumerate(graphs):
                for dst, src in zip(static, inputs(2 * turn + s)):
                    dst.copy_(src)
        torch.cuda.synchronize()
        for _ in range(5):
            for st, (graph, _, _) in zip(streams, graphs):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for s, (_, _, res) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(res, want[2 * turn + s]))


def test_on_another_stream(S):
    c = group_case([40, 9], 512, 256, torch.bfloat16, 6)
    want = S.grouped_linear(c["a"], c["w"], c["off"], bias=c["b"], activation="silu", residual=c["r"])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = S.grouped_linear(c["a"], c["w"], c["off"], bias=c["b"], activation="silu", residual=c["r"])
    st.synchronize()
    assert torch.equal(got, want)


def test_no_tokens_and_no_rows(S):
    x = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    idx = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    rows, plan = S.sort_tokens(x, idx, 4, row_align=8)
    assert rows.shape == (28, 64) and not rows.any()
    rows, plan = S.sort_tokens(x, idx, 4)
    w = torch.randn((4, 32, 64), device="cuda").bfloat16().requires_grad_()
    b = torch.randn((4, 32), device="cuda").bfloat16().requires_grad_()
    h = S.grouped_linear(rows, w, plan["offsets"], bias=b, activation="relu")
    out = S.unsort_tokens(h, plan, weights=torch.empty((0, 2), device="cuda"))
    assert rows.shape == (0, 64) and h.shape == (0, 32) and out.shape == (0, 32)
    gx, gw, gb = torch.autograd.grad(out, [x, w, b], torch.empty_like(out))
    assert gx.shape == (0, 64) and not gw.any() and not gb.any()


def test_row_offsets_past_32_bits(S, K):
    """Rows whose elements lie beyond 2^31: addressing is 64-bit."""
    T, d, E, k = 66000, 16384, 4, 2     # 132000 rows x 16384 = 2.16e9 elements
    g = gen(1)
    idx = torch.randint(0, E, (T, 1), generator=g, device="cuda", dtype=torch.int32)
    idx = torch.cat([idx, (idx + 1) % E], 1).contiguous()
    x = torch.randn((T, d), generator=g, device="cuda", dtype=torch.bfloat16)
    rows, plan = S.sort_tokens(x, idx, E)
    sr = plan["slot_row"].view(T, k).long()
    for t in (0, T // 2, T - 1):
        assert torch.equal(rows[sr[t, 0]], x[t]) and torch.equal(rows[sr[t, 1]], x[t])
    last = int(sr.argmax())
    assert int(sr.max()) == T * k - 1 and torch.equal(rows[T * k - 1], x[last // k])
    out = S.unsort_tokens(rows, plan)
    assert torch.equal(out, (2 * x.float()).bfloat16())


# ------------------------------------------------------------------------------ refusals
def test_refusals(S, K):
    from swiftmoe_b200._lib import SwiftMoEError
    x = torch.randn((6, 16), device="cuda").bfloat16()
    idx, w = routing(6, 4, 2, 1)
    rows, plan = S.sort_tokens(x, idx, 4)
    off = plan["offsets"]
    wt = torch.randn((4, 24, 16), device="cuda").bfloat16()

    def refused(f):
        with pytest.raises(SwiftMoEError):
            f()

    refused(lambda: S.sort_tokens(x.cpu(), idx, 4))
    refused(lambda: S.sort_tokens(x.double(), idx, 4))
    refused(lambda: S.sort_tokens(x, idx.long(), 4))
    refused(lambda: S.sort_tokens(x[:5].contiguous(), idx, 4))
    refused(lambda: S.sort_tokens(x.t().contiguous().t(), idx, 4))
    refused(lambda: S.sort_tokens(x, idx, 4, weights=w.half()))
    refused(lambda: S.sort_tokens(x, idx, 4, weights=w[:, :1].contiguous()))
    refused(lambda: S.sort_tokens(x, torch.zeros((6, 33), dtype=torch.int32, device="cuda"), 40))   # k > 32
    refused(lambda: S.unsort_tokens(rows[:11].contiguous(), plan))       # fewer rows than the plan's
    refused(lambda: S.unsort_tokens(rows, plan, residual=x.half()))
    refused(lambda: S.unsort_tokens(rows, plan, residual=x[:, :8].contiguous()))
    refused(lambda: S.unsort_tokens(rows, plan, weights=w.double()))
    refused(lambda: K.sort_rows(x, plan, y=rows))                        # dw without weights
    refused(lambda: K.unsort_rows(rows, plan, x=x))
    refused(lambda: S.grouped_linear(rows.float(), wt.float(), off))     # 16-bit only
    refused(lambda: S.grouped_linear(rows, wt.half(), off))
    refused(lambda: S.grouped_linear(rows, wt, off[:-1].contiguous()))
    refused(lambda: S.grouped_linear(rows, wt, off.long()))
    refused(lambda: S.grouped_linear(rows, wt, off, activation="tanh"))
    refused(lambda: S.grouped_linear(rows, wt, off, bias=wt[:, :, 0].contiguous().half()))
    refused(lambda: S.grouped_linear(rows, wt, off, bias=wt[0, :, 0].contiguous()))
    refused(lambda: S.grouped_linear(rows, wt, off, residual=rows))
    refused(lambda: S.grouped_linear(rows, wt[:, :, :8].contiguous(), off))
    refused(lambda: S.grouped_linear(rows, wt[:, :20].contiguous(), off))                          # N % 8
    refused(lambda: S.grouped_linear(rows[:, :12].contiguous(), wt[:, :, :12].contiguous(), off))  # K % 8
    flat = torch.randn(12 * 16 + 1, device="cuda").bfloat16()[1:].view(12, 16)
    refused(lambda: S.grouped_linear(flat, wt, off))                     # 2-byte aligned
    refused(lambda: K.linear_act_bwd(rows, off, "gelu"))                 # no pre-activations
    refused(lambda: K.linear_wgrad(rows, x, off))                        # row counts differ
    # an unaligned row pointer is fine where rows are moved element by element
    got, _ = S.sort_tokens(torch.cat([x.reshape(-1), x.reshape(-1)[:1]])[:-1].view(6, 16), idx, 4)
    assert torch.equal(got, rows)
    shifted = torch.empty(6 * 16 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 16)
    shifted.copy_(x)
    assert torch.equal(S.sort_tokens(shifted, idx, 4)[0], rows)
