"""Edges of sort_tokens, unsort_tokens and grouped_linear: pre-activations past the 16-bit
range, the activations over their whole range, plans that change between forward and
backward, gradients of some inputs only."""
import gc
import math
import weakref

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.autograd]

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(scope="module")
def S():
    import swiftmoe_b200
    return swiftmoe_b200


@pytest.fixture(scope="module")
def K():
    from swiftmoe_b200 import kernels
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half_step(ref, dtype):
    f = torch.finfo(dtype)
    return f.eps / 2 * ref.abs() + f.smallest_normal * f.eps / 2


def close(got, ref, bound):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off; worst error / bound "
                           f"{float((err / bound.clamp(min=1e-300)).nan_to_num(nan=math.inf).max()):.3f}")


def phi_of(z):
    """The normal distribution function and density."""
    return 0.5 * torch.erfc(-z / math.sqrt(2)), torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def two_u(z):
    return 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * phi_of(z)[0]
    if name == "gelu_tanh":
        return z * torch.sigmoid(two_u(z))
    return z * torch.sigmoid(z) if name == "silu" else z.clone()


def slope64(z, name):
    """(act'(z), the sum of its terms' magnitudes); finite for every finite z."""
    if name == "relu":
        s = (z > 0).double()
        return s, s
    if name == "gelu":
        p, d = phi_of(z)
        return p + z * d, p + z.abs() * d
    if name == "gelu_tanh":
        a, b = torch.sigmoid(two_u(z)), torch.sigmoid(-two_u(z))
        t = z * a * b * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
        return a + t, a + t.abs()
    if name == "silu":
        a, b = torch.sigmoid(z), torch.sigmoid(-z)
        return a + z * a * b, a + (z * a * b).abs()
    return torch.ones_like(z), torch.ones_like(z)


def relative(z, name):
    """Relative error of an activation evaluated in fp32.  An exponential's argument of size A
    is off by a few roundings, 2^-22 A; the rest of the evaluation by 2^-19."""
    size = {"gelu": 0.5 * z * z, "gelu_tanh": two_u(z).abs(), "silu": z.abs()}.get(name)
    if size is None:
        return torch.zeros_like(z)
    return 2.0 ** -19 + 2.0 ** -21 * size.clamp(max=200)


# -------------------------------------------------------------------------- activations
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
def test_activation_over_its_whole_range(S, act, dtype, rows):
    """z = the fp32 bias of a layer of zeros: relative accuracy down to the smallest normal
    number, in the tails too."""
    z = torch.cat([torch.linspace(-14, 14, 40000), torch.linspace(-100, 100, 8000),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 3e4, -3e4, -1e20, -3e38])]).cuda()
    n = z.numel()
    out = S.grouped_linear(torch.zeros((rows, 8), dtype=dtype, device="cuda"),
                           torch.zeros((1, n, 8), dtype=dtype, device="cuda"),
                           torch.tensor([0, rows], dtype=torch.int32, device="cuda"), bias=z.view(1, n), activation=act)
    z = z.double()
    ref = act64(z, act)
    big = ref.abs() > torch.finfo(dtype).max
    assert torch.equal(out[:, big], ref[big].to(dtype).expand(rows, -1))
    ref, z = ref[~big], z[~big]
    err = relative(z, act) * ref.abs() + 2.0 ** -126
    close(out[:, ~big], ref, half_step(ref, dtype) + (1 + torch.finfo(dtype).eps) * err)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS[1:])
def test_slope_of_every_16_bit_number(K, act, dtype):
    z = torch.arange(-32768, 32768, device="cuda").to(torch.int16).view(dtype).view(64, 1024)
    dz, _ = K.linear_act_bwd(torch.ones_like(z), torch.tensor([0, 64], dtype=torch.int32, device="cuda"), act, z)
    assert torch.equal(dz.isnan() & ~z.isnan(), torch.zeros_like(z, dtype=torch.bool))
    if act != "relu":
        assert dz[z.isnan()].isnan().all()
    assert (dz[z == math.inf] == 1).all() and (dz[z == -math.inf] == 0).all()
    ok = z.isfinite()
    z, dz = z[ok].double(), dz[ok]
    ref, mag = slope64(z, act)
    # beyond |z| = 200 every slope is 0 or 1 (and z d may overflow nowhere: d is 0)
    far = z.abs() > 200
    ref = torch.where(far, (z > 0).double(), ref)
    mag = torch.where(far, ref, mag)
    close(dz, ref, half_step(ref, dtype) + (1 + torch.finfo(dtype).eps) * (relative(z, act) * mag + 2.0 ** -126))


@pytest.mark.parametrize("rows", [2, 40, 300])
@pytest.mark.parametrize("act", ACTS)
def test_finite_gradients_where_pre_activations_leave_fp16(S, act, rows):
    """fp16: z = -70000 and, with a residual that brings the sum back, z = 70000 are finite in
    the forward's fp32 arithmetic; the kept pre-activations are infinite there."""
    g, d, n = gen(rows), 64, 24
    a = torch.randn((rows, d), generator=g, device="cuda").half()
    w = (torch.randn((1, n, d), generator=g, device="cuda") / 8).half()
    r = torch.randn((rows, n), generator=g, device="cuda").half()
    b = torch.zeros((1, n), device="cuda")
    dout = torch.randn((rows, n), generator=g, device="cuda").half()
    a[1] = 0
    a[:, 0] = 0
    a[1, 0] = 1000.0
    w[0, 3, 0], w[0, 5, 0] = 70.0, -70.0
    r[1, 3] = -40000.0
    if act == "none" or act == "relu":
        w[0, 5, 0] = -60.0 if act == "none" else -70.0
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (a, w, b, r)]
    out = S.grouped_linear(a, w, off, bias=b, activation=act, residual=r)
    got = torch.autograd.grad(out, leaves, dout)
    a, w, r = a.detach().double(), w.detach()[0].double(), r.detach().double()
    z = a @ w.T
    assert out.isfinite().all() and float(z[1, 3].detach()) == 70000.0
    close(out[1], act64(z[1], act) + r[1], half_step(act64(z[1], act) + r[1], torch.float16) * 1.01 + 70000 * 2.0 ** -19)
    do = dout.double()
    slope = torch.where(z.abs() > 200, (z > 0).double() if act != "none" else torch.ones_like(z), slope64(z, act)[0])
    dz = do * slope
    # the rounding of the kept z (half a step, |act''| < 1.2; relu's jump), of dz and of the result
    zerr = half_step(z, torch.float16) * (z.abs() <= 200) + (d / 16 + 16) * 2.0 ** -23 * (a.abs() @ w.abs().T)
    serr = (z.abs() <= zerr).double() if act == "relu" else 1.2 * zerr * (z.abs() <= 200) * (act != "none")
    e = do.abs() * serr + half_step(dz, torch.float16) * 1.01 + 2.0 ** -18 * do.abs()
    for x, ref, err in ((got[0], dz @ w, e @ w.abs() + 2.0 ** -19 * (dz.abs() @ w.abs())),
                        (got[1][0], dz.T @ a, e.T @ a.abs() + 2.0 ** -18 * (dz.abs().T @ a.abs())),
                        (got[2][0], dz.sum(0), e.sum(0) + rows * 2.0 ** -23 * dz.abs().sum(0)), (got[3], do, 0 * do)):
        assert x.isfinite().all()
        close(x, ref, half_step(ref, x.dtype) * 1.01 + err)


# ----------------------------------------------------------------------------- the plan
def routed(S, capacity=0, align=1):
    g = gen(5)
    T, E, k, d = 60, 5, 2, 32
    idx = torch.stack([torch.randperm(E, generator=g, device="cuda")[:k] for _ in range(T)]).to(torch.int32)
    x = torch.randn((T, d), generator=g, device="cuda").bfloat16().requires_grad_()
    w = torch.rand((T, k), generator=g, device="cuda").requires_grad_()
    wt = (torch.randn((E, d, d), generator=g, device="cuda") / 6).bfloat16().requires_grad_()
    rows, plan = S.sort_tokens(x, idx, E, weights=w, capacity=capacity, row_align=align)
    return x, w, wt, rows, plan


def test_load_counts_may_be_updated_before_the_backward(S):
    def grads(change):
        x, w, wt, rows, plan = routed(S)
        out = S.unsort_tokens(S.grouped_linear(rows, wt, plan["offsets"]), plan, weights=w)
        if change:
            plan["counts"].add_(7).mul_(3)
        return torch.autograd.grad(out, [x, w, wt], torch.ones_like(out))

    assert all(torch.equal(p, q) for p, q in zip(grads(False), grads(True)))


def test_plan_arrays_own_their_memory(S):
    """Keeping one of them keeps no other one, nor the plan's scratch."""
    plan = routed(S)[4]
    arrays = [plan[n] for n in ("counts", "offsets", "slot_row", "row_token")]
    assert len({t.untyped_storage().data_ptr() for t in arrays}) == 4
    for t in arrays:
        assert t.untyped_storage().nbytes() == t.numel() * 4


@pytest.mark.parametrize("name", ["slot_row", "offsets", "row_token"])
@pytest.mark.parametrize("align", [1, 8])
def test_a_plan_changed_in_place_is_not_used_for_gradients(S, name, align):
    """What a backward reads of the plan is as it was in the forward, or the backward is refused."""
    def run(change):
        x, w, _, rows, plan = routed(S, align=align)
        out = S.unsort_tokens(rows, plan, weights=w)
        keep = plan[name].clone()
        if change:
            plan[name].zero_()
        try:
            return torch.autograd.grad(out, [x, w], torch.ones_like(out)), None
        except RuntimeError as e:
            plan[name].copy_(keep)
            return None, str(e)

    want, _ = run(False)
    got, error = run(True)
    if error is None:
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    else:
        assert "modified by an inplace operation" in error
    if name == "slot_row":
        assert error is not None
        # sort's own backward, too
        x, w, _, rows, plan = routed(S, align=align)
        plan["slot_row"].zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(rows, [x], torch.ones_like(rows))


def test_a_plan_entry_replaced_before_the_backward_has_no_influence(S):
    def grads(change):
        x, w, _, rows, plan = routed(S)
        out = S.unsort_tokens(rows, plan, weights=w)
        if change:
            plan["slot_row"] = torch.zeros_like(plan["slot_row"])
            plan["offsets"] = torch.zeros_like(plan["offsets"])
            plan["rows_cap"] = 1
        return torch.autograd.grad(out, [x, w], torch.ones_like(out))

    assert all(torch.equal(p, q) for p, q in zip(grads(False), grads(True)))


# ------------------------------------------------------------------ gradients of some inputs
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,d,E,k,cap,align", [(60, 32, 5, 2, 0, 1), (2500, 264, 16, 4, 500, 8), (33, 1027, 40, 32, 3, 4),
                                               (700, 1032, 12, 10, 0, 1)])
def test_gradient_of_the_weights_alone(S, dtype, T, d, E, k, cap, align):
    g = gen(T)
    idx = torch.stack([torch.randperm(E, generator=g, device="cuda")[:k] for _ in range(T)]).to(torch.int32)
    w = torch.rand((T, k), generator=g, device="cuda").requires_grad_()
    x = torch.randn((T, d), generator=g, device="cuda").to(dtype)

    def both(call, other, dout, terms=None):
        o = other.detach().requires_grad_()
        want = torch.autograd.grad(call(o), [o, w], dout)[1]
        out = call(other.detach())
        gc.collect()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        (got,) = torch.autograd.grad(out, [w], dout)
        peak = torch.cuda.max_memory_allocated() - before
        if terms is None:
            assert torch.equal(got, want)
        else:   # the same products in another fp32 order: a lane's own terms, then lanes and warps
            x_, y_, sr = terms
            mag = torch.where((sr >= 0).unsqueeze(2), y_.double()[sr.clamp(min=0)], 0.0).mul(x_.double().unsqueeze(1))
            close(got, want.double(), 2 * (d / 32 + 16) * 2.0 ** -24 * mag.abs().sum(2))
        return peak

    rows, plan = S.sort_tokens(x, idx, E, capacity=cap, row_align=align)
    drows, dout = torch.randn_like(rows), torch.randn_like(x)
    dw_bytes = -(-T * k * 4 // 512) * 512
    # the gradient itself is all that is allocated
    assert both(lambda t: S.sort_tokens(t, idx, E, weights=w, capacity=cap, row_align=align)[0], x, drows,
                (x, drows, plan["slot_row"].view(T, k).long())) <= dw_bytes
    assert both(lambda t: S.unsort_tokens(t, plan, weights=w), rows, dout) <= dw_bytes


@pytest.mark.parametrize("needs", ["a", "w", "b", "r"])
def test_grouped_linear_keeps_what_its_gradients_need(S, needs):
    g = gen(1)
    off = torch.tensor([0, 30, 50], dtype=torch.int32, device="cuda")

    def made():
        t = dict(a=torch.randn((50, 64), generator=g, device="cuda"), w=torch.randn((2, 24, 64), generator=g, device="cuda"),
                 b=torch.randn((2, 24), generator=g, device="cuda"), r=torch.randn((50, 24), generator=g, device="cuda"))
        return {n: v.bfloat16() for n, v in t.items()}

    t = made()
    t[needs].requires_grad_()
    leaf, dead = t[needs], {n: weakref.ref(v) for n, v in t.items() if n != needs}
    out = S.grouped_linear(t["a"], t["w"], off, bias=t["b"], activation="gelu", residual=t["r"])
    del t
    gc.collect()
    kept = {n for n, v in dead.items() if v() is not None}
    assert kept == {"a": {"w"}, "w": {"a"}, "b": set(), "r": set()}[needs]
    (grad,) = torch.autograd.grad(out, [leaf], torch.ones_like(out))
    assert grad.shape == leaf.shape


@pytest.mark.parametrize("total", [40, 1 << 30])
def test_offsets_past_the_plan_read_nothing_behind_it(S, K, total):
    """Rows of a larger tensor than the plan's, and a plan whose total says they are its own:
    its rows as they should be, the ones behind it zeros."""
    x, _, _, _, plan = routed(S, align=8)
    cap, x = plan["rows_cap"], x.detach()
    want = K.sort_rows(x, plan)
    got = K.sort_rows(x, plan, rows_cap=cap + 500)
    assert torch.equal(got[:cap], want) and not got[cap:].any()
    assert plan["row_token"].numel() == cap
    total_ = int(plan["offsets"][-1])
    plan["row_token"][total_:] = -1
    plan["offsets"][-1] = cap + total
    got = K.sort_rows(x, plan, rows_cap=cap + 500)
    assert torch.equal(got[:cap], want) and not got[cap:].any()


# ----------------------------------------------------------------------------- refusals
def test_sizes_past_32_bits(S):
    from swiftmoe_b200._lib import SwiftMoEError
    x, idx = torch.randn((6, 16), device="cuda").bfloat16(), torch.zeros((6, 2), dtype=torch.int32, device="cuda")
    big = 1 << 32
    for kw in (dict(num_experts=big + 4), dict(num_experts=0), dict(num_experts=4097), dict(num_experts=4, row_align=big + 1),
               dict(num_experts=4, row_align=0), dict(num_experts=4, row_align=1025)):
        with pytest.raises(SwiftMoEError):
            S.sort_tokens(x, idx, **kw)
    # more than every slot: all of them are kept
    rows, plan = S.sort_tokens(x, idx, 4, capacity=big + 5)
    assert plan["rows_cap"] == 12 and torch.equal(rows, x.repeat_interleave(2, 0))


def test_shapes_and_overlaps_are_refused_as_such(S, K):
    from swiftmoe_b200._lib import SwiftMoEError
    n = lambda *s: torch.randn(s, device="cuda").bfloat16()  # noqa: E731
    a, w, r, off = n(12, 16), n(2, 16, 16), n(12, 16), torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda")
    both = n(18, 16)
    wg = w.clone().requires_grad_()

    def refused(f):
        with pytest.raises(SwiftMoEError):
            f()

    refused(lambda: S.grouped_linear(a[0], wg, off))                          # the same with and without gradients
    refused(lambda: S.grouped_linear(a[0], w, off))
    refused(lambda: S.grouped_linear(a, wg[0], off))
    refused(lambda: S.grouped_linear(a, wg[0, 0], off))
    refused(lambda: K.linear_act_bwd(a[0], off, "none"))
    refused(lambda: K.linear_act_bwd(a, off[:0], "none", bias_dtype=torch.bfloat16))
    refused(lambda: K.linear_wgrad(a, r, off[:0]))
    refused(lambda: K.linear_wgrad(a, r, off[:1]))
    refused(lambda: K.grouped_linear_bwd(r, None, None, off, "none", need_a=False, need_w=False))
    refused(lambda: K.grouped_linear_bwd(r, None, w, off, "none"))
    refused(lambda: K.grouped_linear_bwd(r, a, None, off, "none"))
    refused(lambda: K.grouped_linear(a, w, off, out=a))
    refused(lambda: K.grouped_linear(both[:12], w, off, out=both[6:]))
    refused(lambda: K.grouped_linear(a, w, off, None, "none", both[:12], out=both[6:]))
    refused(lambda: K.grouped_linear(a, w, off, None, "relu", r, preact=r))
    refused(lambda: K.grouped_linear(a, w, off, None, "relu", out=r, preact=r))
    refused(lambda: K.grouped_linear(a, w, off, None, "relu", preact=a))
    neighbours = n(24, 16)
    out = K.grouped_linear(a, w, off, None, "relu", out=neighbours[:12], preact=neighbours[12:])
    assert torch.equal(out, S.grouped_linear(a, w, off, activation="relu"))
