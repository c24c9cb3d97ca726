"""Edges of sort_tokens, unsort_tokens and grouped_linear: pre-activations past the 16-bit
range."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.autograd]

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(scope="module")
def S():
    import swiftmoe_b200
    return swiftmoe_b200


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


# -------------------------------------------------------------------------- activations
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
