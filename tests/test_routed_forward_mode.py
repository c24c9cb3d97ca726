"""The routed-row operators have reverse-mode gradients only; forward-mode tangents are refused
before anything runs, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import swiftmoe_b200 as S
from swiftmoe_b200._lib import SwiftMoEError


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(device, grad):
    x = torch.randn((6, 32), device=device).bfloat16()
    idx = torch.zeros((6, 2), dtype=torch.int32, device=device)
    w = torch.rand((6, 2), device=device)
    rows = torch.randn((12, 32), device=device).bfloat16()
    off = torch.tensor([0, 12], dtype=torch.int32, device=device)
    plan = dict(slot_row=torch.arange(12, dtype=torch.int32, device=device), offsets=off, rows_cap=12, T=6, k=2, row_align=1)
    wt = torch.randn((1, 32, 32), device=device).bfloat16()
    b, r = torch.zeros((1, 32), device=device), torch.zeros_like(rows)

    def dual(t):
        return fwd.make_dual(t, torch.ones_like(t))

    with fwd.dual_level(), torch.set_grad_enabled(grad):
        for call in (lambda: S.sort_tokens(dual(x), idx, 1), lambda: S.sort_tokens(x, idx, 1, weights=dual(w)),
                     lambda: S.unsort_tokens(dual(rows), plan), lambda: S.unsort_tokens(rows, plan, dual(w)),
                     lambda: S.unsort_tokens(rows, plan, residual=dual(x)), lambda: S.grouped_linear(dual(rows), wt, off),
                     lambda: S.grouped_linear(rows, dual(wt), off), lambda: S.grouped_linear(rows, wt, off, bias=dual(b)),
                     lambda: S.grouped_linear(rows, wt, off, residual=dual(r))):
            with pytest.raises(SwiftMoEError, match="forward-mode"):
                call()
        if device == "cuda":   # without a tangent they are served
            assert S.sort_tokens(x, idx, 1)[0].shape == rows.shape
            assert S.unsort_tokens(rows, plan, w, x).shape == x.shape
            assert S.grouped_linear(rows, wt, off, b, "silu", r).shape == rows.shape


def test_function_transforms_are_refused():
    x, idx = torch.randn(6, 32), torch.zeros((6, 2), dtype=torch.int32)
    with pytest.raises(SwiftMoEError, match="forward-mode"):
        torch.func.jvp(lambda t: S.sort_tokens(t, idx, 1)[0], (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: S.sort_tokens(t, idx, 1)[0].sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: S.sort_tokens(t, idx, 1)[0])(x.unsqueeze(0))
