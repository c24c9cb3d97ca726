"""Tokens with more slots than a row has 16-byte pieces (k > d * size / 16)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,d,k", [(33, 72, 32), (9, 8, 2), (70, 32, 8)])
def test_combine(dtype, T, d, k):
    from swiftmoe_b200 import kernels as K
    g = torch.Generator(device="cuda").manual_seed(T)
    y = torch.randn((T * k, d), generator=g, device="cuda").to(dtype)
    slot_row = torch.randperm(T * k, generator=g, device="cuda").to(torch.int32)
    w = torch.rand((T, k), generator=g, device="cuda")
    out = K.combine(y, slot_row, w, T, k)
    terms = y.double()[slot_row.long()].view(T, k, d) * w.double().unsqueeze(2)
    bound = torch.finfo(dtype).eps / 2 * terms.sum(1).abs() * 1.001 + 2 * k * 2.0 ** -24 * terms.abs().sum(1)
    assert ((out.double() - terms.sum(1)).abs() <= bound).all()


def test_layer_fused_as_staged():
    import swiftmoe_b200 as S
    torch.manual_seed(3)
    m = S.UltimateMoE(8, 32, use_fp16=False, dtype=torch.bfloat16, top_k=8, use_nccl_opt=False, device="cuda")
    x = torch.randn(50, 32, device="cuda").bfloat16()
    fused = m(x)
    m._force_staged = True      # permutes row by row
    assert torch.equal(fused, m(x))
