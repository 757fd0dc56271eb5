"""Values of the sequence-block operators far out: gates from 200 to infinity on either side."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("gate", [200.0, 1e4, 6e4, float("inf")])
@pytest.mark.parametrize("t", [1, 70])
def test_gates_far_out_are_0_and_1(gate, dtype, t):
    """An open gate keeps the state, a closed one takes the input, whatever the other one holds (1e38 here): to the bit."""
    from vae_amd import layers
    g = torch.Generator().manual_seed(t)
    B, D = 3, 12
    x = torch.randn(B, t, D, generator=g).to(dtype).cuda().requires_grad_()
    h0 = (torch.randn(B, D, generator=g) * 1e38).cuda().requires_grad_()
    dy, dh = torch.randn(B, t, D, generator=g).to(dtype).cuda(), torch.randn(B, D, generator=g).cuda()
    shut = torch.full_like(x, -gate).requires_grad_()
    y, h = layers.gated_scan(x, shut, h0)
    assert torch.equal(y, x) and torch.equal(h, x[:, -1].float())
    dx, dg, dh0 = torch.autograd.grad([y, h], [x, shut, h0], [dy, dh])
    want = dy.float()
    want[:, -1] += dh
    assert torch.equal(dx, want.to(dtype)) and (dg == 0).all() and (dh0 == 0).all()
    keep = torch.full_like(x, gate).requires_grad_()
    s = torch.randn(B, D, generator=g).cuda().requires_grad_()
    big = (torch.randn(B, t, D, generator=g) * (1e38 if dtype != torch.float16 else 6e4)).to(dtype).cuda().requires_grad_()
    y, h = layers.gated_scan(big, keep, s)
    # (some of these values are infinite in fp16: 0 times infinity is a NaN, which the state then keeps)
    lost = big.detach().isinf().cumsum(1) > 0
    held = torch.where(lost, float("nan"), s.detach()[:, None])
    assert torch.allclose(y.float(), held.to(dtype).float(), rtol=0, atol=0, equal_nan=True)
    assert torch.allclose(h, held[:, -1], rtol=0, atol=0, equal_nan=True)
    dx, dg = torch.autograd.grad([y, h], [big, keep], [dy, dh])
    assert (dx == 0).all() and (dg[~lost] == 0).all() and dg[lost].isnan().all()
