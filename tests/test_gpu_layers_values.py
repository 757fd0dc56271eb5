"""Values of the sequence-block operators far out: activations and gates from 20 to infinity on either side, GELU's tail.

Below 2^-126 an exponential may be 0: its value times a factor of at most 128 is then off by 2^-119 at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LOST = 2.0 ** -119
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
FAR = [20.0, 50.0, 87.0, 87.5, 88.0, 88.5, 90.0, 104.0, 200.0, 1e4, 6e4, 1e19, 3e19, 1e20, 1e30, 1e35, 3e38, float("inf")]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def act_limits(p, act, slope):
    """act and act' in 64 bits; at -inf (and +inf) their limits."""
    if act == "leaky":
        return torch.where(p > 0, p, 0.0 * p.sign() if slope == 0 else slope * p), torch.where(p > 0, 1.0, slope).double()
    q = p.clamp(-1e300, 1e300)  # (a limit: what multiplies the vanishing factor is finite)
    s, c = torch.sigmoid(q), torch.special.ndtr(q)
    if act == "sigmoid":
        return s, s * torch.sigmoid(-q)
    if act == "silu":
        return torch.where(p == float("inf"), p, q * s), s * (1 + q * torch.sigmoid(-q))
    return torch.where(p == float("inf"), p, q * c), c + q * torch.exp(-(q.clamp(-1e3, 1e3)) ** 2 / 2) * 0.3989422804014327


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act,slope", [("leaky", 0.0), ("leaky", 0.25), ("sigmoid", 0.0), ("gelu", 0.0), ("silu", 0.0)])
@pytest.mark.parametrize("rows", [40, 700])
def test_activations_far_out(act, slope, dtype, rows):
    """Through the form of few rows and through tiles.  One product a value: p is the input itself.  A sigmoid's exponent loses |p| U for
    16-bit results; act' sees p as it is kept (2^-11 of it for bf16), which moves it by |p act''| 2^-11, |act''| <= 2 |act'| out here."""
    from vae_amd import layers
    x = torch.tensor(FAR + [-v for v in FAR] + [float("nan")], dtype=torch.float64).to(dtype).cuda()
    x = x.repeat(-(-rows // len(x)))[:rows, None].contiguous().requires_grad_()
    y = layers.linear(x, torch.ones(1, 1, dtype=dtype, device="cuda"), act=act, slope=slope)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    p = x.detach().double()
    v, d = act_limits(p, act, slope)
    nan = p.isnan()
    assert (y.isnan() == nan).all(), p[y.isnan() != nan]
    assert not dx[~nan].isnan().any(), p[dx.isnan() & ~nan]
    fine = ~nan & v.isfinite()
    assert (y.double()[~nan & ~fine] == v[~nan & ~fine]).all()
    near = p.abs().clamp(max=128)
    tol = (half(dtype) + 32 * U + 2 * near * U) * v.abs() + LOST + smallest(dtype)
    assert ((y.double() - v).abs() <= tol)[fine].all(), p[fine & ~((y.double() - v).abs() <= tol)]
    tol = (half(dtype) + 32 * U + near * 2.0 ** -9) * d.abs() + LOST + smallest(dtype)
    if act == "leaky":
        tol = half(dtype) * d.abs()
    assert ((dx.double() - d).abs() <= tol)[~nan].all(), p[~nan & ~((dx.double() - d).abs() <= tol)]


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


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [1, 3000])
def test_gelu_to_its_tail(dtype, rows):
    """GELU and its derivative relative to their values, down to 1e-36.  fp32: exp and its correction lose 3 U, 1 / (1 + c |p|) 3 U, eight steps of
    the polynomial 3 U, the products 3 U, its fit 0.2 U: 13 U, and a half step of the result.  For 16-bit results exp loses p^2 U more,
    170 U at p = -13; their derivative sees p as it is kept (2^-11 of it for bf16, |act''| <= 0.8 + p^2 phi)."""
    from vae_amd import layers
    x = torch.linspace(-13, 13, 3000, dtype=torch.float64).to(dtype).cuda()
    w = torch.ones(1, 1, dtype=dtype, device="cuda")
    if rows == 1:  # (the form of one row: a product of one value each, the weights carry the points)
        got = layers.linear(torch.ones(1, 1, dtype=dtype, device="cuda"), x[:, None].contiguous(), act="gelu")[0]
        dx = None
    else:
        xg = x[:, None].clone().requires_grad_()
        y = layers.linear(xg, w, act="gelu")
        got = y.detach()[:, 0]
        dx = torch.autograd.grad(y, xg, torch.ones_like(y))[0][:, 0]
    p = x.double()  # (torch.special.ndtr is (1 + erf) / 2, which loses the tail)
    cdf, pdf = 0.5 * torch.special.erfc(-p * 0.5 ** 0.5), torch.exp(-p * p / 2) * 0.3989422804014327
    v = p * cdf
    off = 13 * U if dtype == torch.float32 else (13 + p * p) * U
    err = (got.double() - v).abs()
    assert (err <= (half(dtype) + off) * v.abs() + LOST + smallest(dtype)).all(), float((err / v.abs().clamp(min=1e-30)).max())
    if dx is not None:
        d = cdf + p * pdf
        kept = 2.0 ** -11 * p.abs() * (2 * pdf + p * p * pdf) if dtype == torch.bfloat16 else 0.0
        err = (dx.double() - d).abs()
        assert (err <= half(dtype) * d.abs() + (off + 2 * U) * (cdf + p.abs() * pdf) + kept + LOST + smallest(dtype)).all(), float(err.max())


def test_sigmoid_to_a_unit():
    """fp32.  exp(-|g|) = e is off by 2.2 U (2^t by a unit in the last place, its correction 0.2 U): 1 / (1 + e) by half of that at most and its
    own rounding of U, the product e / (1 + e) by all of it and two roundings."""
    from vae_amd import layers
    g = torch.linspace(-30, 30, 1000001, dtype=torch.float64).float().cuda()
    y = layers.linear(g[:, None].contiguous(), torch.ones(1, 1, device="cuda"), act="sigmoid")[:, 0]
    want = torch.sigmoid(g.double())
    off = (y.double() - want).abs() / want / U
    assert off[g >= 0].max() <= 2.1, float(off[g >= 0].max())
    assert off[g < 0].max() <= 4.2, float(off[g < 0].max())
