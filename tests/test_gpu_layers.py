"""Layer norm, linear and gated scan (vae_amd.layers) against plain implementations in 64 bits.

Tolerances count roundings: U = 2^-24 is half a step of fp32, `half(dtype)` half a step of the output's type.  An output is off by
at most half(dtype) |value| for its own rounding plus what the fp32 arithmetic before it loses; the latter is bounded next to each
check from the 64-bit values of the terms that are added."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # half a step of the subnormals is below this


def rnd(shape, dtype, seed, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + mean).to(dtype).cuda()


def check(name, got, want, tol):
    """|got - want| <= half a step of got's type at `want` + tol, where tol bounds the fp32 error before the rounding."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    g, w = got.double(), want.double()
    allowed = half(got.dtype) * (w.abs() + tol) + tol + smallest(got.dtype)
    bad = ~((g - w).abs() <= allowed)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((g - w).abs().max()):.3e} "
                           f"(allowed there {float(allowed.flatten()[(g - w).abs().flatten().argmax()]):.3e})")


# ------------------------------------------------------------------------------------------------ layer norm
def norm64(x, w, b, dy, eps):
    """Values, and bounds of the fp32 error: a sum of C terms in registers, lane shuffles and LDS adds each term at most
    C/lanes + 20 times <= depth; (x - mean) carries the mean's error and one rounding, rstd the variance's."""
    x = x.double()
    C = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xhat = (x - mean) * rstd
    w_ = w.double() if w is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    b_ = b.double() if b is not None else torch.zeros(C, dtype=torch.float64, device=x.device)
    y = xhat * w_ + b_
    depth = 90
    e_mean = depth * U * x.abs().mean(-1, keepdim=True)
    e_c = e_mean + U * (x.abs() + mean.abs())  # of x - mean
    # relative error of rstd: half of the variance's, whose terms are off by 2 |x - mean| e_c each
    e_rstd = 0.5 * ((2 * (x - mean).abs() * e_c).mean(-1, keepdim=True) / (var + eps)) + (depth + 4) * U
    e_xhat = e_c * rstd + xhat.abs() * (e_rstd + 2 * U)
    e_y = e_xhat * w_.abs() + 2 * U * ((xhat * w_).abs() + b_.abs())
    out = {"y": (y, e_y)}
    if dy is not None:
        dy = dy.double()
        g = dy * w_
        c1, c2 = g.mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True)
        t = g - c1 - xhat * c2
        e_c1 = (depth + 2) * U * g.abs().mean(-1, keepdim=True)
        e_c2 = (depth + 3) * U * (g * xhat).abs().mean(-1, keepdim=True) + (g.abs() * e_xhat).mean(-1, keepdim=True)
        e_t = U * g.abs() + e_c1 + xhat.abs() * e_c2 + e_xhat * c2.abs() + 3 * U * (g.abs() + c1.abs() + (xhat * c2).abs())
        out["dx"] = (rstd * t, rstd * (e_t + t.abs() * (e_rstd + 2 * U)))
        rows = x.numel() // C
        # a lane adds at most rows / 1 terms in turn; partials join in at most 80 more steps
        n = rows + 80
        out["dw"] = ((dy * xhat).reshape(-1, C).sum(0), (n * U * (dy * xhat).abs() + dy.abs() * e_xhat).reshape(-1, C).sum(0))
        out["db"] = (dy.reshape(-1, C).sum(0), n * U * dy.abs().reshape(-1, C).sum(0))
    return out


def run_norm(x, w, b, dy, eps=1e-5):
    from vae_amd import layers
    x = x.detach().requires_grad_()
    leaves = [x] + [t.detach().requires_grad_() for t in (w, b) if t is not None]
    y = layers.layer_norm(x, leaves[1] if w is not None else None, leaves[-1] if b is not None else None, eps)
    grads = torch.autograd.grad(y, leaves, dy)
    out = {"y": y.detach(), "dx": grads[0]}
    if w is not None:
        out["dw"] = grads[1]
    if b is not None:
        out["db"] = grads[-1]
    return out


NORM_SIZES = [(1, 1), (1, 7), (3, 8), (5, 30), (300, 63), (17, 64), (9, 65), (33, 129), (7, 257), (130, 512), (6, 1000), (5, 1025),
              (4100, 100), (3, 2049), (2, 4100), (1500, 1024), (3, 8195), (2, 16385), (2, 33001), (1, 70000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_norm_values_and_gradients(rows, cols, dtype):
    x, dy = rnd((rows, cols), dtype, 1, 1.5, 0.3), rnd((rows, cols), dtype, 2)
    for wd in {torch.float32, dtype}:
        w, b = rnd(cols, wd, 3, 0.2, 1.0), rnd(cols, wd, 4, 0.1)
        got, want = run_norm(x, w, b, dy), norm64(x, w, b, dy, 1e-5)
        for k, (v, tol) in want.items():
            check(k, got[k], v, tol)


@pytest.mark.parametrize("rows,cols", [(600, 8200), (4, 12288), (300, 12291), (3, 16384), (300, 18801), (300, 18838), (300, 18843)])
def test_norm_rows_of_a_whole_workgroup(rows, cols):
    x, dy = rnd((rows, cols), torch.float32, 1, 1.5, 0.3), rnd((rows, cols), torch.float32, 2)
    w, b = rnd(cols, torch.float32, 3, 0.2, 1.0), rnd(cols, torch.float32, 4, 0.1)
    got, want = run_norm(x, w, b, dy), norm64(x, w, b, dy, 1e-5)
    for k, (v, tol) in want.items():
        check(k, got[k], v, tol)


@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_norm_without_parameters(has_w, has_b):
    x, dy = rnd((37, 200), torch.bfloat16, 1), rnd((37, 200), torch.bfloat16, 2)
    w = rnd(200, torch.float32, 3, 0.2, 1.0) if has_w else None
    b = rnd(200, torch.float32, 4) if has_b else None
    got, want = run_norm(x, w, b, dy), norm64(x, w, b, dy, 1e-5)
    for k in got:
        check(k, got[k], *want[k])


def test_norm_strided_rows_and_leading_dims():
    from vae_amd import layers
    base = rnd((4, 6, 90), torch.float32, 5)
    w, b = rnd(40, torch.float32, 3), rnd(40, torch.float32, 4)
    for x in (base[..., 7:47], base[:, ::2, 7:47], base.transpose(0, 1)[..., 1:41], base[:, :1, 3:43].expand(4, 6, 40),
              base.permute(1, 2, 0)[:, :40, :].transpose(1, 2)):
        want = norm64(x, w, b, None, 1e-5)["y"]
        check("y", layers.layer_norm(x, w, b), *want)
        dy = rnd(x.shape[:-1] + (80,), torch.float32, 6)[..., ::2]  # a gradient whose columns are strided
        xg = x.detach().clone().requires_grad_()
        (dx,) = torch.autograd.grad(layers.layer_norm(xg, w, b), xg, dy)
        check("dx", dx, *norm64(x, w, b, dy, 1e-5)["dx"])


def test_norm_constant_and_far_rows():
    """Variance 0 (rstd = 1/sqrt(eps)), a mean 1000 times the deviation, and values at 1e4."""
    x = torch.cat([torch.full((1, 256), 3.25), 1000 + torch.randn(3, 256, generator=torch.Generator().manual_seed(1)),
                   1e4 * torch.randn(2, 256, generator=torch.Generator().manual_seed(2))]).cuda()
    dy, w, b = rnd(x.shape, torch.float32, 2), rnd(256, torch.float32, 3), rnd(256, torch.float32, 4)
    got, want = run_norm(x, w, b, dy), norm64(x, w, b, dy, 1e-5)
    for k, (v, tol) in want.items():
        check(k, got[k], v, tol)


def test_norm_a_nan_row_stays_a_row():
    from vae_amd import layers
    for cols in (20, 700, 9000):
        x = rnd((9, cols), torch.float32, 1)
        clean = layers.layer_norm(x)
        x[4, cols // 2] = float("nan")
        y = layers.layer_norm(x)
        assert y[4].isnan().all()
        keep = [i for i in range(9) if i != 4]
        assert torch.equal(y[keep], clean[keep])


def test_norm_rows_behind_the_last_stay_as_they_were():
    """Rows and columns around a strided output region are not written (through the C entry)."""
    from vae_amd import _lib as L
    x = rnd((7, 50), torch.float32, 1)
    out = torch.full((9, 60), -7.0, device="cuda")
    L.check(L.lib().vae_layer_norm_forward(x.data_ptr(), 50, None, None, out.data_ptr(), 60, None, None, 7, 50, 1e-5, 0, 0,
                                           torch.cuda.current_stream().cuda_stream), "forward")
    check("y", out[:7, :50], *norm64(x, None, None, None, 1e-5)["y"])
    assert (out[7:] == -7).all() and (out[:, 50:] == -7).all()


def test_norm_only_the_gradients_asked_for():
    from vae_amd import layers
    x, dy = rnd((40, 96), torch.float32, 1), rnd((40, 96), torch.float32, 2)
    w, b = rnd(96, torch.float32, 3), rnd(96, torch.float32, 4)
    want = norm64(x, w, b, dy, 1e-5)
    for pick in ("x", "w", "b"):
        t = {"x": x.clone(), "w": w.clone(), "b": b.clone()}
        t[pick].requires_grad_()
        y = layers.layer_norm(t["x"], t["w"], t["b"])
        (g,) = torch.autograd.grad(y, t[pick], dy)
        check(pick, g, *want["d" + pick])


# ---------------------------------------------------------------------------------------------------- linear
SLOPE = 0.2
CURVE = {"none": 0.0, "leaky": 0.0, "sigmoid": 0.1, "gelu": 0.8, "silu": 0.5}  # max |act''|


def act64(p, act):
    if act == "leaky":
        return torch.where(p > 0, p, SLOPE * p), torch.where(p > 0, 1.0, SLOPE).double()
    if act == "sigmoid":
        s = torch.sigmoid(p)
        return s, s * torch.sigmoid(-p)
    if act == "gelu":
        c = torch.special.ndtr(p)
        return p * c, c + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(p)
        return p * s, s * (1 + p * torch.sigmoid(-p))
    return p, torch.ones_like(p)


def linear64(x, w, b, r, dy, act):
    """Values and bounds.  A sum of K products of the operands (exact in fp32 for 16-bit operands, one rounding for fp32) loses at
    most (K + 8) U of the sum of their magnitudes in whatever order it is added.  dp is rounded to the operands' type before
    its two products; p, which act' is taken at, is kept in fp16 for bf16 tensors (2^-11), in fp32 otherwise."""
    dt = x.dtype
    x, w = x.double().reshape(-1, x.shape[-1]), w.double()
    K, N = x.shape[1], w.shape[0]
    p, mag = x @ w.t(), x.abs() @ w.abs().t()
    e_p = (K + 8) * U * mag
    if b is not None:
        p = p + b.double()
        e_p = e_p + U * (p.abs() + b.double().abs())
    y, d = act64(p, act)
    e_y = (1.2 if act != "none" else 1.0) * e_p + 16 * U * (y.abs() + (act == "gelu") * p.abs())
    if r is not None:
        r = r.double().reshape(-1, N)
        y = y + r
        e_y = e_y + U * (y.abs() + r.abs())
    out = {"y": (y, e_y)}
    if dy is not None:
        dy = dy.double().reshape(-1, N)
        dp = dy * d
        kept = 2.0 ** -11 if dt == torch.bfloat16 else U
        e_d = 0 if act in ("none", "leaky") else CURVE[act] * (kept * p.abs() + e_p + 2.0 ** -24) + 16 * U
        e_dp = dy.abs() * e_d + (2 * U * dp.abs() if act != "none" else 0)
        if act == "leaky":  # p within its error of 0 may fall on either side
            e_dp = e_dp + torch.where(p.abs() <= e_p, dy.abs() * (1 - SLOPE), 0.0)
        r_dp = (half(dt) * dp.abs() + smallest(dt)) if (act != "none" and dt != torch.float32) else 0.0
        e_op = e_dp + r_dp
        M = x.shape[0]
        out["dx"] = (dp @ w, (N + 8) * U * (dp.abs() @ w.abs()) + (e_op @ w.abs() if act != "none" else 0))
        out["dw"] = (dp.t() @ x, (M + 8) * U * (dp.abs().t() @ x.abs()) + (e_op.t() @ x.abs() if act != "none" else 0))
        if b is not None:
            out["db"] = (dp.sum(0), (M + 8) * U * dp.abs().sum(0) + (e_dp.sum(0) if act != "none" else 0))
    return out


def run_linear(x, w, b, r, dy, act):
    from vae_amd import layers
    t = {"x": x, "w": w, "b": b, "r": r}
    t = {k: v.detach().requires_grad_() for k, v in t.items() if v is not None}
    y = layers.linear(t["x"], t["w"], t.get("b"), act=act, slope=SLOPE, residual=t.get("r"))
    grads = torch.autograd.grad(y, list(t.values()), dy)
    out = {"y": y.detach().reshape(-1, w.shape[0])}
    for k, g in zip(t, grads):
        out["d" + k] = g.reshape(-1, g.shape[-1]) if k in "xr" else g
    if r is not None:
        assert torch.equal(out.pop("dr"), dy.reshape(-1, w.shape[0]))
    return out


def linear_case(m, n, k, dtype, act, bias=True, residual=True):
    x, w = rnd((m, k), dtype, 1), rnd((n, k), dtype, 2, k ** -0.5)
    b = rnd((n,), dtype, 3, 0.3) if bias else None
    r = rnd((m, n), dtype, 4) if residual else None
    dy = rnd((m, n), dtype, 5)
    got, want = run_linear(x, w, b, r, dy, act), linear64(x, w, b, r, dy, act)
    for key, (v, tol) in want.items():
        check(key, got[key], v, tol)


LINEAR_SIZES = [(1, 1, 1), (1, 100, 288), (2, 16, 64), (3, 5, 7), (16, 512, 512), (17, 33, 65), (33, 40, 1000), (64, 64, 64), (65, 129, 31),
                (130, 260, 200), (257, 96, 1000), (1000, 30, 30), (5000, 100, 288)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", LINEAR_SIZES)
def test_linear_values_and_gradients(m, n, k, dtype):
    linear_case(m, n, k, dtype, "gelu")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ["none", "leaky", "sigmoid", "silu"])
@pytest.mark.parametrize("m", [1, 70])
def test_linear_activations(act, dtype, m):
    linear_case(m, 72, 136, dtype, act)
    linear_case(m, 37, 41, dtype, act, bias=False, residual=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(2050, 2056, 200), (4096, 1024, 520), (2047, 2049, 131)])
def test_linear_large_tiles(m, n, k, dtype):
    linear_case(m, n, k, dtype, "silu")
    linear_case(m, n, k, dtype, "none", bias=True, residual=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(4100, 2568, 264), (4100, 264, 2568), (264, 4104, 2568)])
def test_linear_largest_tiles(m, n, k, dtype):
    """Forward, dx and dW in turn are the product of many outputs."""
    linear_case(m, n, k, dtype, "silu")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(100, 70, 4000), (65, 1, 2001), (100, 4000, 70), (70, 4000, 4001), (300, 500, 8000), (2000, 1030, 2048)])
@pytest.mark.parametrize("act", ["leaky", "gelu"])
def test_linear_few_outputs_of_long_sums(m, n, k, dtype, act):
    """Sums of thousands of terms for few outputs: split over k."""
    linear_case(m, n, k, dtype, act)
    linear_case(m, n, k, dtype, "none", bias=False, residual=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(4100, 2571, 2051), (4100, 2571, 2048), (4100, 2568, 2051), (2051, 4103, 2565)])
def test_linear_large_and_ragged(m, n, k, dtype):
    """Rows that are no whole 16-byte pieces, large enough to be laid out anew for the products."""
    linear_case(m, n, k, dtype, "silu")
    linear_case(m, n, k, dtype, "none", bias=False, residual=False)
    x, w = rnd((m, k), dtype, 1).requires_grad_(), rnd((n, k), dtype, 2, k ** -0.5).requires_grad_()
    from vae_amd import layers
    dy = rnd((m, n), dtype, 5)
    want = linear64(x.detach(), w.detach(), None, None, dy, "none")
    for leaf, name in ((x, "dx"), (w, "dw")):  # one gradient at a time
        got, = torch.autograd.grad(layers.linear(x, w), leaf, dy)
        check(name, got, *want[name])


def test_linear_strides():
    from vae_amd import layers
    for dtype in DTYPES:
        xb, wb, rb = rnd((5, 9, 200), dtype, 1), rnd((50, 120), dtype, 2, 0.1), rnd((5, 9, 77), dtype, 4)
        for x, w, r in ((xb[..., 3:99], wb[:, 5:101], rb[..., 1:51]), (xb[:, ::2, :96], wb[::2, :96], rb[:, ::2, 1:26]),
                        (xb.transpose(0, 1)[..., 8:104], wb[:, :96], rb.transpose(0, 1)[..., :50])):
            want = linear64(x, w, None, r, None, "silu")["y"]
            check("y", layers.linear(x, w, act="silu", residual=r).reshape(want[0].shape), *want)
            dy = rnd(r.shape[:-1] + (2 * r.shape[-1],), dtype, 6)[..., ::2]
            xg, wg = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
            dx, dw = torch.autograd.grad(layers.linear(xg, wg, act="silu", residual=r), [xg, wg], dy)
            want = linear64(x, w, None, r, dy, "silu")
            check("dx", dx.reshape(-1, 96), *want["dx"])
            check("dw", dw, *want["dw"])


def test_linear_transposed_weight_and_empty_batch():
    from vae_amd import layers
    x, w = rnd((10, 24), torch.float32, 1), rnd((24, 12), torch.float32, 2)
    check("y", layers.linear(x, w.t()), *linear64(x, w.t(), None, None, None, "none")["y"])
    e = torch.empty(0, 24, device="cuda", requires_grad=True)
    wg = w.t().contiguous().requires_grad_()
    y = layers.linear(e, wg)
    assert y.shape == (0, 12)
    de, dw = torch.autograd.grad(y, [e, wg], torch.empty(0, 12, device="cuda"))
    assert de.shape == (0, 24) and (dw == 0).all()


def test_linear_far_values_and_nan_rows():
    """act and act' far out in their tails are finite; a NaN row leaves the others as they were."""
    from vae_amd import layers
    for dtype in DTYPES:
        for act in ("sigmoid", "gelu", "silu"):
            x = torch.tensor([[-1e4], [-200.0], [-90.0], [-20.0], [0.0], [20.0], [90.0], [200.0], [1e4]], dtype=dtype, device="cuda").requires_grad_()
            w = torch.ones(1, 1, dtype=dtype, device="cuda")
            y = layers.linear(x, w, act=act)
            (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
            p = x.detach().double()
            v, d = act64(p, act)
            check(act, y.detach(), v, 32 * U * v.abs() + 1e-30)
            check(act + "'", dx, d, half(dtype) * d.abs() + 32 * U * d.abs() + (2.0 ** -11) * p.abs() * d.abs() + 1e-7)
        x = rnd((40, 64), dtype, 1)
        w = rnd((48, 64), dtype, 2)
        clean = layers.linear(x, w, act="silu")
        x[11, 5] = float("nan")
        y = layers.linear(x, w, act="silu")
        assert y[11].isnan().all()
        keep = [i for i in range(40) if i != 11]
        assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("view", [lambda t: t[:, -1:], lambda t: t[:, -1], lambda t: t[:, 2:5], lambda t: t[:, ::3], lambda t: t[1:2, 3:4], lambda t: t[:, :, :40],
                                  lambda t: t[:, None, 1], lambda t: t.transpose(0, 1), lambda t: t[..., ::2], lambda t: t[:1].expand(5, -1, -1)])
def test_views_of_windows_equal_their_copies(view):
    """Steps taken out of windows go in as they lie; values and gradients are those of a copy."""
    from vae_amd import layers
    base = rnd((6, 11, 48), torch.bfloat16, 1)
    x = view(base)
    w, nw = rnd((24, x.shape[-1]), torch.bfloat16, 2), rnd(x.shape[-1], torch.float32, 3)
    res = []
    for t in (x, x.clone(memory_format=torch.contiguous_format)):
        t = t.detach().requires_grad_()
        y, z = layers.linear(t, w, act="silu"), layers.layer_norm(t, nw)
        res.append([y.detach(), z.detach(), *torch.autograd.grad(y, t, torch.ones_like(y)), *torch.autograd.grad(z, t, view(rnd(base.shape, torch.bfloat16, 4)))])
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_linear_one_row_of_any_stride():
    """Through the C entry: the strides of a single row say nothing, 0 among them.  Products of two bf16 values are exact in fp32, so
    dW is its own rounding; dx: a sum of n terms."""
    from vae_amd import _lib as L
    n = k = 2048
    x, dy, w = (rnd(s, torch.bfloat16, 70 + i) for i, s in enumerate(((1, k), (1, n), (n, k))))
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    lib = L.lib()
    ws = torch.empty(lib.vae_dense_workspace_floats(1, n, k, L.ACT_NONE, L.T_BF16), device="cuda")
    L.check(lib.vae_dense_backward(dy.data_ptr(), 0, x.data_ptr(), 0, w.data_ptr(), k, None, dx.data_ptr(), dw.data_ptr(), None,
                                   ws.data_ptr(), 1, n, k, L.ACT_NONE, 0.0, L.T_BF16, L.stream_ptr()), "vae_dense_backward")
    assert torch.equal(dw, (dy.float().t() * x.float()).bfloat16())
    terms = dy.double().t() * w.double()
    check("dx", dx, terms.sum(0, keepdim=True), n * U * terms.abs().sum(0, keepdim=True))


def test_linear_only_the_gradients_asked_for():
    from vae_amd import layers
    x, w, b, dy = rnd((40, 96), torch.float32, 1), rnd((32, 96), torch.float32, 2), rnd((32,), torch.float32, 3), rnd((40, 32), torch.float32, 5)
    for act in ("none", "gelu"):
        want = linear64(x, w, b, None, dy, act)
        for pick in "xwb":
            t = {"x": x.clone(), "w": w.clone(), "b": b.clone()}
            t[pick].requires_grad_()
            (g,) = torch.autograd.grad(layers.linear(t["x"], t["w"], t["b"], act=act), t[pick], dy)
            check(pick, g, *want["d" + pick])


# ------------------------------------------------------------------------------------------------ gated scan
def scan64(x, gate, h0, lengths, dy, dhl):
    """Values and bounds, step by step.  sigmoid and its complement are off by at most 6 U each, a step adds 2 roundings, and joining
    tiles a product and a sum: 12 U of the step's magnitudes, carried along with the state's own factors."""
    B, T, D = x.shape
    x, gate = x.double(), gate.double()
    f, i = torch.sigmoid(gate), torch.sigmoid(-gate)
    live = torch.ones(B, T, 1, dtype=torch.bool, device=x.device)
    if lengths is not None:
        live = (torch.arange(T, device=x.device)[None] < lengths[:, None])[..., None]
        f, i = torch.where(live, f, 1.0), torch.where(live, i, 0.0)
        x = torch.where(live, x, 0.0)
    c = 12 * U
    h = h0.double() if h0 is not None else torch.zeros(B, D, dtype=torch.float64, device=x.device)
    m, e = h.abs(), torch.zeros_like(h)
    hs, ms, es = [h], [m], [e]
    for t in range(T):
        h = f[:, t] * h + i[:, t] * x[:, t]
        e = f[:, t] * e + c * live[:, t] * (f[:, t] * m + i[:, t] * x[:, t].abs())
        m = f[:, t] * m + i[:, t] * x[:, t].abs()
        hs.append(h), ms.append(m), es.append(e)
    stack = lambda v: torch.stack(v, 1)  # noqa: E731
    out = {"y": (torch.where(live, stack(hs[1:]), 0.0), torch.where(live, stack(es[1:]), 0.0)), "h": (h, e)}
    if dy is None and dhl is None:
        return out
    dy = torch.where(live, dy.double(), 0.0) if dy is not None else torch.zeros_like(x)
    q = dhl.double() if dhl is not None else torch.zeros(B, D, dtype=torch.float64, device=x.device)
    qm, qe = q.abs(), torch.zeros_like(q)
    dx, dg, ex, eg = [None] * T, [None] * T, [None] * T, [None] * T
    for t in range(T - 1, -1, -1):
        dh, dm = dy[:, t] + q, dy[:, t].abs() + qm
        de = qe + c * live[:, t] * dm
        dx[t], ex[t] = i[:, t] * dh, i[:, t] * (de + c * dm)
        diff = hs[t] - x[:, t]
        dg[t] = dh * diff * f[:, t] * i[:, t]
        eg[t] = f[:, t] * i[:, t] * (de * diff.abs() + dm * (es[t] + c * (ms[t] + x[:, t].abs())))
        q, qm = f[:, t] * dh, f[:, t] * dm
        qe = f[:, t] * de + c * live[:, t] * qm
    out.update(dx=(stack(dx), stack(ex)), dgate=(stack(dg), stack(eg)), dh0=(q, qe))
    return out


def run_scan(x, gate, h0, lengths, dy, dhl):
    from vae_amd import layers
    t = {"x": x, "gate": gate, "h0": h0}
    t = {k: v.detach().requires_grad_() for k, v in t.items() if v is not None}
    y, h = layers.gated_scan(t["x"], t["gate"], t.get("h0"), lengths=lengths)
    outs = [(o, g) for o, g in ((y, dy), (h, dhl)) if g is not None]
    out = {"y": y.detach(), "h": h.detach()}
    if outs:
        grads = torch.autograd.grad([o for o, _ in outs], list(t.values()), [g for _, g in outs])
        out.update({"d" + k: g for k, g in zip(t, grads)})
    return out


def scan_inputs(b, t, d, dtype, seed=0):
    return (rnd((b, t, d), dtype, seed + 1), rnd((b, t, d), dtype, seed + 2, 1.5, 2.0), rnd((b, d), torch.float32, seed + 3),
            rnd((b, t, d), dtype, seed + 4), rnd((b, d), torch.float32, seed + 5))


def scan_compare(got, want):
    for k in got:
        check(k, got[k], *want[k])


SCAN_SIZES = [(1, 1, 1), (3, 1, 130), (2, 2, 5), (2, 7, 30), (1, 8, 64), (2, 9, 64), (1, 16, 33), (3, 17, 8), (2, 33, 100), (5, 60, 30), (2, 63, 31),
              (1, 64, 129), (2, 65, 64), (1, 127, 7), (1, 128, 256), (2, 129, 40), (1, 300, 513), (1, 1500, 20), (300, 70, 300)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("b,t,d", SCAN_SIZES)
def test_scan_values_and_gradients(b, t, d, dtype):
    x, gate, h0, dy, dhl = scan_inputs(b, t, d, dtype)
    scan_compare(run_scan(x, gate, h0, None, dy, dhl), scan64(x, gate, h0, None, dy, dhl))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("t", [1, 5, 60, 64, 200, 700])
def test_scan_lengths_and_what_padding_holds(t, dtype):
    """Lengths 0, 1, in between and whole; NaN and infinities in the padding change nothing."""
    lengths = torch.tensor([0, 1, t, max(0, t - 1), t // 2, min(t, 8), min(t, 64)], dtype=torch.int32, device="cuda")
    x, gate, h0, dy, dhl = scan_inputs(7, t, 37, dtype)
    want = scan64(x, gate, h0, lengths, dy, dhl)
    dead = (torch.arange(t, device="cuda")[None] >= lengths[:, None])[..., None]
    for fill in (None, float("nan"), float("inf"), torch.finfo(dtype).min):
        if fill is not None:
            x, gate, dy = (torch.where(dead, torch.full_like(v, fill), v) for v in (x, gate, dy))
        got = run_scan(x, gate, h0, lengths, dy, dhl)
        scan_compare(got, want)
        for k in ("y", "dx", "dgate"):
            assert (got[k][dead.expand_as(got[k])] == 0).all(), k
    scan_compare(run_scan(x, gate, h0, lengths.long() + 0, dy, dhl), want)
    over = lengths.clone()
    over[2] = t + 100  # clamped to the number of steps
    over[0] = -5
    scan_compare(run_scan(x, gate, h0, over, dy, dhl), want)


def test_scan_without_state_and_single_outputs():
    x, gate, h0, dy, dhl = scan_inputs(3, 90, 50, torch.float32)
    scan_compare(run_scan(x, gate, None, None, dy, dhl), scan64(x, gate, None, None, dy, dhl))
    scan_compare(run_scan(x, gate, h0, None, None, dhl), scan64(x, gate, h0, None, None, dhl))
    scan_compare(run_scan(x, gate, h0, None, dy, None), scan64(x, gate, h0, None, dy, None))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_scan_long_with_few_channels(dtype):
    """The time axis over many workgroups; gates that forget slowly, so that a state reaches across them."""
    x, gate, h0, dy, dhl = scan_inputs(1, 9001, 24, dtype)
    gate = (gate.float() + 4).to(dtype)
    scan_compare(run_scan(x, gate, h0, None, dy, dhl), scan64(x, gate, h0, None, dy, dhl))
    lengths = torch.tensor([5000], dtype=torch.int32, device="cuda")
    scan_compare(run_scan(x, gate, h0, lengths, dy, dhl), scan64(x, gate, h0, lengths, dy, dhl))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("b, t, d", [(8, 600, 600), (9, 530, 1001)])
def test_scan_between_few_and_many_channels(b, t, d, dtype):
    """Channels for which the two passes cut the time axis differently."""
    x, gate, h0, dy, dhl = scan_inputs(b, t, d, dtype)
    scan_compare(run_scan(x, gate, h0, None, dy, dhl), scan64(x, gate, h0, None, dy, dhl))


def test_scan_strided_views():
    from vae_amd import layers
    for dtype in DTYPES:
        both = rnd((4, 70, 2 * 33 + 1), dtype, 1, 1.5, 1.0)
        x, gate = both[..., 1:34], both[..., 34:]
        want = scan64(x, gate, None, None, None, None)
        y, h = layers.gated_scan(x, gate)
        check("y", y, *want["y"])
        tb = rnd((70, 4, 33), dtype, 2)  # time first
        want = scan64(tb.transpose(0, 1), gate, None, None, None, None)
        check("y", layers.gated_scan(tb.transpose(0, 1), gate)[0], *want["y"])
        cl = rnd((4, 33, 70), dtype, 3)  # features strided, as a Conv1d leaves them
        want = scan64(cl.transpose(1, 2), gate, None, None, None, None)
        check("y", layers.gated_scan(cl.transpose(1, 2), gate)[0], *want["y"])
        dy = rnd((70, 4, 33), dtype, 4).transpose(0, 1)
        xg = x.detach().clone().requires_grad_()
        (dx,) = torch.autograd.grad(layers.gated_scan(xg, gate)[0], xg, dy)
        check("dx", dx, *scan64(x, gate, None, None, dy, None)["dx"])


def test_scan_saturated_gates():
    """Gates at +-200 and +-infinity: f and 1 - f are 0 or 1 and nothing becomes NaN."""
    for v in (200.0, float("inf")):
        x, gate, h0, dy, dhl = scan_inputs(2, 70, 12, torch.float32)
        gate = torch.where(rnd(gate.shape, torch.float32, 9) > 0, v, -v)
        got = run_scan(x, gate, h0, None, dy, dhl)
        want = scan64(x, gate.clamp(-200, 200), h0, None, dy, dhl)
        for k in got:
            check(k, got[k], want[k][0], want[k][1] + 1e-30)


def test_scan_steps_one_by_one_equal_the_whole():
    """A served model advances a step at a time: the fp32 state goes round, results are those of the whole window."""
    from vae_amd import layers
    x, gate, h0, _, _ = scan_inputs(3, 40, 65, torch.bfloat16)
    y, h = layers.gated_scan(x, gate, h0)
    s, ys = h0, []
    for t in range(40):
        o, s = layers.gated_scan(x[:, t:t + 1], gate[:, t:t + 1], s)
        ys.append(o)
    want = scan64(x, gate, h0, None, None, None)
    check("y", torch.cat(ys, 1), *want["y"])
    check("h", s, *want["h"])
    check("whole y", y, *want["y"])
    e = layers.gated_scan(x[:, :0], gate[:, :0], h0)
    assert e[0].shape == (3, 0, 65) and torch.equal(e[1], h0)


# ------------------------------------------------------------------------------------------- all of them
def test_gradients_against_differences():
    """The formulas' gradients against central differences of the 64-bit values: a loss over all three operators."""
    B, T, D = 2, 11, 8
    g = torch.Generator().manual_seed(0)
    p = [torch.randn(s, generator=g, dtype=torch.float64) * 0.5 for s in
         ((B, T, D), (D,), (D,), (2 * D, D), (2 * D,), (D, D), (D,), (B, D))]
    up, uh = torch.randn(B, T, D, generator=g, dtype=torch.float64), torch.randn(B, D, generator=g, dtype=torch.float64)

    def loss64(p):
        x, nw, nb, w1, b1, w2, b2, h0 = p
        u = torch.nn.functional.layer_norm(x, (D,), nw, nb, 1e-5)
        cg = u @ w1.t() + b1
        c, ga = cg[..., :D], cg[..., D:]
        h, hs = h0, []
        for t in range(T):
            f = torch.sigmoid(ga[:, t])
            h = f * h + (1 - f) * c[:, t]
            hs.append(h)
        y = act64(torch.stack(hs, 1) @ w2.t() + b2, "gelu")[0] + x
        return (y * up).sum() + (h * uh).sum()

    from vae_amd import layers
    t = [v.float().cuda().requires_grad_() for v in p]
    x, nw, nb, w1, b1, w2, b2, h0 = t
    cg = layers.linear(layers.layer_norm(x, nw, nb), w1, b1)
    y, h = layers.gated_scan(cg[..., :D], cg[..., D:], h0)
    y = layers.linear(y, w2, b2, act="gelu", residual=x)
    grads = torch.autograd.grad((y * up.float().cuda()).sum() + (h * uh.float().cuda()).sum(), t)
    step = 1e-5
    for v, got in zip(p, grads):
        flat = v.view(-1)
        idx = torch.arange(0, flat.numel(), max(1, flat.numel() // 12))
        num = []
        for i in idx:
            keep = flat[i].item()
            flat[i] = keep + step
            hi = loss64(p)
            flat[i] = keep - step
            lo = loss64(p)
            flat[i] = keep
            num.append((hi - lo) / (2 * step))
        num = torch.stack(num)
        # differences: step^2 of the third derivative (~1e-9 here) and 1e-16 |loss| / step; fp32 values: sums of up to
        # B T D = 176 terms through four operators, 1e-5 of the largest gradient
        scale = float(grads_max(grads))
        assert (got.cpu().double().reshape(-1)[idx] - num).abs().max() <= 1e-5 * scale + 1e-8, v.shape


def grads_max(grads):
    return max(g.abs().max() for g in grads)


def _block(layers, p, x, lengths=None):
    u = layers.layer_norm(x, p["nw"], p["nb"])
    cg = layers.linear(u, p["w1"], p["b1"])
    D = x.shape[-1]
    y, h = layers.gated_scan(cg[..., :D], cg[..., D:], lengths=lengths)
    return layers.linear(y, p["w2"], p["b2"], act="silu", residual=x), h


def _block_params(D, dtype, seed=0):
    return {"nw": rnd(D, torch.float32, seed + 1, 0.1, 1.0).requires_grad_(), "nb": rnd(D, torch.float32, seed + 2, 0.1).requires_grad_(),
            "w1": rnd((2 * D, D), dtype, seed + 3, D ** -0.5).requires_grad_(), "b1": rnd(2 * D, dtype, seed + 4, 0.1).requires_grad_(),
            "w2": rnd((D, D), dtype, seed + 5, D ** -0.5).requires_grad_(), "b2": rnd(D, dtype, seed + 6, 0.1).requires_grad_()}


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_two_runs_give_the_same_bits(dtype):
    from vae_amd import layers
    D = 96
    p, x = _block_params(D, dtype), rnd((6, 1100, D), dtype, 9).requires_grad_()
    dy = rnd((6, 1100, D), dtype, 10)
    runs = []
    for _ in range(2):
        y, h = _block(layers, p, x)
        runs.append([y, h] + list(torch.autograd.grad([y, h], [x] + list(p.values()), [dy, torch.ones_like(h)])))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_captured_block_replays_with_new_inputs():
    """Forward and backward of a block in one graph, replayed between eager work, two graphs in turn."""
    from vae_amd import layers
    D = 64

    def make(seed):
        p, x = _block_params(D, torch.bfloat16, seed), rnd((4, 130, D), torch.bfloat16, seed + 9).requires_grad_()
        dy = rnd((4, 130, D), torch.bfloat16, seed + 10)

        def step():
            y, h = _block(layers, p, x)
            return [y.detach(), h.detach()] + list(torch.autograd.grad([y, h], [x] + list(p.values()), [dy, torch.ones_like(h)]))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        return g, out, step, x

    made = [make(0), make(50)]
    for k in range(4):
        for g, out, step, x in made:
            with torch.no_grad():
                x.copy_(rnd(x.shape, x.dtype, 100 + k))
            g.replay()
            want = step()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    from vae_amd import layers
    D = 128
    p = _block_params(D, torch.float32)
    xs = [rnd((3, 500, D), torch.float32, s) for s in (1, 2)]
    want = [_block(layers, p, x)[0] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    outs = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[k].append(_block(layers, p, xs[k])[0])
    torch.cuda.synchronize()
    for k in range(2):
        for o in outs[k]:
            assert torch.equal(o, want[k])


class RecurrentVAE(torch.nn.Module):
    """A window VAE built from the operators as a user would: norm -> projection -> gated recurrence -> residual linear, the state
    behind the window feeds the mu / logvar heads; trained by vae_amd.train.train."""

    def __init__(self, C, D, latent):
        super().__init__()
        self.latent = latent
        par = lambda *s, scale: torch.nn.Parameter(torch.randn(*s) * scale)  # noqa: E731
        self.win, self.bin = par(D, C, scale=C ** -0.5), par(D, scale=0.0)
        self.nw, self.nb = torch.nn.Parameter(torch.ones(D)), torch.nn.Parameter(torch.zeros(D))
        self.w1, self.b1 = par(2 * D, D, scale=D ** -0.5), par(2 * D, scale=0.1)
        self.w2, self.b2 = par(D, D, scale=D ** -0.5), par(D, scale=0.0)
        self.wh, self.bh = par(2 * latent, D, scale=D ** -0.5), par(2 * latent, scale=0.0)
        self.wd, self.bd = par(D, latent, scale=latent ** -0.5), par(D, scale=0.0)
        self.wo, self.bo = par(C, D, scale=D ** -0.5), par(C, scale=0.0)

    def forward(self, x, eps=None):
        from vae_amd import layers
        h = layers.linear(x.transpose(1, 2), self.win, self.bin)
        cg = layers.linear(layers.layer_norm(h, self.nw, self.nb), self.w1, self.b1)
        D = h.shape[-1]
        s, _ = layers.gated_scan(cg[..., :D], cg[..., D:])
        h = layers.linear(s, self.w2, self.b2, act="gelu", residual=h)
        _, last = layers.gated_scan(h, h)
        z = layers.linear(last, self.wh, self.bh)
        mu, logvar = z[:, :self.latent], z[:, self.latent:]
        eps = torch.randn_like(mu) if eps is None else eps
        zz = mu + eps * torch.exp(0.5 * logvar)
        return layers.linear(layers.linear(zz, self.wd, self.bd, act="silu"), self.wo, self.bo), mu, logvar


def test_a_model_of_the_operators_trains():
    """vae_amd.train.train with the package's optimiser runs it; every parameter gets a finite gradient and moves."""
    import vae_amd
    torch.manual_seed(0)
    m = RecurrentVAE(3, 32, 5).cuda()
    before = {k: v.detach().clone() for k, v in m.named_parameters()}
    data = torch.randn(3, 60 + 64)
    loader = vae_amd.train.DeviceSlidingWindow(data, 60, batch_size=16)
    opt = vae_amd.optim.Adam(m.parameters(), lr=1e-3)
    loss = vae_amd.train.train(m, loader, vae_amd.train.criterion, opt, "cuda", 1)
    assert math.isfinite(loss)
    for k, v in m.named_parameters():
        assert torch.isfinite(v.grad).all(), k
        assert not torch.equal(v, before[k]), k


# ------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    import vae_amd
    from vae_amd import layers
    x = torch.zeros(4, 8, device="cuda")
    E, V = vae_amd.VaeAmdError, ValueError
    for err, call in ((E, lambda: layers.layer_norm(x.double())), (E, lambda: layers.layer_norm(x.cpu())),
                      (V, lambda: layers.layer_norm(x, torch.ones(7, device="cuda"))),
                      (E, lambda: layers.layer_norm(x, torch.ones(8, device="cuda").half())),
                      (E, lambda: layers.layer_norm(x, torch.ones(8))),
                      (V, lambda: layers.layer_norm(torch.zeros(4, 0, device="cuda"))),
                      (E, lambda: layers.layer_norm(x.half(), torch.ones(8, device="cuda"), torch.ones(8, device="cuda").half())),
                      (V, lambda: layers.linear(x, torch.zeros(3, 7, device="cuda"))),
                      (V, lambda: layers.linear(x, torch.zeros(8, device="cuda"))),
                      (V, lambda: layers.linear(x, torch.zeros(3, 8, device="cuda"), act="tanh")),
                      (E, lambda: layers.linear(x, torch.zeros(3, 8, device="cuda").half())),
                      (V, lambda: layers.linear(x, torch.zeros(3, 8, device="cuda"), torch.zeros(4, device="cuda"))),
                      (V, lambda: layers.linear(x, torch.zeros(3, 8, device="cuda"), residual=torch.zeros(1, 3, device="cuda"))),
                      (V, lambda: layers.gated_scan(x, x)),
                      (V, lambda: layers.gated_scan(x[None], x[None, :2])),
                      (E, lambda: layers.gated_scan(x[None], x[None].half())),
                      (V, lambda: layers.gated_scan(x[None], x[None], torch.zeros(2, 8, device="cuda"))),
                      (E, lambda: layers.gated_scan(x[None].half(), x[None].half(), torch.zeros(1, 8, device="cuda").half())),
                      (E, lambda: layers.gated_scan(x[None], x[None], lengths=torch.ones(1, device="cuda"))),
                      (E, lambda: layers.gated_scan(x[None], x[None], lengths=torch.ones(1, dtype=torch.int32)))):
        with pytest.raises(err):
            call()
    xg = x.clone().requires_grad_()
    (g,) = torch.autograd.grad((layers.layer_norm(xg) * xg).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        g.sum().backward()


# ------------------------------------------------------------------------------------------------ beyond 2^31 elements
def _long(*shape):
    t = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
    assert t.numel() > 2 ** 31
    for part in t.view(-1).split(2 ** 28):
        part.normal_()
    return t


def test_norm_beyond_32_bits_of_offset():
    """The last rows of a tensor of 2.2e9 elements, alone in having a gradient."""
    from vae_amd import layers
    rows, cols, n = 2_000_001, 1100, 40
    x = _long(rows, cols).requires_grad_()
    w, b = rnd(cols, torch.float32, 3, 0.2, 1.0).requires_grad_(), rnd(cols, torch.float32, 4, 0.1).requires_grad_()
    y = layers.layer_norm(x, w, b)
    dy = torch.zeros_like(y)
    dy[-n:] = rnd((n, cols), torch.bfloat16, 5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want = norm64(x.detach()[-n:], w.detach(), b.detach(), dy[-n:], 1e-5)
    for name, got in (("y", y.detach()[-n:]), ("dx", dx[-n:]), ("dw", dw), ("db", db)):
        check(name, got, *want[name])


@pytest.mark.parametrize("m,n,k", [(1_048_616, 24, 2104), (1_048_616, 24, 2101), (262_184, 8200, 64)])
def test_linear_beyond_32_bits_of_offset(m, n, k):
    """x, then y, of more than 2^31 elements: as above."""
    from vae_amd import layers
    last = 40
    x = (_long(m, k) if m * k > 2 ** 31 else rnd((m, k), torch.bfloat16, 1)).requires_grad_()
    w = rnd((n, k), torch.bfloat16, 2, k ** -0.5).requires_grad_()
    y = layers.linear(x, w, act="leaky", slope=SLOPE)
    dy = torch.zeros_like(y)
    dy[-last:] = rnd((last, n), torch.bfloat16, 5)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = linear64(x.detach()[-last:], w.detach(), None, None, dy[-last:], "leaky")
    for name, got in (("y", y.detach()[-last:]), ("dx", dx[-last:]), ("dw", dw)):
        check(name, got, *want[name])


def test_scan_beyond_32_bits_of_offset():
    """The last sequences of a long batch, and the last steps of a long series (behind a step that forgets everything)."""
    b, t, d = 70_000, 8, 4096
    x, gate, dy = _long(b, t, d), _long(b, t, d), _long(b, t, d)
    h0, dhl = rnd((b, d), torch.float32, 3), rnd((b, d), torch.float32, 5)
    got, n = run_scan(x, gate, h0, None, dy, dhl), 3
    scan_compare({k: v[-n:] for k, v in got.items()}, scan64(x[-n:], gate[-n:], h0[-n:], None, dy[-n:], dhl[-n:]))
    del got
    x, gate, dy = (v.view(1, -1, d)[:, :540_000] for v in (x, gate, dy))
    assert x.numel() > 2 ** 31
    n = 200
    gate[:, -n] = -100.0
    got = run_scan(x, gate, None, None, dy, dhl[-1:])
    want = scan64(x[:, -n:], gate[:, -n:], None, None, dy[:, -n:], dhl[-1:])
    for k in ("y", "dx", "dgate"):
        check(k, got[k][:, 1 - n:], *(v[:, 1:] for v in want[k]))
    check("h", got["h"], *want["h"])
