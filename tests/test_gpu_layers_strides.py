"""Strided operands through every form of the sequence-block operators: rows taken out of wider buffers as they lie, with NaN in the gaps.

Tolerances are those of the dense cases (test_gpu_layers.py): strides change where values come from, not how they are added."""
import pytest
import torch

from test_gpu_layers import DTYPES, IDS, SLOPE, U, act64, check, linear64, norm64, rnd, scan64  # noqa: F401

pytestmark = pytest.mark.gpu


def gaps(t, before, behind):
    """t's values in rows of a wider buffer whose other columns are NaN."""
    wide = torch.full(t.shape[:-1] + (before + t.shape[-1] + behind,), float("nan"), dtype=t.dtype, device=t.device)
    view = wide[..., before:before + t.shape[-1]]
    view.copy_(t)
    assert t.numel() == t.shape[-1] or not view.is_contiguous()
    return view


# few rows, tiles of 64, sums split over k, tiles of 128 and of 256 in turn for each product
SHAPES = [(40, 72, 136), (130, 72, 136), (100, 72, 4000), (130, 264, 1000), (2048, 1920, 200), (4100, 2568, 264), (4100, 264, 2568), (264, 4104, 2568)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("before,behind", [(16, 8), (3, 4)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_rows_of_wider_buffers(m, n, k, before, behind, dtype):
    """(16, 8): rows that start on 16 bytes, the direct loads' form; (3, 4): rows at any alignment."""
    from vae_amd import layers
    x, w, r, dy = rnd((m, k), dtype, 1), rnd((n, k), dtype, 2, k ** -0.5), rnd((m, n), dtype, 4), rnd((m, n), dtype, 5)
    b = rnd((n,), dtype, 3, 0.3)
    for act in ("silu", "none"):
        want = linear64(x, w, b, r, dy, act)
        t = [gaps(v, before, behind).detach().requires_grad_() for v in (x, w, r)]
        bias = b.clone().requires_grad_()
        y = layers.linear(t[0], t[1], bias, act=act, residual=t[2])
        dx, dw, dr, db = torch.autograd.grad(y, t + [bias], gaps(dy, before, behind))
        for name, got in (("y", y.detach()), ("dx", dx), ("dw", dw), ("db", db)):
            check(name, got, *want[name])
        assert torch.equal(dr, dy)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(2050, 2051, 203), (1500, 3001, 2005)])
def test_linear_ragged_rows_of_wider_buffers(m, n, k, dtype):
    """Rows that are no whole pieces: as they lie, or laid out anew for the larger tiles."""
    from vae_amd import layers
    x, w, dy = rnd((m, k), dtype, 1), rnd((n, k), dtype, 2, k ** -0.5), rnd((m, n), dtype, 5)
    want = linear64(x, w, None, None, dy, "none")
    t = [gaps(v, 1, 2).detach().requires_grad_() for v in (x, w)]
    y = layers.linear(*t)
    dx, dw = torch.autograd.grad(y, t, gaps(dy, 2, 1))
    for name, got in (("y", y.detach()), ("dx", dx), ("dw", dw)):
        check(name, got, *want[name])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 70, 136), (40, 70, 136), (130, 70, 136), (100, 70, 4000), (2048, 1921, 200), (4100, 2571, 264)])
def test_linear_writes_rows_of_a_wider_buffer(m, n, k, dtype):
    """Through the C entry: y's columns at a stride of their own; what lies between them and behind them stays."""
    from vae_amd import _lib as L
    x, w, b, r = rnd((m, k), dtype, 1), rnd((n, k), dtype, 2, k ** -0.5), rnd((n,), dtype, 3, 0.3), gaps(rnd((m, n), dtype, 4), 5, 6)
    code, lib = {torch.float32: L.T_F32, torch.bfloat16: L.T_BF16, torch.float16: L.T_F16}[dtype], L.lib()
    out = torch.full((m + 2, n + 13), -7.0, dtype=dtype, device="cuda")
    ws = torch.empty(max(1, lib.vae_dense_forward_workspace_floats(m, n, k, code)), device="cuda")
    L.check(lib.vae_dense_forward(x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), r.data_ptr(), r.stride(0), out.data_ptr(), n + 13, None, ws.data_ptr(),
                                  m, n, k, L.ACT_SILU, 0.0, code, L.stream_ptr()), "vae_dense_forward")
    check("y", out[:m, :n], *linear64(x, w, b, r, None, "silu")["y"])
    assert (out[m:] == -7).all() and (out[:, n:] == -7).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(50, 5), (50, 30), (50, 100), (50, 1000), (9, 5001), (9, 9000), (5, 20000), (5, 70001)])
def test_norm_rows_of_wider_buffers(rows, cols, dtype):
    from vae_amd import layers
    x, dy = rnd((rows, cols), dtype, 1, 1.5, 0.3), rnd((rows, cols), dtype, 2)
    w, b = rnd(cols, torch.float32, 3, 0.2, 1.0).requires_grad_(), rnd(cols, torch.float32, 4, 0.1).requires_grad_()
    t = gaps(x, 3, 10).detach().requires_grad_()
    y = layers.layer_norm(t, w, b)
    dx, dw, db = torch.autograd.grad(y, (t, w, b), gaps(dy, 7, 2))
    want = norm64(x, w.detach(), b.detach(), dy, 1e-5)
    for name, got in (("y", y.detach()), ("dx", dx), ("dw", dw), ("db", db)):
        check(name, got, *want[name])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("b,t,d", [(3, 1, 33), (2, 9, 33), (2, 40, 65), (4, 70, 33), (2, 300, 100), (1, 9001, 24)])
def test_scan_of_the_halves_of_one_projection(b, t, d, dtype):
    """Both inputs are columns of one tensor with NaN around them; its gradient holds both gradients."""
    from vae_amd import layers
    x, gate, h0 = rnd((b, t, d), dtype, 1), rnd((b, t, d), dtype, 2, 1.5, 2.0), rnd((b, d), torch.float32, 3)
    dy, dhl = rnd((b, t, d), dtype, 4), rnd((b, d), torch.float32, 5)
    both = gaps(torch.cat([x, gate], -1), 1, 2).detach().requires_grad_()
    y, h = layers.gated_scan(*both.chunk(2, -1), h0)
    (grad,) = torch.autograd.grad([y, h], both, [gaps(dy, 2, 1), dhl])
    want = scan64(x, gate, h0, None, dy, dhl)
    for name, got in (("y", y.detach()), ("h", h.detach()), ("dx", grad[..., :d]), ("dgate", grad[..., d:])):
        check(name, got, *want[name])
