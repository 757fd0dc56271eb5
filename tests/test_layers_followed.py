"""Calls of the sequence-block operators that torch follows (forward-mode duals, torch.jit.trace, make_fx), also without any tensor that
asks for a gradient: refused, never an empty result taken for the operator's.  On the CPU with the C entries stubbed."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

OPS = ["layer_norm", "linear", "gated_scan"]


@pytest.fixture
def layers(monkeypatch):
    from vae_amd import _lib as L
    from vae_amd import layers
    monkeypatch.setattr(L, "_device_ok", {None})
    monkeypatch.setattr(layers, "_call", lambda fn, name, device, *args: None)
    return layers


def _op(layers, name, second=False):
    """A function of one tensor: the operator's input, or (second) its other floating-point argument."""
    x, g = torch.randn(2, 4, 8), torch.randn(2, 4, 8)
    w, b = torch.randn(8, 8), torch.randn(8)
    return {("layer_norm", False): (lambda t: layers.layer_norm(t, b), x), ("layer_norm", True): (lambda t: layers.layer_norm(x, b, t), b),
            ("linear", False): (lambda t: layers.linear(t, w), x), ("linear", True): (lambda t: layers.linear(x, w, residual=t), g),
            ("gated_scan", False): (lambda t: layers.gated_scan(t, g)[0], x),
            ("gated_scan", True): (lambda t: layers.gated_scan(x, g, t)[1], torch.randn(2, 8))}[name, second]


@pytest.mark.parametrize("second", [False, True])
@pytest.mark.parametrize("name", OPS)
@pytest.mark.parametrize("no_grad", [False, True])
def test_a_dual_is_refused(layers, name, second, no_grad):
    f, t = _op(layers, name, second)
    with fwad.dual_level():
        f(t)  # (no dual: as ever)
        with torch.set_grad_enabled(not no_grad), pytest.raises(NotImplementedError):
            f(fwad.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("name", OPS)
def test_a_dual_gradient_is_refused(layers, name):
    import vae_amd
    f, t = _op(layers, name)
    t.requires_grad_()
    with fwad.dual_level():
        y = f(t)
        up = torch.ones_like(y)
        torch.autograd.grad(y, t, up, retain_graph=True)
        with pytest.raises(vae_amd.VaeAmdError):
            torch.autograd.grad(y, t, fwad.make_dual(up, up.clone()))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", OPS)
def test_a_trace_is_refused(layers, name, grad):
    import vae_amd
    f, t = _op(layers, name)
    with pytest.raises(vae_amd.VaeAmdError):
        torch.jit.trace(f, (t.requires_grad_(grad),), check_trace=False)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", OPS)
def test_make_fx_is_refused(layers, name, grad):
    import vae_amd
    from torch.fx.experimental.proxy_tensor import make_fx
    f, t = _op(layers, name)
    with pytest.raises(vae_amd.VaeAmdError):
        make_fx(f)(t.requires_grad_(grad))


@pytest.mark.parametrize("name", OPS)
def test_transforms_raise(layers, name):
    f, t = _op(layers, name)
    for call in (lambda: torch.func.vmap(f)(t[None]), lambda: torch.func.jvp(f, (t,), (t,)), lambda: torch.func.grad(lambda v: f(v).sum())(t)):
        with pytest.raises(RuntimeError):
            call()
