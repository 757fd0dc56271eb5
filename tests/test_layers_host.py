"""Host side of the sequence-block operators: no CPU path, argument checks of the C entries (all before any launch), sizes."""
import pytest
import torch


def _fails(rc, text):
    from vae_amd import _lib as L
    assert rc == -1, rc
    assert text in L.lib().vae_last_error().decode(), L.lib().vae_last_error()


def test_no_cpu_fallback():
    import vae_amd
    from vae_amd import layers
    x = torch.zeros(2, 3, 4)
    for call in (lambda: layers.layer_norm(x), lambda: layers.linear(x, torch.zeros(5, 4)), lambda: layers.gated_scan(x, x)):
        with pytest.raises(vae_amd.VaeAmdError):
            call()


def test_layer_norm_entry_checks():
    from vae_amd import _lib as L
    lib, p = L.lib(), 4096  # (an address that no check reads)
    _fails(lib.vae_layer_norm_forward(p, 8, None, None, p, 8, None, None, 4, 8, 1e-5, 3, 0, None), "type")
    _fails(lib.vae_layer_norm_forward(p, 8, None, None, p, 8, None, None, 4, 8, 1e-5, L.T_F32, L.T_BF16, None), "parameters")
    _fails(lib.vae_layer_norm_forward(p, 8, None, None, p, 8, None, None, 4, 0, 1e-5, 0, 0, None), "rows")
    _fails(lib.vae_layer_norm_forward(p, 8, None, None, p, 8, None, None, -1, 8, 1e-5, 0, 0, None), "rows")
    _fails(lib.vae_layer_norm_forward(None, 8, None, None, p, 8, None, None, 4, 8, 1e-5, 0, 0, None), "null")
    _fails(lib.vae_layer_norm_forward(p, 8, None, None, p, 8, p, None, 4, 8, 1e-5, 0, 0, None), "null")
    _fails(lib.vae_layer_norm_forward(p, 7, None, None, p, 8, None, None, 4, 8, 1e-5, 0, 0, None), "stride")
    _fails(lib.vae_layer_norm_backward(p, 8, p, 8, None, p, p, p, 8, p, None, None, 4, 8, 0, 0, None), "null")
    _fails(lib.vae_layer_norm_backward(p, 8, p, 8, None, p, p, p, 7, None, None, None, 4, 8, 0, 0, None), "stride")
    assert lib.vae_layer_norm_forward(None, 8, None, None, None, 8, None, None, 0, 8, 1e-5, 0, 0, None) == 0  # no rows: nothing to do
    assert lib.vae_layer_norm_workspace_floats(0, 8) == 0 and lib.vae_layer_norm_workspace_floats(10, 8) >= 16


def test_dense_entry_checks():
    from vae_amd import _lib as L
    lib, p = L.lib(), 4096
    _fails(lib.vae_dense_forward(p, 8, p, 8, None, None, 0, p, 4, None, None, 2, 4, 8, 0, 0.0, 9, None), "type")
    _fails(lib.vae_dense_forward(p, 8, p, 8, None, None, 0, p, 4, None, None, 2, 4, 8, 5, 0.0, 0, None), "activation")
    _fails(lib.vae_dense_forward(p, 8, p, 8, None, None, 0, p, 4, None, None, 2, 0, 8, 0, 0.0, 0, None), "N = 0")
    _fails(lib.vae_dense_forward(p, 8, None, 8, None, None, 0, p, 4, None, None, 2, 4, 8, 0, 0.0, 0, None), "null")
    _fails(lib.vae_dense_forward(p, 7, p, 8, None, None, 0, p, 4, None, None, 2, 4, 8, 0, 0.0, 0, None), "stride")
    _fails(lib.vae_dense_forward(p, 8, p, 8, None, p, 3, p, 4, None, None, 2, 4, 8, 0, 0.0, 0, None), "stride")
    assert lib.vae_dense_forward_workspace_floats(100, 8, 4096, L.T_F32) >= 2 * 100 * 8  # few outputs, a long sum: split
    _fails(lib.vae_dense_forward(p, 4096, p, 4096, None, None, 0, p, 8, None, None, 100, 8, 4096, 0, 0.0, 0, None), "workspace")
    assert [lib.vae_dense_forward_workspace_floats(*a) for a in ((1, 8, 4096, 0), (100, 8, 64, 0), (4096, 4096, 4096, 0), (0, 8, 64, 0))] == [0] * 4
    _fails(lib.vae_dense_backward(p, 4, p, 8, p, 8, None, p, p, p, p, 2, 4, 8, L.ACT_GELU, 0.0, 0, None), "null")
    _fails(lib.vae_dense_backward(p, 4, p, 8, p, 8, None, p, p, p, None, 2, 4, 8, 0, 0.0, 0, None), "null")
    _fails(lib.vae_dense_backward(p, 4, p, 8, p, 8, None, p, p, p, p, 0, 4, 8, 0, 0.0, 0, None), "no rows")
    assert lib.vae_dense_forward(None, 8, None, 8, None, None, 0, None, 4, None, None, 0, 4, 8, 0, 0.0, 0, None) == 0
    # what act' needs: a byte for the leaky ReLU, fp16 behind bf16 tensors, fp32 else
    assert [lib.vae_dense_aux_bytes(3, 5, a, L.T_BF16) for a in range(5)] == [0, 15, 30, 30, 30]
    assert [lib.vae_dense_aux_bytes(3, 5, a, L.T_F16) for a in range(5)] == [0, 15, 60, 60, 60]


def test_gated_scan_entry_checks():
    from vae_amd import _lib as L
    lib, p = L.lib(), 4096
    _fails(lib.vae_gated_scan_forward(p, 8, 4, p, 8, 4, None, None, p, None, None, None, 1, 2, 4, 7, None), "type")
    _fails(lib.vae_gated_scan_forward(p, 8, 4, p, 8, 4, None, None, p, None, None, None, 1, 0, 4, 0, None), "steps")
    _fails(lib.vae_gated_scan_forward(p, 8, 4, None, 8, 4, None, None, p, None, None, None, 1, 2, 4, 0, None), "null")
    n = lib.vae_gated_scan_workspace_floats(1, 100000, 4, 0)
    assert n > 0 and n % 8 == 0
    _fails(lib.vae_gated_scan_forward(p, 8, 4, p, 8, 4, None, None, p, None, None, None, 1, 100000, 4, 0, None), "null")
    _fails(lib.vae_gated_scan_backward(p, 8, 4, None, p, 8, 4, p, 8, 4, None, None, None, p, p, None, p, 1, 1000, 4, 0, None), "null")
    assert lib.vae_gated_scan_forward(None, 8, 4, None, 8, 4, None, None, None, None, None, None, 0, 2, 4, 0, None) == 0
    assert lib.vae_gated_scan_kept_floats(2, 64, 5) == 0 and lib.vae_gated_scan_kept_floats(2, 65, 5) == 20
