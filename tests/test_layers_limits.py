"""Sizes that the sequence-block operators do not take: seen as they are (64 bits) and refused before any launch.  No GPU."""
import pytest

P = 4096  # an address that no check reads
BIG = 2 ** 32


def _refused(rc, text):
    from vae_amd import _lib as L
    assert rc == -1, rc
    assert text in L.lib().vae_last_error().decode(), L.lib().vae_last_error()


def _norm_fwd(rows, c, dtype=0):
    from vae_amd import _lib as L
    return L.lib().vae_layer_norm_forward(P, c, None, None, P, c, None, None, rows, c, 1e-5, dtype, 0, None)


def _norm_bwd(rows, c, dw=P):
    from vae_amd import _lib as L
    return L.lib().vae_layer_norm_backward(P, c, P, c, None, P, P, None, c, dw, None, P, rows, c, 0, 0, None)


def _dense_fwd(m, n, k, dtype=0):
    from vae_amd import _lib as L
    return L.lib().vae_dense_forward(P, k, P, k, None, None, 0, P, n, None, P, m, n, k, 0, 0.0, dtype, None)


def _dense_bwd(m, n, k, dx=P, dw=P):
    from vae_amd import _lib as L
    return L.lib().vae_dense_backward(P, n, P, k, P, k, None, dx, dw, None, P, m, n, k, 0, 0.0, 0, None)


def _scan_fwd(b, t, d):
    from vae_amd import _lib as L
    return L.lib().vae_gated_scan_forward(P, t * d, d, P, t * d, d, None, None, P, None, None, P, b, t, d, 0, None)


def _scan_bwd(b, t, d):
    from vae_amd import _lib as L
    return L.lib().vae_gated_scan_backward(P, t * d, d, None, P, t * d, d, P, t * d, d, None, None, P, P, P, None, P, b, t, d, 0, None)


@pytest.mark.parametrize("over", [0, 8, 100])
def test_sizes_of_33_bits_do_not_wrap(over):
    big = BIG + over
    for call in (_norm_fwd, _norm_bwd):
        _refused(call(2, big), f"rows of {big}")
        _refused(call(big, 8), f"{big} rows")
    for call in (_dense_fwd, _dense_bwd):
        _refused(call(big, 8, 8), f"M = {big}")
        _refused(call(8, big, 8), f"N = {big}")
        _refused(call(8, 8, big), f"K = {big}")
    for call in (_scan_fwd, _scan_bwd):
        _refused(call(big, 2, 2), f"{big} sequences")
        _refused(call(2, big, 2), f"{big} steps")
        _refused(call(2, 2, big), f"{big} features")


def test_sizes_at_the_limits():
    _refused(_norm_fwd(2 ** 31, 8), "rows")
    _refused(_norm_fwd(1, 2 ** 31), "rows of")
    for call in (_dense_fwd, _dense_bwd):
        for mnk in ((2 ** 30, 8, 8), (8, 2 ** 30, 8), (8, 8, 2 ** 30)):
            _refused(call(*mnk), "M = ")
    for call in (_scan_fwd, _scan_bwd):
        _refused(call(2 ** 16, 1, 2 ** 15), "sequences")
        _refused(call(1, 2 ** 31 - 2 ** 16 + 1, 1), "steps")


def test_queries_of_sizes_that_no_call_takes():
    from vae_amd import _lib as L
    lib = L.lib()
    assert lib.vae_gated_scan_kept_floats(1, BIG + 100, 8) == 0 and lib.vae_gated_scan_kept_floats(1, 100, 8) == 16
    assert lib.vae_gated_scan_workspace_floats(1, BIG + 9001, 24, 0) == 0 and lib.vae_gated_scan_workspace_floats(1, 9001, 24, 0) > 0
    assert lib.vae_layer_norm_workspace_floats(10, BIG + 8) == 0
    assert lib.vae_dense_forward_workspace_floats(BIG + 100, 8, 4096, 0) == 0 and lib.vae_dense_workspace_floats(BIG + 100, 8, 4096, 0, 0) == 0


def test_launches_of_2_to_the_32_threads():
    """Sizes within the limits whose launch would not be: rows of a whole workgroup each, tiles of 64 x 64, columns of 64 channels."""
    _refused(_norm_fwd(2 ** 22, 16385), "more than a launch holds")
    _refused(_norm_bwd(1, 2 ** 27), "more than a launch holds")
    _refused(_dense_fwd(2 ** 30 - 1, 64, 9), "more than a launch holds")
    _refused(_dense_fwd(2 ** 29, 65, 9, 1), "more than a launch holds")
    _refused(_dense_bwd(2 ** 30 - 1, 9, 64, dw=None), "more than a launch holds")
    _refused(_dense_bwd(2 ** 30 - 1, 9, 64), "more than a launch holds")
    _refused(_scan_fwd(2 ** 30, 40, 1), "more than a launch holds")
    _refused(_scan_bwd(2 ** 30, 40, 1), "more than a launch holds")


def test_a_state_is_not_advanced_in_place():
    """The last lanes of a sequence share features with their neighbours: with h_last in h0's memory one could read what the other wrote."""
    from vae_amd import _lib as L
    lib, n = L.lib(), 3 * 7
    for at in (P, P + 4, P + 4 * (n - 1), P - 4 * (n - 1)):
        _refused(lib.vae_gated_scan_forward(P, 7, 7, P, 7, 7, P, None, P, at, None, None, 3, 1, 7, 0, None), "h_last")
        _refused(lib.vae_gated_scan_backward(P, 7, 7, P, P, 7, 7, P, 7, 7, None, None, None, P, P, at, None, 3, 1, 7, 0, None), "dh0")
