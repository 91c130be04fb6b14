"""Refusals of modulated_norm, gated_residual and gated_residual_norm that need no GPU: arguments are
checked before any device call."""
import ctypes

import pytest
import torch

X = torch.zeros((6, 32))


def test_refusals(pkg):
    m, g, b = pkg.modulated_norm, pkg.gated_residual, pkg.gated_residual_norm
    for bad in (torch.zeros(32), torch.zeros((2, 3, 32)), torch.zeros((6, 0))):
        with pytest.raises(pkg.TscError, match=r"x must be \(N, C\)"):
            m(bad)
    for bad in (torch.zeros((5, 32)), X.half()):
        with pytest.raises(pkg.TscError, match="y must have"):
            g(X, bad)
    for bad in ("batch", 1):
        with pytest.raises(pkg.TscError, match="'layer' or 'rms'"):
            m(X, norm=bad)
        with pytest.raises(pkg.TscError, match="post_norm must be"):
            b(X, X, post_norm=bad)
    for f in (lambda: m(X, norm=None), lambda: b(X, X, norm=None)):
        with pytest.raises(pkg.TscError, match="norm must be"):
            f()
    with pytest.raises(pkg.TscError, match="needs a post_norm"):
        g(X, X, post_weight=torch.zeros(32))
    for bad in (torch.zeros(31), torch.zeros(32).half(), torch.zeros((1, 32))):
        with pytest.raises(pkg.TscError, match="weights and biases"):
            m(X, weight=bad)
    for bad in (torch.zeros((2, 32)), torch.zeros(32), torch.zeros((1, 32)).half()):
        with pytest.raises(pkg.TscError, match=r"scale must be \(1, 32\)"):
            m(X, scale=bad)
    with pytest.raises(pkg.TscError, match="gate: each sample's"):
        g(X, X, [0, 3, 6], gate=torch.zeros((32, 2)).t())
    with pytest.raises(pkg.TscError, match="shift: each sample's"):
        m(X, [0, 3, 6], shift=torch.zeros((1, 32)).expand(2, 32))
    for bad in (-1.0, float("nan"), float("inf"), 1e39):
        with pytest.raises(pkg.TscError, match="eps"):
            m(X, eps=bad)
    for bad in (float("nan"), float("inf"), -1e39):
        with pytest.raises(pkg.TscError, match="residual_scale"):
            g(X, X, residual_scale=bad)
    with pytest.raises(pkg.TscError, match="out has the wrong"):
        m(X, out=torch.zeros((6, 31)))
    with pytest.raises(pkg.TscError, match="unsupported dtype"):
        m(X.double())
    with pytest.raises(pkg.TscError, match="not on a GPU"):
        m(X)


def test_c_entry_points_without_a_gpu(pkg):
    lib = pkg.load_library()
    P = ctypes.c_void_p
    ws = lib.tsc_gated_norm_workspace_bytes
    assert ws(2, 2, 1000, 64) >= 3 * 4 * 64 * 4 and ws(2, 0, 0, 64) == 0 and ws(0, 3, 10, 8192) > 0
    assert ws(0, 4, 0, 8) > 0
    for bad in ((3, 1, 1, 8), (0, -1, 1, 8), (0, 1, -1, 8), (0, 1, 2 ** 31, 8), (0, 1, 1, 0), (0, 1, 1, 8193),
                (0, 2 ** 20 + 1, 1, 8)):
        assert ws(*bad) == -1 and lib.tsc_last_error(), bad
    st = lib.tsc_gated_norm(None, 0, P(16), None, None, 1, 1, 8, 0, None, None, None, 0, 1.0, 1, None, None,
                            None, 0, None, 0, 1e-6, 0, None, None, P(16))
    assert st == 1 and b"null context" in lib.tsc_last_error()
    st = lib.tsc_gated_norm_backward(None, 0, P(16), None, None, 1, 1, 8, 0, None, None, None, 0, 1.0, 1, None,
                                     None, None, 0, None, 0, 1e-6, 0, P(16), None, P(16), P(16), P(16), None,
                                     None, None, None, None, None, None, None)
    assert st == 1 and b"null context" in lib.tsc_last_error()
