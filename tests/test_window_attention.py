"""Refusals of sparse_window_attention that need no GPU: arguments are checked before any device call."""
import ctypes

import pytest
import torch


def _t(n, h=2, d=64, dtype=torch.float32):
    return torch.zeros((n, h, d), dtype=dtype)


def test_refusals(pkg):
    f, q = pkg.sparse_window_attention, _t(10)
    for bad in ((q.view(10, 128), q, q), (q, _t(7), _t(8)), (q, _t(10, 2, 128), _t(10, 2, 128))):
        with pytest.raises(pkg.TscError, match=r"\(total, heads, D\)"):
            f(*bad, 4, [0, 10])
    for hk in (3, 4, 0):
        with pytest.raises(pkg.TscError, match="do not divide"):
            f(q, _t(10, hk), _t(10, hk), 4, [0, 10])
    with pytest.raises(pkg.TscError, match="head_dim 96"):
        f(_t(10, 2, 96), _t(10, 2, 96), _t(10, 2, 96), 4, [0, 10])
    with pytest.raises(pkg.TscError, match="share a dtype"):
        f(q, q.half(), q, 4, [0, 10])
    with pytest.raises(pkg.TscError, match="unsupported dtype"):
        f(q.double(), q.double(), q.double(), 4, [0, 10])
    for window, sinks in ((-1, 0), (2 ** 31, 0), (4, -1), (4, 2 ** 31)):
        with pytest.raises(pkg.TscError, match="window .* and sinks"):
            f(q, q, q, window, [0, 10], sinks=sinks)
    for window in (1.5, "4"):
        with pytest.raises(TypeError):
            f(q, q, q, window, [0, 10])
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-46, 1e39):
        with pytest.raises(pkg.TscError, match="scale"):
            f(q, q, q, 4, [0, 10], scale=scale)
    for bad in (_t(9), _t(10).half()):
        with pytest.raises(pkg.TscError, match="out has the wrong"):
            f(q, q, q, 4, [0, 10], out=bad)
    with pytest.raises(pkg.TscError, match="contiguous"):
        f(torch.zeros((10, 64, 2)).transpose(1, 2), q, q, 4, [0, 10])
    with pytest.raises(pkg.TscError, match="contiguous"):
        f(q, torch.zeros((1, 2, 64)).expand(10, 2, 64), q, 4, [0, 10])
    with pytest.raises(pkg.TscError, match="not on"):
        f(q, q, q, 4, [0, 10])


def test_c_entry_points_without_a_gpu(pkg):
    lib = pkg.load_library()
    P = ctypes.c_void_p
    ws = lib.tsc_window_attention_workspace_bytes
    assert ws(2, 1, 1, 40000, 12, 4, 128, 30000, 4, 1, 1, 40000, 0) > 0  # one query: shared out over the keys
    assert ws(2, 1, 20000, 20000, 12, 12, 128, 500, 4, 1, 20000, 20000, 0) == 0
    assert ws(2, 1, 100, 100, 12, 12, 128, 10, 0, 0, 100, 100, 1) >= 12 * 100 * 4
    assert ws(2, 0, 0, 0, 12, 12, 128, 10, 0, 0, 0, 0, 0) == 0
    good = [0, 1, 1, 1, 2, 1, 64, 5, 0, 0, 1, 1, 0]
    assert ws(*good) == 0
    for at, bad in ((0, 3), (1, -1), (1, 65536), (2, -1), (2, 2 ** 31), (3, 2 ** 31), (4, 0), (4, 65536), (5, 0),
                    (5, 3), (6, 32), (7, -1), (8, -1), (10, -1), (11, -1)):
        args = list(good)
        args[at] = bad
        assert ws(*args) == -1 and lib.tsc_last_error(), (at, bad)
    st = lib.tsc_window_attention(None, 0, P(16), P(16), P(16), 64, 64, 64, P(16), P(16), 1, 1, 1, 1, 1, 64, 0.0, 4,
                                  0, 0, 1, 1, 0, None, P(16), None, None)
    assert st == 1 and b"null context" in lib.tsc_last_error()
    st = lib.tsc_window_attention_backward(None, 0, P(16), P(16), P(16), 64, 64, 64, P(16), P(16), 1, 1, 1, 1, 1, 64,
                                           0.0, 4, 0, 0, 1, 1, 0, P(16), None, P(16), P(16), P(16), P(16), P(16),
                                           P(16))
    assert st == 1 and b"null context" in lib.tsc_last_error()


def test_scratch_of_parts_stays_near_the_inputs(pkg):
    """At most four times what q, k, v and out take, or 64 MB."""
    ws = pkg.load_library().tsc_window_attention_workspace_bytes
    split = 0
    for code, size in ((0, 4), (1, 2), (2, 2)):
        for d in (64, 128):
            for h, hk in ((1, 1), (8, 1), (16, 4), (12, 12)):
                for b in (1, 3, 16, 250):
                    for longest in (1, 32, 128, 1000):
                        for kv in (3000, 220000, 4000000):
                            for window in (0, 100, 5000, 2 ** 31 - 1):
                                tq, tkv = b * longest, kv + 1048 * (b - 1)
                                got = ws(code, b, tq, tkv, h, hk, d, window, 4, 1, longest, kv, 0)
                                assert 0 <= got <= max(64 << 20, 8 * d * size * (tq * h + tkv * hk))
                                split += got > 0
    assert split > 200


def test_scales_whose_powers_of_two_overflow_are_refused(pkg):
    """Scores are multiplied with scale log2(e), which fp32 has to hold: 2^128 / log2(e) is 2.3587e38."""
    f, q = pkg.sparse_window_attention, _t(10)
    for scale in (2.36e38, 3.4e38):
        with pytest.raises(pkg.TscError, match="scale"):
            f(q, q, q, 4, [0, 10], scale=scale)
    for scale in (2.35e38, 1e-45):
        with pytest.raises(pkg.TscError, match="not on"):
            f(q, q, q, 4, [0, 10], scale=scale)
