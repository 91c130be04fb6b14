"""Refusals of sparse_diff_attention that need no GPU: arguments are checked before any device call."""
import ctypes

import pytest
import torch


def _t(n, h=2, d=64, dtype=torch.float32):
    return torch.zeros((n, h, d), dtype=dtype)


def test_refusals(pkg):
    f, q, lam = pkg.sparse_diff_attention, _t(10), torch.zeros(2)
    with pytest.raises(pkg.TscError, match=r"\(total, H, D\)"):
        f(q.view(10, 128), q, q, lam, [0, 10])
    with pytest.raises(pkg.TscError, match=r"\(total, H, D\)"):
        f(q, _t(7), _t(8), lam, [0, 10], [0, 7])
    with pytest.raises(pkg.TscError, match=r"\(total, H, D\)"):
        f(q, _t(10, 1), _t(10, 1), lam, [0, 10])
    with pytest.raises(pkg.TscError, match="head_dim 96"):
        f(_t(10, 2, 96), _t(10, 2, 96), _t(10, 2, 96), lam, [0, 10])
    with pytest.raises(pkg.TscError, match="share a dtype"):
        f(q, q.half(), q, lam, [0, 10])
    with pytest.raises(pkg.TscError, match="unsupported dtype"):
        f(q.double(), q.double(), q.double(), lam, [0, 10])
    for bad in (torch.zeros(3), torch.zeros((1, 2)), torch.zeros(2, dtype=torch.float16)):
        with pytest.raises(pkg.TscError, match="lam must be"):
            f(q, q, q, bad, [0, 10])
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(pkg.TscError, match="scale"):
            f(q, q, q, lam, [0, 10], scale=scale)
    with pytest.raises(pkg.TscError, match="out has the wrong"):
        f(q, q, q, lam, [0, 10], out=_t(9))
    with pytest.raises(pkg.TscError, match="contiguous"):
        f(torch.zeros((10, 64, 2)).transpose(1, 2), q, q, lam, [0, 10])
    with pytest.raises(pkg.TscError, match="contiguous"):
        f(q, torch.zeros((1, 2, 64)).expand(10, 2, 64), q, lam, [0, 10])
    with pytest.raises(pkg.TscError, match="not on a GPU"):
        f(q, q, q, lam, [0, 10])


def test_c_entry_points_without_a_gpu(pkg):
    lib = pkg.load_library()
    P = ctypes.c_void_p
    ws = lib.tsc_diff_attention_workspace_bytes
    assert ws(2, 1, 1, 40000, 12, 128, 1, 40000, 0) > 0  # one query: shared out over the keys
    assert ws(2, 1, 20000, 20000, 12, 128, 20000, 20000, 0) == 0
    assert ws(2, 1, 100, 100, 12, 128, 100, 100, 1) >= 2 * 12 * 100 * 4
    assert ws(2, 0, 0, 0, 12, 128, 0, 0, 0) == 0
    for bad in ((3, 1, 1, 1, 1, 64, 1, 1, 0), (0, 1, 1, 1, 1, 32, 1, 1, 0), (0, -1, 1, 1, 1, 64, 1, 1, 0),
                (0, 1, 2 ** 31, 1, 1, 64, 1, 1, 0), (0, 1, 1, 1, 0, 64, 1, 1, 0), (0, 1, 1, 1, 1, 64, -1, 1, 0),
                (0, 1, 1, 1, 1, 64, 1, -1, 0)):
        assert ws(*bad) == -1 and lib.tsc_last_error(), bad
    st = lib.tsc_diff_attention(None, 0, P(16), P(16), P(16), 64, 64, 64, P(16), P(16), P(16), 1, 1, 1,
                                1, 64, 0.0, 1, 1, 0, None, P(16), None, None)
    assert st == 1 and b"null context" in lib.tsc_last_error()
    st = lib.tsc_diff_attention_backward(None, 0, P(16), P(16), P(16), 64, 64, 64, P(16), P(16), P(16),
                                         1, 1, 1, 1, 64, 0.0, 1, 1, 0, P(16), P(16), P(16), P(16),
                                         P(16), P(16), P(16), None)
    assert st == 1 and b"null context" in lib.tsc_last_error()


def test_fp32_grids_of_128_rows_are_not_split(pkg):
    """In fp32 only blocks of 32 queries take a sequence's keys in parts.  Grids of 193 to 255 blocks of
    128 have the other kernel and fewer blocks than CUs: no parts, so no scratch, however uneven the
    keys are; smaller grids on long keys have parts."""
    ws = pkg.load_library().tsc_diff_attention_workspace_bytes
    between = 0
    for d in (64, 128):
        for b in range(1, 41):
            for h in (1, 2, 3, 5, 8, 12, 16, 24):
                for longest in (1, 64, 100, 128, 300, 640, 1500, 4000):
                    blocks = -(-longest // 128) * h * b
                    for total_kv, most in ((2000, 1500), (4000, 3000), (40000, 30000), (90 * b, 90)):
                        if 192 < blocks < 256:
                            between += 1
                            args = (0, b, longest * b, total_kv, h, d, longest, most, 0)
                            assert ws(*args) == 0, args
    assert between > 500
    assert ws(0, 1, 1, 40000, 12, 64, 1, 40000, 0) > 0


def test_scratch_of_a_gradient_without_queries(pkg):
    """dk, dv and dlambda are written all the same, from a partial sum of each block of keys."""
    ws = pkg.load_library().tsc_diff_attention_workspace_bytes
    assert ws(2, 2, 0, 500, 3, 64, 0, 300, 1) > 0 and ws(2, 2, 0, 500, 3, 64, 0, 300, 0) == 0
    assert ws(2, 0, 10, 10, 3, 64, 10, 10, 1) == 0


def test_scratch_of_parts_stays_near_the_inputs(pkg):
    """Every query has scratch for the longest sequence's parts: at most four times what q, k, v and out
    take, or 64 MB."""
    ws = pkg.load_library().tsc_diff_attention_workspace_bytes
    split = 0
    for code, size in ((0, 4), (1, 2), (2, 2)):
        for d in (64, 128):
            for h in (1, 2, 4, 8):
                for b in (1, 3, 16, 64, 250):
                    for longest in (1, 32, 128, 1000):
                        for kv in (3000, 220000, 4000000):
                            tq, tkv = b * longest, kv + 148 * (b - 1)
                            got = ws(code, b, tq, tkv, h, d, longest, kv, 0)
                            assert got <= max(64 << 20, 8 * (tq + tkv) * h * d * size), (code, d, h, b, longest, kv)
                            split += got > 0
    assert split > 200
    assert ws(1, 64, 8192, 229376, 1, 64, 128, 220000, 0) > 0


def test_scales_beyond_fp32_are_refused(pkg):
    """The kernels take the scale in fp32, where 0 means the default."""
    q, lam = _t(10), torch.zeros(2)
    for scale in (1e-46, 1e39, float("inf")):
        with pytest.raises(pkg.TscError, match="scale"):
            pkg.sparse_diff_attention(q, q, q, lam, [0, 10], scale=scale)
    with pytest.raises(pkg.TscError, match="not on a GPU"):  # this one is taken
        pkg.sparse_diff_attention(q, q, q, lam, [0, 10], scale=1e-30)


def test_scales_whose_powers_of_two_overflow_are_refused(pkg):
    """Scores are multiplied with scale log2(e), which fp32 has to hold: 2^128 / log2(e) is 2.3587e38."""
    f, q = pkg.sparse_diff_attention, _t(10)
    for scale in (2.36e38, 3.4e38):
        with pytest.raises(pkg.TscError, match="scale"):
            f(q, q, q, torch.zeros(2), [0, 10], scale=scale)
    for scale in (2.35e38, 1e-45):
        with pytest.raises(pkg.TscError, match="not on"):
            f(q, q, q, torch.zeros(2), [0, 10], scale=scale)
