"""Refusals of group_norm that need no GPU: arguments are checked before any device call."""
import ctypes

import pytest
import torch


def test_group_norm_refuses_bad_arguments(pkg):
    x = torch.zeros((10, 12))
    with pytest.raises(pkg.TscError, match="do not divide"):
        pkg.group_norm(x, 5)
    with pytest.raises(pkg.TscError, match="do not divide"):
        pkg.group_norm(x, 0)
    with pytest.raises(pkg.TscError, match="do not divide"):
        pkg.group_norm(torch.zeros((3, 0)), 1)
    with pytest.raises(pkg.TscError, match=r"\(N, C\) or"):
        pkg.group_norm(torch.zeros(12), 3)
    with pytest.raises(pkg.TscError, match="weight and bias"):
        pkg.group_norm(x, 3, torch.ones(11))
    with pytest.raises(pkg.TscError, match="weight and bias"):
        pkg.group_norm(x, 3, torch.ones(12), torch.zeros(12, dtype=torch.float16))
    with pytest.raises(pkg.TscError, match="out has the wrong"):
        pkg.group_norm(x, 3, out=torch.zeros((9, 12)))
    with pytest.raises(pkg.TscError, match="unsupported dtype"):
        pkg.group_norm(x.double(), 3)
    with pytest.raises(pkg.TscError, match="not on a GPU"):
        pkg.group_norm(x, 3)


def test_workspace_bytes(pkg):
    lib = pkg.load_library()
    f = lib.tsc_groupnorm_workspace_bytes
    assert f(2, 2, 1000, 64, 32, 0) > 0
    assert f(2, 2, 1000, 64, 32, 1) >= f(2, 2, 1000, 64, 32, 0) + 8 * 64 * 2
    for bad in ((3, 1, 10, 64, 32, 0), (0, -1, 10, 64, 32, 0), (0, 1, -1, 64, 32, 0),
                (0, 1, 10, 64, 0, 0), (0, 1, 10, 64, 30, 0), (0, 1, 2 ** 31, 64, 32, 0),
                (0, 1, 10, 65537, 1, 0)):
        assert f(*bad) == -1, bad
        assert lib.tsc_last_error()


def test_null_context(pkg):
    lib = pkg.load_library()
    P = ctypes.c_void_p
    assert lib.tsc_groupnorm(None, 0, P(16), None, 1, 4, 8, 2, None, None, 1e-5, 0, 0, None, P(16),
                             P(16)) == 1
    assert b"null context" in lib.tsc_last_error()
    assert lib.tsc_groupnorm_backward(None, 0, P(16), P(16), None, 1, 4, 8, 2, None, None, 0, 0,
                                      P(16), P(16), P(64), None, None) == 1
    assert b"null context" in lib.tsc_last_error()


def test_cu_rows_of_a_sparse_tensor(pkg):
    coords = torch.tensor([[0, 1, 2, 3], [0, 4, 0, 1], [2, 0, 5, 0]], dtype=torch.int32)
    x = pkg.SparseTensor(torch.zeros((3, 8)), coords)
    assert x.cu_rows.tolist() == [0, 2, 2, 3] and x.cu_rows.dtype == torch.int32
    assert x.replace(torch.ones((3, 4))).cu_rows is x.cu_rows


def test_dual_tensors_are_refused(pkg):
    """There is no forward-mode derivative: a tangent is refused, not dropped."""
    import torch.autograd.forward_ad as fa

    with fa.dual_level():
        def dual(*shape):
            return fa.make_dual(torch.zeros(shape), torch.ones(shape))

        for args in ((dual(10, 12), 3), (torch.zeros(10, 12), 3, dual(12)),
                     (torch.zeros(10, 12), 3, None, dual(12))):
            with pytest.raises(pkg.TscError, match="forward-mode"):
                pkg.group_norm(*args)
            with torch.no_grad(), pytest.raises(pkg.TscError, match="forward-mode"):
                pkg.group_norm(*args)
        q = torch.zeros((10, 2, 64))
        args = [q, q, q, torch.zeros(2)]
        for i in range(4):
            some = [dual(*t.shape) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(pkg.TscError, match="forward-mode"):
                pkg.sparse_diff_attention(*some, [0, 10])


def test_cu_rows_needs_rows_grouped_by_sample(pkg):
    """Offsets cannot say which rows are a sample's where samples are mixed or out of order."""
    def tensor(samples, **kw):
        coords = torch.tensor([[b, i, 0, 0] for i, b in enumerate(samples)], dtype=torch.int32).reshape(-1, 4)
        return pkg.SparseTensor(torch.zeros((len(samples), 8)), coords, **kw)

    for mixed in ([1, 0, 1, 0], [0, 1, 0, 1], [1, 1, 0, 0], [0, 2, 1, 2], [2, 1, 0]):
        with pytest.raises(ValueError, match="grouped by sample"):
            tensor(mixed).cu_rows
    with pytest.raises(ValueError, match="grouped by sample"):  # a layout of other rows
        tensor([0, 0, 1], layout=[(0, 1), (1, 3)]).cu_rows
    with pytest.raises(ValueError, match="grouped by sample"):
        tensor([0, 0, 1], layout=[(1, 3), (0, 1)]).cu_rows
    assert tensor([0, 0, 3]).cu_rows.tolist() == [0, 2, 2, 2, 3]
    assert tensor([]).cu_rows.tolist() == [0, 0]
    x = tensor([0, 0, 1])
    assert x.cu_rows.tolist() == [0, 2, 3]
    other = tensor([0, 1, 1]).coords  # replace keeps the layout; other coordinates are looked at again
    with pytest.raises(ValueError, match="grouped by sample"):
        x.replace(torch.zeros((3, 8)), other).cu_rows
    same = x.replace(torch.zeros((3, 8)), x.coords.clone())
    assert same.cu_rows.tolist() == [0, 2, 3]


def test_cu_rows_has_every_sample_of_a_given_batch_size(pkg):
    """Empty samples after the last row's count too: the offsets pair with a condition's of the batch."""
    coords = torch.tensor([[0, 0, 0, 0], [0, 1, 0, 0], [1, 0, 0, 0]], dtype=torch.int32)
    x = pkg.SparseTensor(torch.zeros((3, 8)), coords, batch_size=4)
    assert x.cu_rows.tolist() == [0, 2, 3, 3, 3] and x.batch_size == 4
    assert x.replace(torch.zeros((3, 2))).cu_rows is x.cu_rows
    none = pkg.SparseTensor(torch.zeros((0, 8)), coords[:0], batch_size=2)
    assert none.cu_rows.tolist() == [0, 0, 0]


def test_workspace_of_no_samples(pkg):
    f = pkg.load_library().tsc_groupnorm_workspace_bytes
    assert f(0, 0, 10, 64, 32, 0) == 0 and f(2, 0, 0, 64, 32, 1) == 0
