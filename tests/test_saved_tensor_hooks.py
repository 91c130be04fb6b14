"""What the gradient calls are given where hooks on saved tensors (torch.autograd.graph.saved_tensors_hooks,
save_on_cpu) give back the values in another layout: the C calls are recorded on the CPU, and what each would
read, by the pointer and the row stride that it is given, is compared with the values that were saved."""
import ctypes
import importlib

import numpy as np
import pytest
import torch

SLACK = 4096  # values around what a hook gives back: a wrong stride reads NaN there, and nothing outside


def _padded(t):
    buf = torch.full((t.numel() + 2 * SLACK,), float("nan"), dtype=t.dtype)
    return buf[SLACK:SLACK + t.numel()]


def _contiguous(t):
    """What offloading gives back of a slice."""
    return _padded(t).view(t.shape).copy_(t) if t.is_floating_point() else t.clone()


def _transposed(t):
    """The last axis outermost."""
    if not t.is_floating_point() or t.dim() < 2:
        return t.clone()
    return _padded(t).view(t.shape[-1], *t.shape[:-1]).movedim(0, -1).copy_(t)


LAYOUTS = [_contiguous, _transposed]


class _Recorder:
    """Takes the place of the library: keeps the arguments of its calls."""

    def __init__(self, at_call):
        self.at_call = at_call

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("workspace_bytes"):
                return 64
            self.at_call(name, [getattr(a, "value", a) for a in args])
            return 0

        return call


def _read(pointer, rows, cols, ld):
    """(rows, cols) fp32 values at a host address, rows ld apart."""
    assert pointer % 4 == 0
    flat = np.ctypeslib.as_array((ctypes.c_float * ((rows - 1) * ld + cols)).from_address(pointer))
    return torch.from_numpy(np.lib.stride_tricks.as_strided(flat, (rows, cols), (4 * ld, 4)).copy())


@pytest.fixture
def record(pkg, monkeypatch):
    """record(at_call): CPU tensors pass for a GPU's and calls of the library go to at_call(name, arguments)."""
    ops = pkg.ops

    def start(at_call):
        monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
        monkeypatch.setattr(ops, "_cu_seqlens", lambda cu, total, dev, what: (None, torch.tensor(cu, dtype=torch.int32)))
        monkeypatch.setattr(ops._lib, "stream_handle", lambda dev: (_Recorder(at_call), None))

    return start


def _step(leaf, call, layout, at):
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), layout):
        o = call()
    torch.autograd.backward(o, [torch.ones_like(t) for t in o])
    assert leaf.grad is not None and at


@pytest.mark.parametrize("layout", LAYOUTS)
def test_window_attention(pkg, record, layout):
    lens, h, hk, d = [5, 7], 4, 2, 64
    n = sum(lens)
    qkv = torch.randn((n, h + 2 * hk, d)).requires_grad_()
    seen = []

    def at_call(name, a):
        if name != "tsc_window_attention_backward":
            return
        seen.append(name)
        for i, (lo, hi) in enumerate(((0, h), (h, h + hk), (h + hk, h + 2 * hk))):
            got = _read(a[2 + i], n, (hi - lo) * d, a[5 + i])
            assert a[2 + i] % 16 == 0 and a[5 + i] % 4 == 0
            assert torch.equal(got, qkv.detach()[:, lo:hi].flatten(1)), "qkv"[i]

    record(at_call)
    _step(qkv, lambda: [pkg.sparse_window_attention(qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:], 3, [0, 5, 12])],
          layout, seen)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_norms(pkg, record, layout):
    n, c = 12, 32
    x, y = torch.randn((n, c)).requires_grad_(), torch.randn((n, c))
    mod = torch.randn((2, 6, c)).requires_grad_()
    seen = []

    def at_call(name, a):
        if name != "tsc_gated_norm_backward":
            return
        seen.append(name)
        for what, at, ld, want in (("x", 2, c, x), ("y", 3, c, y)):
            assert torch.equal(_read(a[at], n, c, ld), want.detach()), what
        for what, at, i in (("gate", 11, 2), ("scale", 17, 4), ("shift", 19, 3)):
            assert torch.equal(_read(a[at], 2, c, a[at + 1]), mod.detach()[:, i]), what

    record(at_call)
    _step(mod, lambda: pkg.gated_residual_norm(x, y, [0, 5, 12], mod[:, 2], scale=mod[:, 4], shift=mod[:, 3]), layout, seen)


@pytest.mark.parametrize("layout", [lambda t: t.double() if t.is_floating_point() else t,
                                    lambda t: t[:-1].clone()])
def test_other_types_and_shapes_are_refused(pkg, record, layout):
    n, c = 12, 32
    x, mod = torch.randn((n, c)).requires_grad_(), torch.randn((2, 6, c)).requires_grad_()
    q = torch.randn((n, 2, 64)).requires_grad_()
    backward = []
    record(lambda name, a: backward.append(name) if name.endswith("backward") else None)
    for call in (lambda: pkg.modulated_norm(x, [0, 5, 12], mod[:, 1], mod[:, 0]),
                 lambda: pkg.sparse_window_attention(q, q, q, 3, [0, 5, 12])):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), layout):
            o = call()
        with pytest.raises(pkg.TscError, match="came back as"):
            o.sum().backward()
    assert not backward


@pytest.mark.parametrize("layout", LAYOUTS)
def test_group_norm(pkg, record, monkeypatch, layout):
    n, c, groups = 12, 32, 4
    x = torch.randn((n, c)).requires_grad_()
    seen = []

    def at_call(name, a):
        if name == "tsc_groupnorm":
            stats = np.ctypeslib.as_array((ctypes.c_float * (2 * groups * 2)).from_address(a[13]))
            stats[:] = np.arange(stats.size)
        if name != "tsc_groupnorm_backward":
            return
        seen.append(name)
        assert torch.equal(_read(a[3], n, c, c), x.detach())
        assert torch.equal(_read(a[13], 2, 2 * groups, 2 * groups).flatten(), torch.arange(4.0 * groups))

    record(at_call)
    monkeypatch.setattr(pkg.ops, "_dev", lambda *ts: 0)
    _step(x, lambda: [pkg.group_norm(x, groups, cu_rows=[0, 5, 12])], layout, seen)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_diff_attention(pkg, record, layout):
    n, h, d = 12, 2, 64
    qkv = torch.randn((n, 3, h, d)).requires_grad_()
    lam, cu = torch.rand(h), torch.tensor([0, 5, 12], dtype=torch.int32)
    seen, sizes = [], {20: 2 * n * h * d, 21: 2 * h * n}  # maps, lse

    def at_call(name, a):
        if name == "tsc_diff_attention":
            for at, size in sizes.items():
                values = np.ctypeslib.as_array((ctypes.c_float * size).from_address(a[at + 2]))
                values[:] = np.arange(size)
        if name != "tsc_diff_attention_backward":
            return
        seen.append(name)
        for i in range(3):
            assert torch.equal(_read(a[2 + i], n, h * d, a[5 + i]), qkv.detach()[:, i].flatten(1)), "qkv"[i]
        for at, size in sizes.items():
            assert torch.equal(_read(a[at], 1, size, size)[0], torch.arange(float(size)))

    record(at_call)
    f = importlib.import_module(pkg.__name__ + ".autograd").DiffAttention
    _step(qkv, lambda: [f.apply(qkv[:, 0], qkv[:, 1], qkv[:, 2], lam, cu, cu, 2, 0.0, 7, 7)], layout, seen)
