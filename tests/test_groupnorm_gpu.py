"""Group norm (and SiLU) over the rows of each sample and its gradients, against the definition in
64 bits on the same rounded inputs.

Tolerances.  An output is rounded once to its type: eps/2 of its value (plus the smallest step near
zero).  Before that the kernel computes in fp32: the mean of n values is a sum whose roundings go by
its terms, however they cancel: |error| <= k 2^-24 sum |x| / n for k roundings on the way of a term.
So x - mean carries roundings of 2^-24 of |x| + mean |x|, and what follows fewer than 32 of 2^-24 of the terms (SiLU's exponential included: its
argument's rounding times |h|, |h| < 8 here): 2^-19 of the sum of the terms' sizes.  Sums over rows are fp32 runs of at most 16 rows
per thread at the sizes here, at most 8 merges, and fp64 beyond: within the same 2^-19 of the sum of the sizes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -19
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _half(t, dtype):
    """Half a step of dtype at the values t."""
    f = torch.finfo(dtype)
    return t.abs() * (f.eps / 2) + f.smallest_normal * f.eps


def _make(lens, c, dtype, seed, offset=0.7):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    x = torch.randn((n, c), generator=g, dtype=torch.float64)
    x = x * (1 + 0.3 * torch.randn(c, generator=g, dtype=torch.float64)) + offset * torch.randn(
        c, generator=g, dtype=torch.float64)
    w = 1 + 0.1 * torch.randn(c, generator=g, dtype=torch.float64)
    b = 0.1 * torch.randn(c, generator=g, dtype=torch.float64)
    dy = torch.randn((n, c), generator=g, dtype=torch.float64)
    return [t.to(dtype) for t in (x, w, b, dy)]


def _oracle(x, groups, w, b, cu, eps, silu, dy=None):
    """Everything in fp64 on the CPU: dict of y, the gradients, and the tolerances' sizes."""
    x = x.double()
    n, c = x.shape
    w = torch.ones(c, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.double()
    r = {k: torch.zeros_like(x) for k in ("y", "ty", "dx", "tdx")}
    r.update({k: torch.zeros(c, dtype=torch.float64) for k in ("dw", "tdw", "db", "tdb")})

    def ch(t):
        return t.repeat_interleave(c // groups)

    for lo, hi in zip(cu, cu[1:]):
        if hi == lo:
            continue
        xs = x[lo:hi]
        m = (hi - lo) * (c // groups)
        mean = ch(xs.reshape(hi - lo, groups, -1).mean((0, 2)))
        var = ch(((xs - mean) ** 2).reshape(hi - lo, groups, -1).mean((0, 2)))
        rstd = 1 / torch.sqrt(var + eps)
        xh = (xs - mean) * rstd
        h = xh * w + b
        sg = 1 / (1 + torch.exp(-h))
        r["y"][lo:hi] = h * sg if silu else h
        amean = ch(xs.abs().reshape(hi - lo, groups, -1).mean((0, 2)))
        txh = (xs.abs() + amean) * rstd  # what xh's rounding goes by
        r["ty"][lo:hi] = txh * w.abs() + b.abs() + h.abs()
        if dy is not None:
            d = dy[lo:hi].double()
            ad = d.abs() * (1 + h.abs()) * (1 + txh * w.abs() / 2)  # size of dh's roundings
            dh = d * (sg * (1 + h * (1 - sg))) if silu else d
            r["db"] += dh.sum(0)
            r["dw"] += (dh * xh).sum(0)
            r["tdb"] += ad.sum(0)
            tw = ad * (xh.abs() + txh)
            r["tdw"] += tw.sum(0)

            def group(t):
                return ch((t * w).sum(0).reshape(groups, -1).sum(1) / m)

            def agroup(t):
                return ch((t * w.abs()).sum(0).reshape(groups, -1).sum(1) / m)

            r["dx"][lo:hi] = rstd * (w * dh - group(dh) - xh * group(dh * xh))
            r["tdx"][lo:hi] = rstd * (w.abs() * ad + agroup(ad) + (xh.abs() + txh) * agroup(tw))
    return r


def _close(got, want, size, dtype, what):
    got = got.detach().double().cpu()
    tol = _half(want, dtype) + F32 * size
    worst = ((got - want).abs() / tol).max().item() if want.numel() else 0.0
    print(f"    {what}: worst error {worst:.3f} of its tolerance", flush=True)
    assert worst <= 1.0, (what, worst)


def _cu(lens):
    return np.cumsum([0] + list(lens)).tolist()


SHAPES = [([1], 32, 32), ([2], 64, 2), ([700, 0, 1, 331], 64, 32), ([5000], 32, 8),
          ([63, 64, 65, 0, 0], 72, 12), ([257, 900], 100, 20), ([311], 13, 13), ([40, 1000], 33, 1),
          ([1500, 20], 1024, 32), ([300], 1000, 8), ([97], 48, 3), ([1] * 130, 16, 4), ([0, 17], 6, 3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,c,groups", SHAPES)
@pytest.mark.parametrize("silu", [False, True])
def test_forward_and_gradients(pkg, dev, dtype, lens, c, groups, silu):
    x, w, b, dy = _make(lens, c, dtype, c + len(lens))
    cu = _cu(lens)
    print(f"  group norm {dtype} {lens[:6]} C={c} G={groups} silu={silu}", flush=True)
    r = _oracle(x, groups, w, b, cu, 1e-5, silu, dy)
    xd, wd, bd = (t.to(dev) for t in (x, w, b))
    y0 = pkg.group_norm(xd, groups, wd, bd, cu, silu=silu)
    leaves = [t.requires_grad_() for t in (xd, wd, bd)]
    y = pkg.group_norm(*leaves[:1], groups, *leaves[1:], cu, silu=silu)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(dev))
    assert torch.equal(y0, y)
    _close(y, r["y"], r["ty"], dtype, "y")
    _close(dx, r["dx"], r["tdx"], dtype, "dx")
    _close(dw, r["dw"], r["tdw"], dtype, "dweight")
    _close(db, r["db"], r["tdb"], dtype, "dbias")


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_missing_parameters(pkg, dev, which):
    lens, c, groups, dtype = [300, 211], 96, 32, torch.float32
    x, w, b, dy = _make(lens, c, dtype, 5)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    r = _oracle(x, groups, w, b, _cu(lens), 1e-5, True, dy)
    leaves = [None if t is None else t.to(dev).requires_grad_() for t in (x, w, b)]
    y = pkg.group_norm(leaves[0], groups, leaves[1], leaves[2], _cu(lens), silu=True)
    y.backward(dy.to(dev))
    _close(y, r["y"], r["ty"], dtype, "y")
    _close(leaves[0].grad, r["dx"], r["tdx"], dtype, "dx")
    if w is not None:
        _close(leaves[1].grad, r["dw"], r["tdw"], dtype, "dweight")
    if b is not None:
        _close(leaves[2].grad, r["db"], r["tdb"], dtype, "dbias")


def test_gradient_against_differences(pkg, dev):
    """The definition's central differences in 64 bits along random directions (step 1e-4: their own
    error is below 1e-7 of the sizes) against the kernel's gradients."""
    lens, c, groups, dtype = [40, 23], 24, 6, torch.float32
    cu = _cu(lens)
    x, w, b, dy = _make(lens, c, dtype, 9)
    r = _oracle(x, groups, w, b, cu, 1e-5, True, dy)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)]
    pkg.group_norm(leaves[0], groups, leaves[1], leaves[2], cu, silu=True).backward(dy.to(dev))
    g = torch.Generator().manual_seed(1)
    for i, (grad, size) in enumerate((("dx", "tdx"), ("dw", "tdw"), ("db", "tdb"))):
        base = [t.double() for t in (x, w, b)]
        u = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        f = []
        for sign in (1, -1):
            moved = list(base)
            moved[i] = base[i] + sign * 1e-4 * u
            f.append((_oracle(moved[0], groups, moved[1], moved[2], cu, 1e-5, True)["y"]
                      * dy.double()).sum().item())
        want = (f[0] - f[1]) / 2e-4
        got = (leaves[i].grad.cpu().double() * u).sum().item()
        tol = ((_half(r[grad], dtype) + F32 * r[size]) * u.abs()).sum().item()
        print(f"  {grad}: {got:.6f} {want:.6f}, off by {abs(got - want) / tol:.3f} of the tolerance", flush=True)
        assert abs(got - want) <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("c,lens", [(32, [1, 0, 40, 1]), (13, [1])])
def test_group_of_one_value_has_no_gradient(pkg, dev, dtype, silu, c, lens):
    """Its norm is 0 whatever the value: dx is zero, not what gamma dh - A rounds to."""
    g = torch.Generator().manual_seed(c)
    cu = [0, *torch.tensor(lens).cumsum(0).tolist()]
    x, w, b, dy = (torch.randn(s, generator=g).to(dtype).to(dev) for s in ((cu[-1], c), (c,), (c,), (cu[-1], c)))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(pkg.group_norm(*leaves[:1], c, *leaves[1:], cu_rows=cu, silu=silu), leaves, dy)
    for lo, hi in zip(cu, cu[1:]):
        assert bool(dx[lo:hi].any()) == (hi - lo > 1)
    assert db.any() and bool(dw.any()) == (max(lens) > 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_spread_beside_a_large_mean(pkg, dev, dtype):
    """Values near 1000 with a spread of 1 (bf16: 16 steps of 8): the variance must not be lost.  The
    sizes in the tolerance grow with |x| + |mean|."""
    g = torch.Generator().manual_seed(2)
    x = (1000 + torch.randn((4000, 32), generator=g) * (1 if dtype == torch.float32 else 30)).to(dtype)
    r = _oracle(x, 4, None, None, [0, 4000], 1e-5, False)
    y = pkg.group_norm(x.to(dev), 4)
    _close(y, r["y"], r["ty"], dtype, "y")
    y = pkg.group_norm(torch.full((500, 8), 1e6, device=dev), 2)  # no spread at all
    assert not y.any()


def test_infinities_and_nan_stay_in_their_group(pkg, dev):
    lens = [400, 300, 5]
    cu = _cu(lens)
    x, w, b, _ = _make(lens, 64, torch.float32, 3)
    xd = x.to(dev)
    clean = pkg.group_norm(xd, 8, w.to(dev), b.to(dev), cu, silu=True)
    xd[17, 3] = float("inf")     # sample 0, group 0
    xd[450, 63] = float("nan")   # sample 1, group 7
    y = pkg.group_norm(xd, 8, w.to(dev), b.to(dev), cu, silu=True)
    assert y[:400, :8].isnan().all() and y[400:700, 56:].isnan().all()
    y[:400, :8] = clean[:400, :8]
    y[400:700, 56:] = clean[400:700, 56:]
    assert torch.equal(y, clean)


def test_rows_outside_every_sample(pkg, dev):
    """Zero in a new result, left alone in a given one; the gradient is zero there; in place works."""
    x, w, b, dy = _make([100], 40, torch.float16, 4)
    cu = [7, 30, 30, 81]
    want = pkg.group_norm(x[7:81].contiguous().to(dev), 5, w.to(dev), b.to(dev), [0, 23, 23, 74])
    xd = x.to(dev).requires_grad_()
    y = pkg.group_norm(xd, 5, w.to(dev), b.to(dev), torch.tensor(cu, device=dev))
    assert not y[:7].any() and not y[81:].any()
    dx, = torch.autograd.grad(y, xd, dy.to(dev))
    assert not dx[:7].any() and not dx[81:].any() and dx[7:81].any()
    r = _oracle(x, 5, w, b, cu, 1e-5, False)
    _close(y[7:81], r["y"][7:81], r["ty"][7:81], torch.float16, "y")
    _close(want, r["y"][7:81], r["ty"][7:81], torch.float16, "y alone")
    out = torch.full_like(xd, 5.0).detach()
    pkg.group_norm(xd.detach(), 5, w.to(dev), b.to(dev), cu, out=out)
    assert bool((out[:7] == 5).all()) and bool((out[81:] == 5).all())
    assert torch.equal(out[7:81], y[7:81])
    inplace = x.to(dev)
    got = pkg.group_norm(inplace, 5, w.to(dev), b.to(dev), cu, out=inplace)
    assert got is inplace and torch.equal(got[7:81], y[7:81])
    assert torch.equal(got[:7], x[:7].to(dev))


def test_dense_batches_and_empty_inputs(pkg, dev):
    x, w, b, dy = _make([3 * 4 * 5 * 6], 32, torch.bfloat16, 6)
    xd = x.to(dev).view(3, 4, 5, 6, 32)
    y = pkg.group_norm(xd, 8, w.to(dev), b.to(dev), silu=True)
    flat = pkg.group_norm(xd.view(-1, 32), 8, w.to(dev), b.to(dev), [0, 120, 240, 360], silu=True)
    assert y.shape == xd.shape and torch.equal(y.view(-1, 32), flat)
    for shape in ((0, 32), (0, 7, 32), (2, 0, 32)):
        e = torch.zeros(shape, dtype=torch.bfloat16, device=dev).requires_grad_()
        we = w.to(dev).requires_grad_()
        z = pkg.group_norm(e, 8, we)
        z.backward(torch.zeros_like(z))
        assert z.shape == e.shape and e.grad.shape == e.shape and not we.grad.any()
    assert not pkg.group_norm(torch.ones((4, 32), device=dev), 8, cu_rows=[0]).any()  # no samples


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_unaligned_buffers(pkg, dev, dtype):
    """Rows of whole 16 bytes that start at no multiple of 16: the shorter loads, same tolerance."""
    x, w, b, dy = _make([500], 64, dtype, 8)
    base = torch.empty(500 * 64 + 8, dtype=dtype, device=dev)
    r = _oracle(x, 16, w, b, [0, 500], 1e-5, True, dy)
    for shift in (1, 2, 4):
        v = base[shift:shift + 500 * 64].view(500, 64)
        v.copy_(x)
        leaf = v.detach().requires_grad_()
        y = pkg.group_norm(leaf, 16, w.to(dev), b.to(dev), silu=True)
        dx, = torch.autograd.grad(y, leaf, dy.to(dev))
        _close(y, r["y"], r["ty"], dtype, f"y at +{shift}")
        _close(dx, r["dx"], r["tdx"], dtype, f"dx at +{shift}")


def test_same_bits_each_time_on_any_stream_and_in_a_graph(pkg, dev):
    """Sums have one order; a captured training step replays to the eager bits with new inputs, with
    eager work in between; two captured graphs share nothing."""
    lens, c, groups = [3000, 1700], 128, 32
    cu = torch.tensor(_cu(lens), dtype=torch.int32, device=dev)
    x, w, b, dy = (t.to(dev) for t in _make(lens, c, torch.bfloat16, 11))

    def step(x, w, b, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = pkg.group_norm(leaves[0], groups, leaves[1], leaves[2], cu, silu=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graphs = []
    for i in range(2):
        xs = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(xs, w, b, dy)
        graphs.append((g, xs, outs))
    for rep in range(3):
        for i, (g, xs, outs) in enumerate(graphs):
            new = x * (1 + 0.1 * rep) + i
            xs.copy_(new)
            g.replay()
        for i, (g, xs, outs) in enumerate(graphs):
            eager = step(x * (1 + 0.1 * rep) + i, w, b, dy)
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(outs, eager)), (rep, i)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("c,groups", [(64, 32), (100, 20), (1024, 8)])
def test_many_uneven_samples(pkg, dev, dtype, c, groups):
    """Hundreds of samples, many of them empty, starting and ending at, before and after tile borders
    (tiles are runs of equal length): every (tile, sample) meeting has its slot."""
    rng = np.random.default_rng(c)
    lens = rng.choice([0, 0, 1, 2, 7, 31, 32, 33, 64, 130], 300).tolist() + [900, 0, 0, 512, 0]
    cu = [5 + v for v in _cu(lens)]
    x, w, b, dy = _make([cu[-1] + 9], c, dtype, c)
    r = _oracle(x, groups, w, b, cu, 1e-5, True, dy)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)]
    y = pkg.group_norm(leaves[0], groups, leaves[1], leaves[2], torch.tensor(cu, device=dev), silu=True)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(dev))
    assert not y[:5].any() and not y[cu[-1]:].any() and not dx[:5].any() and not dx[cu[-1]:].any()
    _close(y, r["y"], r["ty"], dtype, "y")
    _close(dx, r["dx"], r["tdx"], dtype, "dx")
    _close(dw, r["dw"], r["tdw"], dtype, "dweight")
    _close(db, r["db"], r["tdb"], dtype, "dbias")


def test_samples_times_slabs_past_2_32_threads(pkg, dev):
    """140000 samples, all but the last empty, and 65 slabs of 64 channels (an odd count: no vectors): 9.1
    million blocks of 512 threads.  The rows' values and gradients are those of the one sample alone."""
    n, b, c, groups = 300, 140000, 4097, 17
    cu = torch.zeros(b + 1, dtype=torch.int32, device=dev)
    cu[b] = n
    x, w, bias, dy = (t.to(dev) for t in _make([n], c, torch.bfloat16, 15))
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    r = _oracle(x.detach().cpu(), groups, w.detach().cpu(), bias.detach().cpu(), [0, n], 1e-5, True, dy.cpu())
    y = pkg.group_norm(x, groups, w, bias, cu, silu=True)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    for got, want, size in ((y, "y", "ty"), (dx, "dx", "tdx"), (dw, "dw", "tdw"), (db, "db", "tdb")):
        _close(got, r[want], r[size], torch.bfloat16, want)


def test_device_offsets_are_not_read_back(pkg, dev):
    x, w, b, _ = _make([600], 64, torch.float32, 12)
    xd = x.to(dev)
    cu = torch.tensor([0, 200, 600], dtype=torch.int32, device=dev)
    want = pkg.group_norm(xd, 32, cu_rows=[0, 200, 600])
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = pkg.group_norm(xd, 32, cu_rows=cu)
    finally:
        torch.cuda.set_sync_debug_mode(0)
    assert torch.equal(got, want)


def test_more_than_2_31_values(pkg, dev):
    """Offsets past 32 bits: sampled rows against fp64 statistics of each sample."""
    c, groups = 64, 16
    n = 2 ** 31 // c + 5000
    cu = [0, 1000, n - 3000, n]
    x = torch.empty((n, c), dtype=torch.float16, device=dev)
    for i in range(0, n, 1 << 22):
        x[i:i + (1 << 22)].normal_()
    x[n - 3000:] *= 3
    y = pkg.group_norm(x, groups, cu_rows=cu)
    torch.cuda.synchronize()
    for lo, hi in zip(cu, cu[1:]):
        s1 = torch.zeros(groups, dtype=torch.float64, device=dev)
        s2 = torch.zeros_like(s1)
        for i in range(lo, hi, 1 << 22):
            t = x[i:min(hi, i + (1 << 22))].double().view(-1, groups, c // groups)
            s1 += t.sum((0, 2))
            s2 += (t * t).sum((0, 2))
        m = (hi - lo) * (c // groups)
        mean, var = s1 / m, s2 / m - (s1 / m) ** 2
        rows = torch.cat([torch.arange(lo, lo + 500), torch.arange(hi - 500, hi)]).to(dev)
        t = x[rows].double().view(-1, groups, c // groups)
        want = ((t - mean[:, None]) / (var[:, None] + 1e-5).sqrt()).view(-1, c).cpu()
        # runs of up to 2000 rows per thread: their fp32 means and M2 are within 2^-24 * 2000 / 8
        _close(y[rows], want, 2.0 ** 5 * (want.abs() + 1), torch.float16, f"rows {lo}..{hi}")


def test_sparse_group_norm_class(pkg, dev):
    g = torch.Generator().manual_seed(3)
    coords = torch.cat([torch.cat([torch.full((n, 1), i), torch.randint(0, 64, (n, 3), generator=g)], 1)
                        for i, n in enumerate((50, 70))]).int()
    x, w, b, _ = _make([50, 70], 32, torch.bfloat16, 14)
    st = pkg.SparseTensor(x.to(dev), coords.to(dev))
    y = pkg.SparseGroupNorm(8, w.to(dev), b.to(dev), silu=True)(st)
    r = _oracle(x, 8, w, b, [0, 50, 120], 1e-5, True)
    _close(y.feats, r["y"], r["ty"], torch.bfloat16, "y")
    assert y.coords is st.coords and y.cu_rows is st.cu_rows


def test_refusals_on_the_device(pkg, dev):
    x = torch.zeros((10, 12), device=dev)
    with pytest.raises(pkg.TscError, match="contiguous"):
        pkg.group_norm(torch.zeros((10, 24), device=dev)[:, ::2], 3)
    with pytest.raises(pkg.TscError, match="non-decreasing"):
        pkg.group_norm(x, 3, cu_rows=[0, 7, 5, 10])
    with pytest.raises(pkg.TscError, match="non-decreasing"):
        pkg.group_norm(x, 3, cu_rows=[0, 11])
    with pytest.raises(pkg.TscError, match="cu_rows goes with"):
        pkg.group_norm(x.view(2, 5, 12), 3, cu_rows=[0, 10])
    with pytest.raises(pkg.TscError, match="eps"):
        pkg.group_norm(x, 3, eps=-1.0)
    with pytest.raises(pkg.TscError, match="gradients"):
        pkg.group_norm(x.clone().requires_grad_(), 3, out=x)
    base = torch.zeros(12 * 11, device=dev)
    with pytest.raises(pkg.TscError, match="overlaps"):
        pkg.group_norm(base[:120].view(10, 12), 3, out=base[12:].view(10, 12))


def test_a_saved_input_that_is_written_is_refused(pkg, dev):
    """x is saved for the gradient: once any of the library's operators has written to it through `out`,
    the gradient is refused, as after torch's own in-place operations."""
    n, c = 24, 64
    other = torch.randn((n, c), device=dev)
    w = torch.ones(c, device=dev, requires_grad=True)
    lam = torch.ones(1, device=dev)
    nbr = torch.full((n, 27), -1, dtype=torch.int32, device=dev)
    wc = torch.zeros((c, 3, 3, 3, c), device=dev)

    def norm(out):
        pkg.group_norm(other, 8, out=out)

    def attend(out):
        o = other.view(n, 1, c)
        pkg.sparse_diff_attention(o, o, o, lam, [0, n], out=out.view(n, 1, c))

    def attend_one_map(out):
        o = other.view(n, 1, c)
        pkg.sparse_attention(o, o, o, [0, n], out=out)

    writers = [norm, attend, attend_one_map, lambda out: pkg.layer_norm(other, out=out),
               lambda out: pkg.silu(other, out=out), lambda out: pkg.add(other, other, out=out),
               lambda out: pkg.sparse_linear(other, torch.eye(c, device=dev), out=out),
               lambda out: pkg.sparse_conv3d(other, wc, None, nbr, out=out),
               lambda out: pkg.sparse_resblock(other, nbr, wc, None, wc, None, out=out)]
    for i, write in enumerate(writers):
        x = torch.randn((n, c), device=dev)
        y = pkg.group_norm(x, 8, w)
        with torch.no_grad():
            write(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    x = torch.randn((n, c), device=dev)
    y = pkg.group_norm(x, 8, w)
    with pytest.raises(pkg.TscError):  # refused, so not written
        pkg.group_norm(other, 8, eps=-1.0, out=x)
    y.sum().backward()
    leaf = torch.zeros((n, c), device=dev, requires_grad=True)
    with pytest.raises(pkg.TscError, match="gradients"):
        pkg.group_norm(other, 8, out=leaf)
    with torch.no_grad():
        pkg.group_norm(other, 8, out=leaf)
    with torch.inference_mode():
        pkg.group_norm(other, 8, out=torch.zeros((n, c), device=dev))


def test_c_calls_without_samples_or_rows(pkg, dev):
    """B = 0: every row is outside, zeroed with zero_rest or left as it was, and the parameters' gradients
    are sums over nothing; the same for N = 0.  Captured and replayed as well."""
    import ctypes
    import sys

    P = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
    mod = sys.modules["trellis2_amd._lib"]
    lib, h = mod.stream_handle(0)
    n, c = 1000, 37
    for code, dtype in ((0, torch.float32), (1, torch.float16), (2, torch.bfloat16)):
        x = torch.ones((n, c), dtype=dtype, device=dev)
        for rest in (0, 1):
            y, dx, dw, db = (torch.full_like(t, 5.0) for t in (x, x, x[0], x[0]))
            assert lib.tsc_groupnorm(h, code, P(x), None, 0, n, c, 1, None, None, 1e-5, 0, rest, None, None,
                                     P(y)) == 0
            assert lib.tsc_groupnorm_backward(h, code, P(x), P(x), None, 0, n, c, 1, None, None, 0, rest, None,
                                              None, P(dx), P(dw), P(db)) == 0
            assert bool((y == 5 * (1 - rest)).all()) and bool((dx == 5 * (1 - rest)).all())
            assert not dw.any() and not db.any()
        ws, st = torch.zeros(1 << 14, device=dev), torch.zeros(8, device=dev)
        dw, db = torch.full_like(x[0], 5.0), torch.full_like(x[0], 5.0)
        assert lib.tsc_groupnorm_backward(h, code, None, None, None, 2, 0, c, 1, None, None, 0, 1, P(st), P(ws),
                                          None, P(dw), P(db)) == 0
        assert not dw.any() and not db.any()
    y = torch.empty((n, c), device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert lib.tsc_groupnorm(mod.stream_handle(0)[1], 0, P(y), None, 0, n, c, 1, None, None, 1e-5, 0, 1, None,
                                 None, P(y)) == 0
    for _ in range(3):
        y.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert not y.any()


def test_c_gradients_over_inputs_are_refused(pkg, dev):
    """dgamma over gamma above all: blocks that make dx still read gamma when dgamma is written."""
    import ctypes
    import sys

    P = lambda t: ctypes.c_void_p(t.data_ptr())
    lib, h = sys.modules["trellis2_amd._lib"].stream_handle(0)
    n, c = 64, 32
    bufs = {k: torch.ones((n, c), device=dev) for k in ("x", "dy", "dx")}
    bufs.update({k: torch.ones(c, device=dev) for k in ("gamma", "beta", "dgamma", "dbeta")})
    stats, ws = torch.ones((1, 8, 2), device=dev), torch.zeros(1 << 16, device=dev)

    def call(**other):
        b = {**bufs, **other}
        return lib.tsc_groupnorm_backward(h, 0, P(b["dy"]), P(b["x"]), None, 1, n, c, 8, P(b["gamma"]), P(b["beta"]),
                                          0, 1, P(stats), P(ws), P(b["dx"]), P(b["dgamma"]), P(b["dbeta"]))

    assert call() == 0
    for over in ({"dgamma": bufs["gamma"]}, {"dbeta": bufs["gamma"]}, {"dbeta": bufs["beta"]},
                 {"dgamma": bufs["x"][-1]}, {"dbeta": bufs["dy"]}, {"dgamma": bufs["dx"]},
                 {"dbeta": bufs["dgamma"]}, {"dx": bufs["x"]}, {"dx": bufs["dy"]}, {"gamma": bufs["dx"][3]},
                 {"dgamma": stats}):
        assert call(**over) == 1 and b"overlap" in lib.tsc_last_error(), list(over)
