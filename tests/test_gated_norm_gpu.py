"""The norms before and after a block and their gradients against the definition in 64 bits, with the
running bounds of _running.py.  A row's sums add a value at most 48 times (16 of a lane's, 6 over its
wave, 16 waves), a sample's sums at most 256 times (a block's rows and its waves; the blocks are added
up in fp64; rows here are at most 5000, 1024 blocks)."""
import numpy as np
import pytest
import torch

from tests._running import V, check

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
ROW, COL = 48, 256
NAMES = ("x", "y", "pw", "pb", "gate", "w", "b", "scale", "shift")


def _cu(lens):
    return np.cumsum([0] + list(lens)).tolist()


def _make(lens, c, dtype, seed, post="layer", affine=True, mod=True, n=None):
    g = torch.Generator().manual_seed(seed)
    n, b = sum(lens) if n is None else n, len(lens)

    def normal(*s):
        return torch.randn(s, generator=g)

    t = {"x": normal(n, c) * (1 + 0.3 * normal(c)) + 0.7 * normal(c),
         "y": normal(n, c) * (1 + 0.3 * normal(c)) + 0.7 * normal(c)}
    m = 0.3 * normal(b, 6, c)
    if affine:
        t["w"], t["b"] = 1 + 0.2 * normal(c), 0.2 * normal(c)
        if post:
            t["pw"], t["pb"] = 1 + 0.2 * normal(c), 0.2 * normal(c)
    t = {k: v.to(dtype) for k, v in t.items()}
    if mod:
        m = m.to(dtype)
        t["gate"], t["scale"], t["shift"] = m[:, 1], m[:, 3], m[:, 4]
    return t, {"dr": normal(n, c).to(dtype), "dh": normal(n, c).to(dtype)}


def _norm(x, kind, c, eps):
    if kind == "layer":
        x = x - x.sum(1, ROW, True) * (1 / c)
    rstd = ((x * x).sum(1, ROW, True) * (1 / c) + eps).rsqrt()
    return x * rstd, rstd


def _through(d, xh, rstd, kind, c):
    t = d - xh * ((d * xh).sum(1, ROW, True) * (1 / c))
    return (t - d.sum(1, ROW, True) * (1 / c) if kind == "layer" else t) * rstd


def _oracle(t, d, cu, dtype, op, post, norm, rs=1.0, eps=1e-6):
    """name -> (value, bound).  Rows outside the samples are zero."""
    v = {k: V(x.double()) for k, x in t.items()}
    n, c = t["x"].shape
    lens = [b - a for a, b in zip(cu, cu[1:])]
    sample = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    rows = slice(cu[0], cu[-1])
    one, zero = V(torch.ones(1, dtype=torch.float64)), V(torch.zeros(1, dtype=torch.float64))

    def by_row(name, none):
        return v[name].rows(sample) if name in v else none

    def of_sample(x):
        parts = [V(x.val[a - cu[0]:b - cu[0]], x.err[a - cu[0]:b - cu[0]]).sum(0, COL) for a, b in zip(cu, cu[1:])]
        return V(torch.stack([p.val for p in parts]), torch.stack([p.err for p in parts]))

    def full(x):
        out = V(torch.zeros((n, c), dtype=torch.float64))
        out.val[rows], out.err[rows] = x.val, x.err
        return out

    x, o = v["x"].rows(rows), {}
    if op != "mn":
        gate, pw, pb = by_row("gate", one), v.get("pw", one), v.get("pb", zero)
        yh, ys = _norm(v["y"].rows(rows), post, c, eps) if post else (v["y"].rows(rows), None)
        z = yh * pw + pb
        x = x * rs + gate * z
        o["r"] = full(x)
    if op != "gr":
        f, w, b = by_row("scale", zero) + 1.0, v.get("w", one), v.get("b", zero)
        xh, xs = _norm(x, norm, c, eps)
        u = xh * w + b
        o["h"] = full(u * f + by_row("shift", zero))
    if d is None:
        return {k: x.rounded(dtype) for k, x in o.items()}
    dx = None if op == "mn" else V(d["dr"][rows].double())
    if op != "gr":
        dh = V(d["dh"][rows].double())
        P, Q = of_sample(dh * xh), of_sample(dh)
        fs = v["scale"] + 1.0 if "scale" in v else V(torch.ones((len(lens), 1), dtype=torch.float64))
        o["dscale"], o["dshift"] = P * w + Q * b, Q
        o["dw"], o["db"] = (P * fs).sum(0, 1), (Q * fs).sum(0, 1)
        di = _through(dh * f * w, xh, xs, norm, c)
        dx = di if dx is None else dx + di
    if op != "mn":
        P, Q = of_sample(dx * yh), of_sample(dx)
        gs = v["gate"] if "gate" in v else V(torch.ones((len(lens), 1), dtype=torch.float64))
        o["dgate"] = P * pw + Q * pb
        o["dpw"], o["dpb"] = (P * gs).sum(0, 1), (Q * gs).sum(0, 1)
        dy = dx * gate * pw
        o["dy"] = full(_through(dy, yh, ys, post, c) if post else dy)
        dx = dx * rs
    o["dx"] = full(dx)
    return {k: x.rounded(dtype) for k, x in o.items()}


def _call(pkg, op, t, cu, post, norm, rs=1.0, eps=1e-6, **kw):
    pre = {"norm": norm, "weight": t.get("w"), "bias": t.get("b"), "scale": t.get("scale"), "shift": t.get("shift")}
    aft = {"gate": t.get("gate"), "residual_scale": rs, "post_norm": post, "post_weight": t.get("pw"),
           "post_bias": t.get("pb")}
    if op == "mn":
        return {"h": pkg.modulated_norm(t["x"], cu, eps=eps, **pre, **kw)}
    if op == "gr":
        return {"r": pkg.gated_residual(t["x"], t["y"], cu, eps=eps, **aft, **kw)}
    r, h = pkg.gated_residual_norm(t["x"], t["y"], cu, eps=eps, **pre, **aft)
    return {"r": r, "h": h}


_USED = {"mn": ("x", "w", "b", "scale", "shift"), "gr": ("x", "y", "pw", "pb", "gate"), "grn": NAMES}


def _run(pkg, dev, op, t, d, cu, post, norm, **kw):
    t = {k: x.to(dev).detach().requires_grad_() for k, x in t.items() if k in _USED[op]}
    o = _call(pkg, op, t, cu, post, norm, **kw)
    grads = torch.autograd.grad(list(o.values()), list(t.values()), [d["d" + k].to(dev) for k in o])
    return {**{k: x.detach() for k, x in o.items()}, **{"d" + k: x for k, x in zip(t, grads)}}


def _both(pkg, dev, op, lens, c, dtype, post, norm, affine=True, mod=True, rs=1.0, seed=0):
    t, d = _make(lens, c, dtype, seed + c, post, affine, mod)
    cu = _cu(lens)
    print(f"  {op} {dtype} C={c} {lens} {post} {norm} affine={affine} mod={mod}", flush=True)
    want = _oracle(t, d, cu, dtype, op, post, norm, rs)
    got = _run(pkg, dev, op, t, d, cu, post, norm, rs=rs)
    plain = _call(pkg, op, {k: x.to(dev) for k, x in t.items()}, cu, post, norm, rs=rs)
    torch.cuda.synchronize()
    for k in plain:
        assert torch.equal(plain[k], got[k])
    for k in got:
        check(got[k], want[k], k)


WIDTHS = [1, 2, 7, 8, 33, 64, 72, 100, 128, 200, 320, 512, 520, 1000, 1024, 1025, 1032, 1536, 2048, 4100, 8192]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("op", ["mn", "gr", "grn"])
def test_widths(pkg, dev, dtype, op, c):
    """Each way a row is laid over lanes: parts of a wave, a wave, a block; vectors and single values.
    A layer norm of one value has zero variance: rms there."""
    kind = "layer" if c > 2 else "rms"
    _both(pkg, dev, op, [5, 0, 1, 30], c, dtype, kind, kind, rs=0.75)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("post,norm", [(None, "layer"), ("rms", "layer"), ("layer", "rms"), (None, "rms"), ("rms", "rms")])
@pytest.mark.parametrize("affine,mod", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("op", ["mn", "gr", "grn"])
def test_kinds_and_missing_parameters(pkg, dev, dtype, op, post, norm, affine, mod):
    _both(pkg, dev, op, [70, 3], 96, dtype, post, norm, affine, mod, rs=-0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [0, 0, 1], [5000], [1, 0, 2, 0, 3, 4000, 0], [1] * 15 + [900], [1] * 16 + [900],
                                  [3] * 700, [0] * 300 + [7] + [0] * 100])
@pytest.mark.parametrize("op", ["mn", "grn"])
def test_samples(pkg, dev, dtype, op, lens):
    """No rows, one, many samples in a block's rows, more than one block's search and sums take at once."""
    _both(pkg, dev, op, lens, 64, dtype, "rms", "layer")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("op", ["mn", "gr", "grn"])
@pytest.mark.parametrize("c", [64, 1536])
def test_rows_outside_every_sample(pkg, dev, dtype, op, c):
    """They are zero in new results and gradients, whatever they hold, and left alone in a given output."""
    t, d = _make([20, 31], c, dtype, 3, n=60)
    cu = [4, 24, 55]
    for k in ("x", "y"):
        t[k][:4], t[k][55:] = float("nan"), float("inf")
    for k in d:
        d[k][:4], d[k][55:] = float("inf"), float("nan")
    want = _oracle(t, d, cu, dtype, op, "layer", "rms")
    got = _run(pkg, dev, op, t, d, torch.tensor(cu, device=dev), "layer", "rms")
    for k in got:
        check(got[k], want[k], k)
    if op != "grn":
        out = torch.full((60, c), 7.0, dtype=dtype, device=dev)
        o = _call(pkg, op, {k: x.to(dev) for k, x in t.items()}, cu, "layer", "rms", out=out)
        (k, v), = o.items()
        assert v is out and torch.equal(out[4:55], got[k][4:55])
        assert bool((out[:4] == 7).all()) and bool((out[55:] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place_and_unaligned(pkg, dev, dtype):
    """out may be x or y; buffers that are aligned to their elements only."""
    t, d = _make([40, 23], 128, dtype, 4)
    cu = _cu([40, 23])
    t = {k: x.to(dev) for k, x in t.items()}
    want_h, want_r = _call(pkg, "mn", t, cu, None, "rms")["h"], _call(pkg, "gr", t, cu, "layer", None)["r"]
    for name, op, want in (("x", "mn", want_h), ("x", "gr", want_r), ("y", "gr", want_r)):
        s = {**t, name: t[name].clone()}
        _call(pkg, op, s, cu, "layer" if op == "gr" else None, "rms" if op == "mn" else None, out=s[name])
        assert torch.equal(s[name], want)
    off = {}
    for k, x in t.items():
        if x.is_contiguous():
            off[k] = torch.empty(x.numel() + 1, dtype=dtype, device=dev)[1:].view(x.shape).copy_(x)
        else:
            off[k] = torch.empty((2, 6 * 128 + 1), dtype=dtype, device=dev)[:, 1:129].copy_(x)
    ref = _oracle({k: x.cpu() for k, x in t.items()}, d, cu, dtype, "grn", "layer", "rms")
    got = _run(pkg, dev, "grn", off, d, cu, "layer", "rms")
    for k in got:
        check(got[k], ref[k], k)


@pytest.mark.parametrize("op,missing", [("grn", "r"), ("grn", "h")])
def test_one_output_without_a_gradient(pkg, dev, op, missing):
    t, d = _make([50, 9], 64, torch.float32, 5)
    cu = _cu([50, 9])
    d["d" + missing] = torch.zeros_like(d["dr"])
    want = _oracle(t, d, cu, torch.float32, op, "rms", "layer")
    t = {k: x.to(dev).detach().requires_grad_() for k, x in t.items()}
    o = _call(pkg, op, t, cu, "rms", "layer")
    kept = "h" if missing == "r" else "r"
    grads = torch.autograd.grad(o[kept], list(t.values()), d["d" + kept].to(dev), allow_unused=True)
    for k, g in zip(t, grads):
        check(torch.zeros_like(t[k]) if g is None else g, want["d" + k], "d" + k)


def test_gradient_against_differences(pkg, dev):
    """Central differences of the definition in 64 bits (step 1e-4, their own error of order 1e-7) along
    random directions."""
    t, d = _make([9, 14], 24, torch.float32, 6)
    cu = _cu([9, 14])
    want = _oracle(t, d, cu, torch.float32, "grn", "rms", "layer", 0.5)
    got = _run(pkg, dev, "grn", t, d, cu, "rms", "layer", rs=0.5)
    g = torch.Generator().manual_seed(1)
    for k in t:
        w = torch.randn(t[k].shape, generator=g, dtype=torch.float64)
        f = []
        for sign in (1, -1):
            o = _oracle({**t, k: t[k].double() + sign * 1e-4 * w}, None, cu, torch.float32, "grn", "rms", "layer", 0.5)
            f.append(sum((o[m][0] * d["d" + m].double()).sum().item() for m in ("r", "h")))
        diff, dot = (f[0] - f[1]) / 2e-4, (got["d" + k].cpu().double() * w).sum().item()
        tol = (want["d" + k][1] * w.abs()).sum().item() + 1e-6 * (abs(diff) + 1)
        print(f"  d{k}: {dot:.6f} {diff:.6f}, off by {abs(dot - diff) / tol:.3f} of the tolerance", flush=True)
        assert abs(dot - diff) <= tol


@pytest.mark.parametrize("dtype", TYPES)
def test_small_spread_beside_a_large_mean(pkg, dev, dtype):
    """Rows whose mean is hundreds of times their spread: sums of squares of raw values would lose it."""
    t, d = _make([33], 320, dtype, 7)
    t["x"] = (100 + 0.5 * torch.randn((33, 320), generator=torch.Generator().manual_seed(8))).to(dtype)
    cu = [0, 33]
    want = _oracle(t, d, cu, dtype, "mn", None, "layer")
    got = _run(pkg, dev, "mn", t, d, cu, None, "layer")
    for k in got:
        check(got[k], want[k], k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_non_finite_rows_stay_rows(pkg, dev, dtype):
    """A row of infinities or NaN makes neither another row nor another sample's sums so."""
    t, d = _make([30, 30], 64, dtype, 9)
    cu = _cu([30, 30])
    t["x"][31], t["y"][40, 3] = float("inf"), float("nan")
    got = _run(pkg, dev, "grn", t, d, cu, "layer", "layer")
    ok = [i for i in range(60) if i not in (31, 40)]
    for k in ("r", "h", "dx", "dy"):
        assert got[k][ok].isfinite().all(), k
    for k in ("dgate", "dscale", "dshift"):
        assert got[k][0].isfinite().all(), k


def test_device_offsets_are_not_read(pkg, dev):
    t, d = _make([40, 21], 64, torch.bfloat16, 10)
    t = {k: x.to(dev) for k, x in t.items()}
    cu = torch.tensor([0, 40, 61], dtype=torch.int32, device=dev)
    want = _call(pkg, "grn", t, [0, 40, 61], "rms", "layer")
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = _call(pkg, "grn", t, cu, "rms", "layer")
    finally:
        torch.cuda.set_sync_debug_mode(0)
    for k in got:
        assert torch.equal(got[k], want[k])
    for bad in ([-5, 40, 900], [61, 30, 0], [40, 40, 7]):  # values out of range or falling: no access outside
        _call(pkg, "grn", t, torch.tensor(bad, device=dev), "rms", "layer")
    clamped = _call(pkg, "mn", t, torch.tensor([-5, 40, 900], device=dev), None, "layer")
    assert torch.equal(clamped["h"], _call(pkg, "mn", t, cu, None, "layer")["h"])
    torch.cuda.synchronize()


@pytest.mark.parametrize("c", [64, 1536])
def test_captured_step_and_streams(pkg, dev, c):
    """A training step captured into a graph and replayed between eager work on other inputs, and calls on
    another stream: the same bits as eager ones on the current stream."""
    dtype, lens = torch.bfloat16, [300, 211]
    cu = torch.tensor(_cu(lens), dtype=torch.int32, device=dev)
    runs = []
    for seed in (11, 12):
        t, d = _make(lens, c, dtype, seed)
        runs.append(({k: x.to(dev) for k, x in t.items()}, {k: x.to(dev) for k, x in d.items()}))
    want = [_run(pkg, dev, "grn", t, d, cu, "rms", "layer") for t, d in runs]
    t = {k: x.clone().requires_grad_() for k, x in runs[0][0].items()}
    d = {k: x.clone() for k, x in runs[0][1].items()}

    def step():
        o = _call(pkg, "grn", t, cu, "rms", "layer")
        return {**o, **{"d" + k: g for k, g in zip(t, torch.autograd.grad(list(o.values()), list(t.values()), [d["dr"], d["dh"]]))}}

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in want[0]:
        assert torch.equal(got[k], want[0][k]), k
    del got
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for i in (1, 0, 1):
        with torch.no_grad():
            for k in t:
                t[k].copy_(runs[i][0][k])
            for k in d:
                d[k].copy_(runs[i][1][k])
        graph.replay()
        _run(pkg, dev, "grn", *runs[1 - i], cu, "rms", "layer")
        torch.cuda.synchronize()
        for k in want[i]:
            assert torch.equal(out[k].detach(), want[i][k]), (i, k)


def test_autograd_refusals(pkg, dev):
    t, _ = _make([8], 32, torch.float32, 13)
    x = t["x"].to(dev).requires_grad_()
    with pytest.raises(pkg.TscError, match="where gradients are wanted"):
        pkg.modulated_norm(x, out=torch.empty_like(x))
    out = torch.empty((8, 32), device=dev)
    y = out * 1
    leaf = out.clone().requires_grad_()
    z = (leaf * y).sum()
    pkg.modulated_norm(x.detach(), out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(pkg.TscError, match="forward-mode"):
            pkg.gated_residual(dual, dual)
    o = pkg.modulated_norm(x, norm="rms")
    g, = torch.autograd.grad(o.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="does not require grad"):
        g.sum().backward()


def test_wide_rows_and_c_refusals(pkg, dev):
    x = torch.zeros((2, 8200), device=dev)
    with pytest.raises(pkg.TscError, match="exceeds 8192"):
        pkg.modulated_norm(x)
    x = torch.zeros((4, 32), device=dev)
    buf = torch.zeros(300, device=dev)
    with pytest.raises(pkg.TscError, match="overlaps x or y"):
        pkg.modulated_norm(buf[:128].view(4, 32), out=buf[4:132].view(4, 32))
    assert not pkg.modulated_norm(x, [0]).any()  # no samples: zeros
    assert pkg.modulated_norm(x[:0], [0, 0]).shape == (0, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [100, 1536])
def test_one_tensor_in_several_places(pkg, dev, dtype, c):
    """x as y, and one modulation as gate, scale and shift: outputs as of copies, gradients summed over the places."""
    t, d = _make([70, 30], c, dtype, 53, None)
    t = {k: x.to(dev) for k, x in t.items()}
    t["y"] = t["x"].clone()
    t["scale"] = t["shift"] = t["gate"]
    d = [x.to(dev) for x in d.values()]

    def run(x, y, gate, scale, shift):
        o = pkg.gated_residual_norm(x, y, [0, 70, 100], gate, weight=t["w"], bias=t["b"], scale=scale, shift=shift)
        return o, torch.autograd.grad(o, list({id(a): a for a in (x, y, gate, scale, shift)}.values()), d)

    names = ("x", "y", "gate", "scale", "shift")
    apart, parts = run(*(t[k].clone().requires_grad_() for k in names))
    x, m = t["x"].clone().requires_grad_(), t["gate"].clone().requires_grad_()
    once, (dx, dm) = run(x, x, m, m, m)
    assert torch.equal(once[0], apart[0]) and torch.equal(once[1], apart[1])
    for got, of in ((dx, parts[:2]), (dm, parts[2:])):
        size = sum(p.double().abs() for p in of)
        # an addition in the type less than there are places, of half a step of at most the sum of the sizes each
        eps = torch.finfo(dtype).eps
        bound = (len(of) - 1) * eps / 2 * size * (1 + eps) + (2.0 ** -24 if dtype == torch.float16 else 0.0)
        assert ((got.double() - sum(p.double() for p in of)).abs() <= bound).all()


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 8192), (torch.float16, 1000)])
def test_more_than_two_to_the_31_values(pkg, dev, dtype, c):
    """The last rows of a matrix of more than 2^31 values have what they have by themselves."""
    n = 2 ** 31 // c + 5000
    g = torch.Generator(device=dev).manual_seed(59)
    x, y, dr, dh = (torch.randn((n, c), generator=g, device=dev, dtype=dtype) for _ in range(4))
    m = (0.3 * torch.randn((2, 3, c), generator=g, device=dev)).to(dtype)
    print(f"  {n} x {c} {dtype}", flush=True)

    def run(rows, cu, mod):
        leaves = [t[rows].detach().requires_grad_() for t in (x, y)]
        r, h = pkg.gated_residual_norm(*leaves, cu, mod[:, 0], 0.5, "rms", scale=mod[:, 1], shift=mod[:, 2])
        return (r.detach(), h.detach(), *torch.autograd.grad([r, h], leaves, [dr[rows], dh[rows]]))

    all_rows = run(slice(None), [0, 3000, n], m)
    last = run(slice(n - 900, n), [0, 900], m[1:])
    for a, b in zip(all_rows, last):
        assert torch.equal(a[-900:], b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("samples", [2, 20])
@pytest.mark.parametrize("post,norm", [(1, 2), (2, 1)])
def test_c_gradients_of_parameters_that_are_not_given(pkg, dev, dtype, samples, post, norm):
    """The C call's NULL for a weight, bias, gate, scale or shift means ones or zeros, and its gradient may be wanted all
    the same: the bits that explicit ones and zeros have."""
    n, c = 40 * samples, 72
    g = torch.Generator().manual_seed(79)
    x, y, dr, dh = (torch.randn((n, c), generator=g).to(dtype).to(dev) for _ in range(4))
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    lib, handle = pkg.ops._lib.stream_handle(0)

    def run(pw, pb, gate, w, b, scale, shift):
        p = [None if t is None else t.data_ptr() for t in (pw, pb, gate, w, b, scale, shift)]
        args = (handle, code, x.data_ptr(), y.data_ptr(), None, samples, n, c, post, p[0], p[1], p[2], c, 0.5, norm, p[3],
                p[4], p[5], c, p[6], c, 1e-6, 1)
        stats = torch.empty((2, n, 2), device=dev)
        r, h, dx, dy = (torch.full_like(x, float("nan")) for _ in range(4))
        grads = {k: torch.full((c,) if k in ("dpw", "dpb", "dw", "db") else (samples, c), float("nan"), dtype=dtype, device=dev)
                 for k in ("dgate", "dpw", "dpb", "dscale", "dshift", "dw", "db")}
        assert lib.tsc_gated_norm(*args, stats.data_ptr(), r.data_ptr(), h.data_ptr()) == 0
        ws = torch.empty((lib.tsc_gated_norm_workspace_bytes(code, samples, n, c),), dtype=torch.uint8, device=dev)
        assert lib.tsc_gated_norm_backward(*args, stats.data_ptr(), dr.data_ptr(), dh.data_ptr(), ws.data_ptr(),
                                           dx.data_ptr(), dy.data_ptr(), *(t.data_ptr() for t in grads.values())) == 0
        return {"r": r, "h": h, "dx": dx, "dy": dy, **grads}

    one, zero = torch.ones(c, dtype=dtype, device=dev), torch.zeros(c, dtype=dtype, device=dev)
    ones, zeros = torch.ones((samples, c), dtype=dtype, device=dev), torch.zeros((samples, c), dtype=dtype, device=dev)
    want = run(one, zero, ones, one, zero, zeros, zeros)
    for name, got in (("none", run(None, None, None, None, None, None, None)),
                      ("weights", run(one, None, None, one, None, None, None)),
                      ("modulation", run(None, None, ones, None, None, zeros, zeros))):
        for k in want:
            assert torch.equal(got[k], want[k]), (name, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("op,c,lens", [("grn", 1536, [1500]), ("grn", 1536, [1, 0, 2, 0, 3, 2594, 0]), ("grn", 1000, [3, 0, 1, 5] * 330),
                                       ("grn", 1000, [1990, 7, 1993]), ("grn", 1025, [2, 1] * 420 + [940]), ("grn", 8192, [301, 0, 401]),
                                       ("mn", 1536, [3, 0, 1, 5, 2] * 235), ("gr", 1536, [1400, 2, 1198])])
def test_rows_of_blocks(pkg, dev, dtype, op, c, lens):
    """Rows wider than a wave's, several to each block: the rows ahead come round, three and other numbers of them, and
    the sums of a block's rows have many samples, a part of one, or both."""
    most = 256 * max(1, (8 if op == "grn" else 16) * 64 // (-(-c // 512) * 64))  # blocks at 8 values a lane
    assert sum(lens) > most
    _both(pkg, dev, op, lens, c, dtype, "layer", "rms", rs=0.75)


def test_outputs_over_parameters_are_refused(pkg, dev):
    """Blocks read them while others write their rows."""
    n, c = 40, 32
    buf = torch.zeros((n + 9, c), device=dev)
    x, out, outside = torch.ones((n, c), device=dev), buf[2:2 + n], buf[2 + n:]
    cu = [0, 20, n]
    for kw in ({"scale": out[38:]}, {"shift": buf[:3][1:]}, {"weight": out[0]}, {"bias": out[-1]}):
        with pytest.raises(pkg.TscError, match="overlaps a parameter"):
            pkg.modulated_norm(x, cu, out=out, **kw)
    for kw in ({"gate": out[5::20][:2]}, {"post_weight": out[0]}, {"post_bias": out[7]}):
        with pytest.raises(pkg.TscError, match="overlaps a parameter"):
            pkg.gated_residual(x, x, cu, post_norm="layer", out=out, **kw)
    offsets = out.view(torch.int32).flatten()[:3]
    with pytest.raises(pkg.TscError, match="overlaps a parameter"):
        pkg.modulated_norm(x, offsets, out=out)
    assert pkg.modulated_norm(x, cu, outside[:2], outside[2:4], weight=outside[4], bias=outside[5], out=out) is out
    lib, handle = pkg.ops._lib.stream_handle(0)
    for stats in (x, out, outside):
        st = lib.tsc_gated_norm(handle, 0, x.data_ptr(), None, None, 1, n, c, 0, None, None, None, 0, 1.0, 1, outside.data_ptr(),
                                None, None, 0, None, 0, 1e-6, 0, stats.data_ptr(), None, out.data_ptr())
        assert st == 1 and b"overlaps" in lib.tsc_last_error()
