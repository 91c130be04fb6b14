"""Window attention and its gradients against the definition in 64 bits on the same inputs.

Tolerances, with u = eps / 2 of the type (half a step), and 2^-25 of absolute error where an fp16 value is
below its normal range (half its smallest step):
  scores   a dot product of D terms in fp32: (D + 4) 2^-24 of the sum of its terms' sizes; a probability is
           off by e = twice that (its own and its denominator's), and 2^-20 for the exponential and the sums
  out      each P is rounded to the type once: (u + e) of sum P |v|, and one rounding: u |out|
  dP, r    fp32 dot products of D terms; r = do . out is taken from out with what its rounding left, which
           is off by the rounding of P, and by u of what was left
  dS       P (error of dP and r) + (u + e) |dS|; dq, dk: their sums against |k|, |q|, one rounding
  dv       (u + e) P^T |do|, one rounding
Sums of fp32 products: 2^-20 of the sum of the sizes (fewer than 16 roundings on a term's way through the
accumulator at equal size; rows here are at most 9000 long)."""
import math

import numpy as np
import pytest
import torch

from tests._running import check

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
ACC = 2.0 ** -20


def _cu(lens):
    return np.cumsum([0] + list(lens)).tolist()


def _make(lq, lkv, h, hk, d, dtype, seed, spread=1.2):
    g = torch.Generator().manual_seed(seed)

    def n(*s):
        return torch.randn(s, generator=g)

    t = (n(sum(lq), h, d) * spread, n(sum(lkv), hk, d) * spread, n(sum(lkv), hk, d), n(sum(lq), h, d))
    return [x.to(dtype) for x in t]


def _sees(n, m, window, sinks, causal):
    p, j = torch.arange(n)[:, None] + m - n, torch.arange(m)[None]
    s = j < sinks
    s = s | ((p - j).abs() <= window) if window is not None else s | (j >= 0)
    return s & (j <= p) if causal else s


def _oracle(q, k, v, do, cq, ck, dtype, window, sinks=0, causal=False, scale=None):
    """fp64 results and their tolerances: name -> (value, tolerance)."""
    h, d = q.shape[1:]
    hk = k.shape[1]
    z = scale or 1 / math.sqrt(d)
    f = torch.finfo(dtype)
    u = f.eps / 2
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    Q, DO = (t.double().transpose(0, 1) for t in (q, do))
    K, V = (t.double().transpose(0, 1).repeat_interleave(h // hk, 0) for t in (k, v))
    r = {n: torch.zeros_like(t) for n, t in (("out", Q), ("dq", Q), ("dk", K), ("dv", V))}
    t = {n: torch.zeros_like(x) for n, x in r.items()}
    for b in range(len(cq) - 1):
        a, c = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        if a.start == a.stop or c.start == c.stop:
            continue
        qs, ks, vs, ds = Q[:, a], K[:, c], V[:, c], DO[:, a]
        av, ad = vs.abs(), ds.abs()
        see = _sees(a.stop - a.start, c.stop - c.start, window, sinks, causal)
        s = (qs @ ks.transpose(1, 2) * z).masked_fill(~see, -math.inf)
        P = torch.softmax(s, 2).nan_to_num(0.0)
        size = (qs.abs() @ ks.abs().transpose(1, 2)).masked_fill(~see, 0.0).amax(2, keepdim=True) * z
        E = 2 * (d + 4) * 2.0 ** -24 * size + ACC
        out = P @ vs
        tO = (u + E) * (P @ av) + sub * (see.double() @ av)
        r["out"][:, a], t["out"][:, a] = out, tO + u * out.abs() + sub
        dP = ds @ vs.transpose(1, 2)
        e_dP = (d + 4) * 2.0 ** -24 * (ad @ av.transpose(1, 2))
        rr = (ds * out).sum(2, keepdim=True)
        e_r = (ad * (tO + (2 * u * u + ACC) * out.abs() + sub)).sum(2, keepdim=True)
        r["dv"][:, c] = P.transpose(1, 2) @ ds
        t["dv"][:, c] = ((u + E + ACC) * P + sub * see).transpose(1, 2) @ ad
        dS = P * (dP - rr)
        tS = P * (e_dP + e_r) + (u + E) * dS.abs() + sub * see + ACC * P * (dP.abs() + rr.abs()) + ACC * dS.abs()
        r["dq"][:, a], t["dq"][:, a] = dS @ ks * z, tS @ ks.abs() * z
        r["dk"][:, c], t["dk"][:, c] = dS.transpose(1, 2) @ qs * z, tS.transpose(1, 2) @ qs.abs() * z
    for n in ("dk", "dv"):  # shared key heads
        r[n], t[n] = (x.view(hk, h // hk, -1, d).sum(1) for x in (r[n], t[n]))
    for n in ("dq", "dk", "dv"):
        t[n] += u * r[n].abs() + sub
    return {n: (r[n].transpose(0, 1), t[n].transpose(0, 1)) for n in r}


def _run(pkg, dev, q, k, v, do, window, cq, ck, **kw):
    leaves = [t.to(dev).detach().requires_grad_() for t in (q, k, v)]
    o = pkg.sparse_window_attention(*leaves, window, cq, ck, **kw)
    grads = torch.autograd.grad(o, leaves, do.to(dev))
    return dict(zip(("out", "dq", "dk", "dv"), (o.detach(), *grads)))


def _both(pkg, dev, lq, lkv, h, hk, d, dtype, window, sinks=0, causal=False, seed=0, **kw):
    q, k, v, do = _make(lq, lkv or lq, h, hk, d, dtype, seed + d + sum(lq))
    cq = _cu(lq)
    ck = cq if lkv is None else _cu(lkv)
    print(f"  window attention {dtype} D={d} H={h}/{hk} {lq} {lkv} w={window} s={sinks} causal={causal}", flush=True)
    want = _oracle(q, k, v, do, cq, ck, dtype, window, sinks, causal)
    got = _run(pkg, dev, q, k, v, do, window, cq, ck, sinks=sinks, causal=causal, **kw)
    plain = pkg.sparse_window_attention(*(t.to(dev) for t in (q, k, v)), window, cq, ck, sinks=sinks, causal=causal, **kw)
    torch.cuda.synchronize()
    assert torch.equal(plain, got["out"])
    for n in got:
        check(got[n], want[n], n)
    return got


WINDOWS = [(0, 0), (0, 3), (5, 0), (31, 1), (32, 33), (64, 4), (200, 70), (None, 0), (None, 5), (3, 1000), (2 ** 31 - 1, 2 ** 31 - 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("causal", [False, True])
def test_windows_and_sinks(pkg, dev, dtype, d, window, sinks, causal):
    _both(pkg, dev, [0, 1, 33, 0, 300, 257], None, 4, 2, d, dtype, window, sinks, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,hk", [(1, 1), (3, 1), (5, 5), (6, 2), (8, 1), (40, 1), (16, 16), (9, 9)])
@pytest.mark.parametrize("causal", [False, True])
def test_head_layouts(pkg, dev, dtype, d, h, hk, causal):
    _both(pkg, dev, [70, 3, 129], None, h, hk, d, dtype, 20, 2, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv", [([1], [1]), ([5], [1]), ([70, 0, 300, 1, 40], [0, 129, 500, 5, 0]),
                                    ([31, 32, 33], [65, 64, 63]), ([17], [95]), ([600], [97]), ([3, 1], [900, 33])])
@pytest.mark.parametrize("window,sinks,causal", [(40, 3, False), (40, 3, True), (7, 0, True), (None, 0, True)])
def test_queries_at_the_end_of_other_keys(pkg, dev, dtype, d, lq, lkv, window, sinks, causal):
    """More keys than queries: the queries are the last rows.  Fewer: the first queries stand before the first
    key, and with causal, or far from it, they see none."""
    _both(pkg, dev, lq, lkv, 4, 2, d, dtype, window, sinks, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv,h,hk", [([1], [9000], 2, 1), ([1, 1, 1], [3000, 1, 517], 8, 1), ([7, 0, 33], [2000, 40, 5000], 4, 4),
                                         ([100], [4097], 2, 2), ([1] * 9, [800] * 8 + [4000], 16, 4)])
@pytest.mark.parametrize("window,sinks,causal", [(1000, 4, True), (4000, 70, True), (2500, 0, False), (None, 0, False)])
def test_few_queries_on_many_keys(pkg, dev, dtype, d, lq, lkv, h, hk, window, sinks, causal):
    _both(pkg, dev, lq, lkv, h, hk, d, dtype, window, sinks, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,lq,h,hk", [(128, [1500, 1300], 12, 12), (64, [2100, 900], 16, 4), (128, [4000], 8, 2),
                                       (64, [900] * 4, 16, 16), (128, [300] * 9 + [1, 2500], 5, 5)])
@pytest.mark.parametrize("window,sinks,causal", [(100, 4, False), (255, 16, True), (700, 40, False)])
def test_larger_grids(pkg, dev, dtype, d, lq, h, hk, window, sinks, causal):
    """Grids past one block per CU and sequences of many tiles; the first and the last key head."""
    q, k, v, do = _make(lq, lq, h, hk, d, dtype, h)
    cq = _cu(lq)
    print(f"  window attention larger {dtype} D={d} {lq} H={h}/{hk} w={window} {causal}", flush=True)
    got = _run(pkg, dev, q, k, v, do, window, cq, None, sinks=sinks, causal=causal)
    g = h // hk
    ks = sorted({0, hk - 1})
    qs = [x * g + i for x in ks for i in range(g)]
    want = _oracle(q[:, qs], k[:, ks], v[:, ks], do[:, qs], cq, cq, dtype, window, sinks, causal)
    for n in got:
        check(got[n][:, qs if n in ("out", "dq") else ks], want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,n", [(64, 100), (65, 100), (64, 200), (43, 300), (64, 300), (193, 100), (85, 300),
                                 (64, 500), (257, 100), (64, 600), (107, 300), (577, 70)])
def test_grids_on_both_sides_of_each_rule(pkg, dev, dtype, d, h, n):
    """Blocks of 32 or of 128 rows, in one or more rounds over the CUs, in each of the three passes."""
    q, k, v, do = _make([n], [n], h, h, d, dtype, h + n)
    print(f"  window attention grid {dtype} D={d} H={h} n={n}", flush=True)
    got = _run(pkg, dev, q, k, v, do, 60, [0, n], None, sinks=3)
    hs = [0, h - 1]
    want = _oracle(*(t[:, hs] for t in (q, k, v, do)), [0, n], [0, n], dtype, 60, 3)
    for name in got:
        check(got[name][:, hs], want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_no_window_is_sparse_attention(pkg, dev, dtype, d):
    """Without a bound it is the framework's attention over whole sequences, each within its rounding."""
    lens = [300, 1, 77]
    q, k, v, do = _make(lens, lens, 3, 3, d, dtype, 2)
    want = _oracle(q, k, v, do, _cu(lens), _cu(lens), dtype, None)["out"]
    a = [t.to(dev) for t in (q, k, v)]
    got, full = pkg.sparse_window_attention(*a, None, _cu(lens)), pkg.sparse_attention(*a, _cu(lens))
    check(got, want, "window")
    check(got, (full.double().cpu(), 2 * want[1]), "against sparse_attention")


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_of_a_fused_projection(pkg, dev, dtype):
    lens, h, d = [150, 77], 3, 64
    q, k, v, do = _make(lens, lens, h, h, d, dtype, 5)
    cq = _cu(lens)
    want = _run(pkg, dev, q, k, v, do, 30, cq, None, sinks=2)
    qkv = torch.stack([q, k, v], 1).to(dev).requires_grad_()
    o = pkg.sparse_window_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], 30, cq, sinks=2)
    g, = torch.autograd.grad(o, qkv, do.to(dev))
    assert torch.equal(o, want["out"])
    for i, n in enumerate(("dq", "dk", "dv")):
        assert torch.equal(g[:, i], want[n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hk", [1, 2])
def test_rows_outside_every_sequence(pkg, dev, dtype, d, hk):
    """Whatever stands in rows outside the sequences stays out; those rows are zero in new results and left
    alone in a given one."""
    h = 2
    q, k, v, do = _make([100], [90], h, hk, d, dtype, 6)
    cq, ck = [5, 5, 40, 83], [3, 8, 60, 71]
    for t, lo, hi in ((q, 5, 83), (k, 3, 71), (v, 3, 71), (do, 5, 83)):
        t[:lo] = float("nan")
        t[hi:] = float("inf")
    clean = [torch.nan_to_num(t, nan=0, posinf=0) for t in (q, k, v, do)]
    want = _oracle(*clean, cq, ck, dtype, 10, 2)
    got = _run(pkg, dev, q, k, v, do, 10, torch.tensor(cq, device=dev), torch.tensor(ck, device=dev), sinks=2)
    for n in got:
        check(got[n], want[n], n)
    for n, lo, hi in (("out", 5, 83), ("dq", 5, 83), ("dk", 3, 71), ("dv", 3, 71)):
        assert not got[n][:lo].any() and not got[n][hi:].any()
    out = torch.full((100, h, d), 7.0, dtype=dtype, device=dev)
    args = [t.to(dev) for t in (q, k, v)]
    plain = pkg.sparse_window_attention(*args, 10, cq, ck, sinks=2)
    assert pkg.sparse_window_attention(*args, 10, cq, ck, sinks=2, out=out) is out
    assert torch.equal(out[5:83], plain[5:83])
    assert bool((out[:5] == 7).all()) and bool((out[83:] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,h,hk", [([200], 2, 2), ([700, 900], 16, 4)])
@pytest.mark.parametrize("causal", [False, True])
def test_infinities_and_nan_stay_with_who_sees_them(pkg, dev, dtype, d, lens, h, hk, causal):
    """NaN or infinity in a key's k or v, or in a query's q or do: outputs and gradients of the rows it takes
    no part in have the bits they have without it; the others are not finite."""
    window, sinks, n = 40, 2, lens[0]
    base = _make(lens, lens, h, hk, d, dtype, 7)
    cq = _cu(lens)
    kw = dict(sinks=sinks, causal=causal)
    want = _run(pkg, dev, *base, window, cq, None, **kw)
    see = torch.zeros((sum(lens), sum(lens)), dtype=torch.bool)
    for a, b in zip(cq, cq[1:]):
        see[a:b, a:b] = _sees(b - a, b - a, window, sinks, causal)
    for what, row, value in ((2, 100, math.inf), (2, 131, math.nan), (1, 97, math.nan), (0, 64, math.nan), (3, 150, math.inf),
                             (3, 33, math.nan), (0, 111, math.inf)):
        t = [x.clone() for x in base]
        t[what][row, :, 3] = value
        got = {n: x.cpu() for n, x in _run(pkg, dev, *t, window, cq, None, **kw).items()}
        # queries whose rows it touches directly, and keys; then through them the other side's gradients
        if what in (1, 2):
            queries = see[:, row]
            keys = see[queries].any(0)
        else:
            queries = torch.zeros(sum(lens), dtype=torch.bool)
            queries[row] = True
            keys = see[row]
        for name in got:
            hit = queries if name in ("out", "dq") else keys
            same = torch.equal(got[name][~hit], want[name].cpu()[~hit])
            print(f"    {'qkvd'[what]}[{row}] = {value}: {name} of {int((~hit).sum())} other rows "
                  f"{'the same' if same else 'CHANGED'}", flush=True)
            assert same
        if what == 2:
            assert not got["out"][queries][..., 3].isfinite().any()
        if what == 3:
            assert not got["dv"][row].isfinite()[..., 3].any() and torch.equal(got["out"], want["out"].cpu())


@pytest.mark.parametrize("dtype", TYPES)
def test_many_sinks_and_blocks(pkg, dev, dtype):
    """Sinks that fill several blocks of keys, all of whose gradients come from every query."""
    _both(pkg, dev, [1500, 40], None, 4, 2, 64, dtype, 16, 300, False)
    _both(pkg, dev, [1500, 40], None, 4, 2, 64, dtype, 16, 300, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
def test_moving_maxima(pkg, dev, dtype, d):
    """Scores that climb along the keys, with one late key far above the rest."""
    n, h = 700, 2
    q, k, v, do = _make([n], [n], h, h, d, dtype, d, spread=0.3)
    q[..., 0] = 1.0
    k[..., 0] = (0.25 * torch.arange(n, dtype=torch.float32)[:, None]).to(dtype)
    k[650, :, 1] = 90.0
    for window in (None, 150):
        want = _oracle(q, k, v, do, [0, n], [0, n], dtype, window, 3)
        got = _run(pkg, dev, q, k, v, do, window, [0, n], None, sinks=3)
        for name in got:
            check(got[name], want[name], name)


def test_gradient_against_differences(pkg, dev):
    """Central differences of the definition in 64 bits (step 1e-4; their own error is of order 1e-8)
    along random directions."""
    lq, lkv, h, hk, d, dtype = [9, 20], [31, 7], 4, 2, 64, torch.float32
    t = _make(lq, lkv, h, hk, d, dtype, 1)
    do, cq, ck = t[3], _cu(lq), _cu(lkv)
    opt = (5, 2, False)
    want = _oracle(*t, cq, ck, dtype, *opt)
    got = _run(pkg, dev, *t, 5, cq, ck, sinks=2)
    g = torch.Generator().manual_seed(2)
    for i, name in enumerate(("dq", "dk", "dv")):
        w = torch.randn(t[i].shape, generator=g, dtype=torch.float64)
        f = []
        for sign in (1, -1):
            m = [x.double() for x in t[:3]]
            m[i] = m[i] + sign * 1e-4 * w
            f.append((_oracle(*m, do, cq, ck, dtype, *opt)["out"][0] * do.double()).sum().item())
        diff = (f[0] - f[1]) / 2e-4
        tol = (want[name][1] * w.abs()).sum().item() + 1e-6 * abs(diff)
        dot = (got[name].cpu().double() * w).sum().item()
        print(f"  {name}: {dot:.6f} {diff:.6f}, off by {abs(dot - diff) / tol:.3f} of the tolerance", flush=True)
        assert abs(dot - diff) <= tol


def test_hints_and_offsets(pkg, dev):
    """Too small lengths still cover every row; device offsets give the host offsets' bits and are not
    read back; values out of range or falling read nothing outside."""
    lens, h, d, dtype = [700, 3, 260], 3, 128, torch.bfloat16
    q, k, v, do = _make(lens, lens, h, h, d, dtype, 9)
    cq = _cu(lens)
    want = _run(pkg, dev, q, k, v, do, 50, cq, None, sinks=4)
    cd = torch.tensor(cq, dtype=torch.int32, device=dev)
    small = _run(pkg, dev, q, k, v, do, 50, cd, cd, sinks=4, max_seqlen_q=1, max_seqlen_kv=1)
    ref = _oracle(q, k, v, do, cq, cq, dtype, 50, 4)
    for n in want:
        check(small[n], ref[n], n)
    args = [t.to(dev) for t in (q, k, v)]
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = pkg.sparse_window_attention(*args, 50, cd, sinks=4)
    finally:
        torch.cuda.set_sync_debug_mode(0)
    check(got, ref["out"], "out")
    for bad in ([-9, 700, 703, 5000], [963, 500, 200, 0], [100, 100, 7, 900]):
        _run(pkg, dev, q, k, v, do, 50, torch.tensor(bad, device=dev), cd, sinks=4)
    torch.cuda.synchronize()


@pytest.mark.parametrize("d", [64, 128])
def test_captured_step_and_streams(pkg, dev, d):
    """A training step captured into a graph and replayed between eager work on other inputs, and calls on
    another stream: the same bits as eager ones on the current stream."""
    lens, h, hk, dtype = [300, 211], 4, 2, torch.bfloat16
    cu = torch.tensor(_cu(lens), dtype=torch.int32, device=dev)
    runs = [[x.to(dev) for x in _make(lens, lens, h, hk, d, dtype, s)] for s in (11, 12)]
    want = [_run(pkg, dev, *r, 40, cu, cu, sinks=3) for r in runs]
    leaves = [x.detach().clone().requires_grad_() for x in runs[0][:3]]
    do = runs[0][3].clone()

    def step():
        o = pkg.sparse_window_attention(*leaves, 40, cu, cu, sinks=3)
        return dict(zip(("out", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do))))

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for n in got:
        assert torch.equal(got[n], want[0][n]), n
    del got
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for i in (1, 0, 1):
        with torch.no_grad():
            for x, y in zip((*leaves, do), runs[i]):
                x.copy_(y)
        graph.replay()
        _run(pkg, dev, *runs[1 - i], 40, cu, cu, sinks=3)
        torch.cuda.synchronize()
        for n in want[i]:
            assert torch.equal(out[n].detach(), want[i][n]), (i, n)


def test_token_by_token(pkg, dev):
    """A prompt in one call, and its last rows as single tokens on the longer cache (captured with the keys'
    offsets on the device, replayed as the cache grows): the same rows within their tolerances."""
    n, h, hk, d, dtype, window, sinks = 400, 8, 2, 64, torch.bfloat16, 100, 4
    q, k, v, do = _make([n], [n], h, hk, d, dtype, 13)
    want = _oracle(q, k, v, do, [0, n], [0, n], dtype, window, sinks, True)["out"]
    q, k, v = (t.to(dev) for t in (q, k, v))
    check(pkg.sparse_window_attention(q, k, v, window, [0, n], sinks=sinks, causal=True), want, "prompt")
    token = q[:1].clone()
    cq, ck = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 1], [0, 1]))
    side = torch.cuda.Stream(dev)

    def call():
        return pkg.sparse_window_attention(token, k, v, window, cq, ck, sinks=sinks, causal=True, max_seqlen_q=1,
                                           max_seqlen_kv=n)

    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call()
    got = torch.empty_like(q)
    for i in range(n):
        token.copy_(q[i:i + 1])
        ck.copy_(torch.tensor([0, i + 1], dtype=torch.int32))
        graph.replay()
        got[i:i + 1].copy_(out)
    check(got, want, "token by token")


def test_autograd_refusals(pkg, dev):
    q = torch.randn((8, 2, 64), device=dev).requires_grad_()
    f = pkg.sparse_window_attention
    with pytest.raises(pkg.TscError, match="where gradients are wanted"):
        f(q, q, q, 4, [0, 8], out=torch.empty_like(q))
    o = f(q, q, q, 4, [0, 8])
    with torch.no_grad():
        o.mul_(2)  # the gradient needs the output
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q.detach(), torch.ones_like(q))
        with pytest.raises(pkg.TscError, match="forward-mode"):
            f(dual, q.detach(), q.detach(), 4, [0, 8])
    with pytest.raises(pkg.TscError, match="is needed where k has"):
        f(q, q[:5], q[:5], 4, [0, 8])
    with pytest.raises(pkg.TscError, match="differ in length"):
        f(q, q, q, 4, [0, 8], [0, 4, 8])
    buf = torch.zeros(8 * 128 * 4, device=dev)
    with pytest.raises(pkg.TscError, match="overlaps"):
        x = buf[:1024].view(8, 2, 64)
        f(x, x, x, 4, [0, 8], out=buf[512:1536].view(8, 2, 64))


def test_gradient_of_a_view_and_of_one_leaf(pkg, dev):
    """An incoming gradient that is a slice of a larger one, and gradients of some inputs only."""
    q, k, v, do = _make([90], [90], 2, 1, 64, torch.bfloat16, 15)
    want = _run(pkg, dev, q, k, v, do, 20, [0, 90], None)
    a = [t.to(dev) for t in (q, k, v)]
    leaf = a[0].clone().requires_grad_()
    o = pkg.sparse_window_attention(leaf, a[1], a[2], 20, [0, 90])
    big = torch.zeros((90 * 128 + 5,), dtype=torch.bfloat16, device=dev)
    big[5:] = do.to(dev).flatten()
    g, = torch.autograd.grad(o, leaf, big[5:].view(90, 2, 64))
    assert torch.equal(g, want["dq"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv,sinks", [([2000], None, 1), ([1500, 0, 7, 40, 900], None, 37), ([900, 700], [1000, 900], 4),
                                          ([2500, 20], None, 130), ([1200, 600], [1000, 30], 33)])
@pytest.mark.parametrize("causal", [False, True])
def test_sinks_with_blocks_of_their_own(pkg, dev, dtype, d, lq, lkv, sinks, causal):
    """Long sequences, short windows: the rows of the sinks are shared out, and sequences shorter than the
    sinks, without queries, and lengths given too small still have theirs."""
    h, hk, window = 4, 2, 20
    ws = pkg.load_library().tsc_window_attention_workspace_bytes
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    most = (max(lq), max(lkv or lq))
    sizes = (code, len(lq), sum(lq), sum(lkv or lq), h, hk, d, window)
    assert ws(*sizes, sinks, int(causal), *most, 1) > ws(*sizes, 0, int(causal), *most, 1)
    _both(pkg, dev, lq, lkv, h, hk, d, dtype, window, sinks, causal)
    if lkv is None:
        _both(pkg, dev, lq, lkv, h, hk, d, dtype, window, sinks, causal, max_seqlen_q=most[0], max_seqlen_kv=3 * sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv,h,hk", [([200], None, 2, 2), ([2500], None, 16, 16), ([1, 1], [3000, 40], 2, 1)])
def test_scores_that_are_all_minus_infinity(pkg, dev, dtype, d, lq, lkv, h, hk):
    """A softmax of nothing but -inf is NaN, in whichever blocks and parts the row is; of no keys at all it is
    zeros; and rows that see other keys as well have what they have without those."""
    q, k, v, do = _make(lq, lkv or lq, h, hk, d, dtype, 23)
    cq, ck = _cu(lq), _cu(lkv or lq)
    q[..., 3] = q[..., 3].abs() + 0.5
    print(f"  scores of -inf {dtype} D={d} {lq} {lkv}", flush=True)
    if lkv is None:
        k[100, :, 3] = -math.inf
        got = {n: x.cpu() for n, x in _run(pkg, dev, q, k, v, do, 0, cq, ck, causal=True).items()}
        others = torch.arange(sum(lq)) != 100
        for n in got:  # query 100 sees key 100 alone, and nobody else does
            assert got[n][100].isnan().all() and got[n][others].isfinite().all(), n
        got = _run(pkg, dev, q, k, v, do, 5, cq, ck, causal=True)
        assert got["out"].isfinite().all() and got["dv"].isfinite().all()
        assert not got["dv"][100].any()
    else:
        k[:, :, 3] = -math.inf
        got = pkg.sparse_window_attention(*(t.to(dev) for t in (q, k, v)), 5000, cq, ck)
        assert got.isnan().all()
        k[2500, :, 3] = 1.0  # the one key with a weight
        got = pkg.sparse_window_attention(*(t.to(dev) for t in (q, k, v)), 5000, cq, ck)
        alone = v[2500].repeat_interleave(h // hk, 0)
        # its weight p may be a rounding of the score away from 1, and p v / p is three operations; in 16 bits p is 1
        assert ((got[0].cpu().double() - alone.double()).abs() <= 4 * 2.0 ** -23 * alone.double().abs()).all()
        assert got[1].isnan().all()
    got = pkg.sparse_window_attention(q.to(dev), k[:0].to(dev), v[:0].to(dev), 5, cq, [0] * len(cq))
    assert not got.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
def test_one_tensor_as_all_inputs(pkg, dev, dtype, d):
    """q, k and v in the same memory: the gradient is the sum of the three."""
    q, _, _, do = _make([300], [300], 3, 3, d, dtype, 31)
    one = q.to(dev).requires_grad_()
    o = pkg.sparse_window_attention(one, one, one, 30, [0, 300], sinks=2)
    g, = torch.autograd.grad(o, one, do.to(dev))
    parts = _run(pkg, dev, q, q, q, do, 30, [0, 300], None, sinks=2)
    assert torch.equal(o.detach(), parts["out"])
    size = parts["dq"].double().abs() + parts["dk"].double().abs() + parts["dv"].double().abs()
    total = parts["dq"].double() + parts["dk"].double() + parts["dv"].double()
    # two additions in the type, of half a step of at most the sum of the sizes each
    assert ((g.double() - total).abs() <= 2 * torch.finfo(dtype).eps / 2 * size * (1 + torch.finfo(dtype).eps)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,n", [(106, 300), (108, 300), (319, 70), (321, 70)])
def test_grids_about_320_tiles(pkg, dev, dtype, h, n):
    """Both sides of the rule for blocks of 256 rows at 64 dimensions in 16 bits."""
    q, k, v, do = _make([n], [n], h, h, 64, dtype, h + n)
    print(f"  window attention grid {dtype} H={h} n={n}", flush=True)
    got = _run(pkg, dev, q, k, v, do, 60, [0, n], None, sinks=3)
    hs = [0, h - 1]
    want = _oracle(*(t[:, hs] for t in (q, k, v, do)), [0, n], [0, n], dtype, 60, 3)
    for name in got:
        check(got[name][:, hs], want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_wide_row_strides(pkg, dev, dtype, d):
    """Rows 2^24 values apart: offsets past 2^32 bytes and, within a tile, past 2^30; one value more is refused."""
    n, h, ld = 220, 2, 1 << 24
    q, k, v, do = _make([n], [n], h, h, d, dtype, 37)
    print(f"  wide strides {dtype} D={d}", flush=True)
    buf = torch.empty((n, ld), dtype=dtype, device=dev)
    got = []
    for t in (q, k, v):
        view = buf[:, len(got) * h * d:(len(got) + 1) * h * d]
        view.copy_(t.view(n, -1))
        got.append(view.unflatten(1, (h, d)))
    want = _run(pkg, dev, q, k, v, do, 50, [0, n], None, sinks=1)
    leaves = [t.detach().requires_grad_() for t in got]
    o = pkg.sparse_window_attention(*leaves, 50, [0, n], sinks=1)
    assert torch.equal(o.detach(), want["out"])
    for g, name in zip(torch.autograd.grad(o, leaves, do.to(dev)), ("dq", "dk", "dv")):
        assert torch.equal(g, want[name]), name
    far = torch.as_strided(buf, (2, h, d), (ld + 16, d, 1))
    with pytest.raises(pkg.TscError, match="row stride"):
        pkg.sparse_window_attention(far, far, far, 5, [0, 2])


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_more_than_two_to_the_31_values(pkg, dev, dtype, d):
    """A million and more tokens: the last ones, of a second sequence, against the definition on what they see."""
    h, n = 16, 2 ** 31 // (16 * d) + 5000
    g = torch.Generator(device=dev).manual_seed(41)
    q, k, v, do = (torch.randn((n, h, d), generator=g, device=dev, dtype=dtype) for _ in range(4))
    got = {}
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = pkg.sparse_window_attention(*leaves, 40, [0, 3000, n])
    got["out"] = o.detach()
    got["dq"], got["dk"], got["dv"] = torch.autograd.grad(o, leaves, do)
    tail, hs = 400, [0, h - 1]
    want = _oracle(*(t[-tail:, hs].detach().cpu() for t in (q, k, v, do)), [0, tail], [0, tail], dtype, 40)
    print(f"  {n} tokens {dtype} D={d}", flush=True)
    for name in got:  # the cut row sees less; rows 80 on neither see it nor are seen through it
        check(got[name][-tail + 80:, hs], tuple(x[80:] for x in want[name]), name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_infinities_and_nan_in_wide_grids(pkg, dev, dtype, d, causal):
    """The same with 320 tiles of 128 rows and of 128 keys, which the wide kernels of all three passes take, and a
    window with tiles that all rows of a block see: at a block's ends, within its run, at a window's edge."""
    window, sinks, n, h = 400, 2, 2500, 16
    base = _make([n], [n], h, h, d, dtype, 73)
    kw = dict(sinks=sinks, causal=causal)
    print(f"  infinities and NaN {dtype} D={d} n={n} causal={causal}", flush=True)
    want = {x: t.cpu() for x, t in _run(pkg, dev, *base, window, [0, n], None, **kw).items()}
    see = _sees(n, n, window, sinks, causal)
    for what, row, value in ((2, 1100, math.inf), (2, 1279, math.nan), (2, 1, -math.inf), (1, 1021, math.nan), (1, 1500, math.inf),
                             (0, 1290, math.inf), (0, 1400, math.nan), (0, 2499, -math.inf), (3, 1150, math.inf), (3, 640, math.nan)):
        t = [x.clone() for x in base]
        t[what][row, :, 3] = value
        got = {x: y.cpu() for x, y in _run(pkg, dev, *t, window, [0, n], None, **kw).items()}
        if what in (1, 2):
            queries = see[:, row]
            keys = see[queries].any(0)
        else:
            queries = torch.zeros(n, dtype=torch.bool)
            queries[row] = True
            keys = see[row]
        for name in got:
            hit = queries if name in ("out", "dq") else keys
            other = (got[name][~hit] != want[name][~hit]).flatten(1).any(1).sum().item()
            print(f"    {'qkvd'[what]}[{row}] = {value}: {name} of {int((~hit).sum())} other rows, {other} CHANGED", flush=True)
            assert torch.equal(got[name][~hit], want[name][~hit])
        if what == 2:
            assert not got["out"][queries][..., 3].isfinite().any()
        if what == 3:
            assert not got["dv"][row].isfinite()[..., 3].any() and torch.equal(got["out"], want["out"])


def test_outputs_over_offsets_and_statistics_are_refused(pkg, dev):
    n, h, d = 40, 2, 64
    x, out = torch.ones((n, h, d), device=dev), torch.zeros((n, h, d), device=dev)
    with pytest.raises(pkg.TscError, match="out overlaps an input"):
        pkg.sparse_window_attention(x, x, x, 4, out.view(torch.int32).flatten()[5:8], out=out)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    lib, handle = pkg.ops._lib.stream_handle(0)
    for lse in (x, out, cu):
        p = x.data_ptr()
        st = lib.tsc_window_attention(handle, 0, p, p, p, h * d, h * d, h * d, cu.data_ptr(), cu.data_ptr(), 1, n, n, h, h, d,
                                      0.0, 4, 0, 0, n, n, 0, None, out.data_ptr(), None, lse.data_ptr())
        assert st == 1 and b"overlap" in lib.tsc_last_error()


def test_c_scales(pkg, dev):
    """NaN, infinity and what overflows once it is multiplied with log2(e) are refused; 0 and less mean the default."""
    n, h, d = 40, 2, 64
    x = torch.randn((n, h, d), generator=torch.Generator().manual_seed(83)).to(dev)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    lib, handle = pkg.ops._lib.stream_handle(0)
    p = x.data_ptr()
    out, dq, dk, dv = (torch.full_like(x, 7.0) for _ in range(4))
    lse = torch.zeros((n, h), device=dev)
    ws = torch.empty((lib.tsc_window_attention_workspace_bytes(0, 1, n, n, h, h, d, 4, 0, 0, n, n, 1),), dtype=torch.uint8,
                     device=dev)

    def run(scale):
        a = (handle, 0, p, p, p, h * d, h * d, h * d, cu.data_ptr(), cu.data_ptr(), 1, n, n, h, h, d, scale, 4, 0, 0, n, n, 0)
        return (lib.tsc_window_attention(*a, None, out.data_ptr(), None, lse.data_ptr()),
                lib.tsc_window_attention_backward(*a, out.data_ptr(), None, lse.data_ptr(), p, ws.data_ptr(), dq.data_ptr(),
                                                  dk.data_ptr(), dv.data_ptr()))

    for scale in (float("nan"), float("inf"), 3e38):
        assert run(scale) == (1, 1) and b"scale" in lib.tsc_last_error()
    assert bool((out == 7).all())
    for scale in (0.0, -1.0, float("-inf")):
        assert run(scale) == (0, 0)
        assert torch.equal(out, pkg.sparse_window_attention(x, x, x, 4, cu))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,h,hk", [(128, 12, 12), (64, 16, 4)])
@pytest.mark.parametrize("lens", [[30] * 120 + [0] * 3 + [1] * 40 + [257], [600, 1, 1, 1, 1, 1, 1, 1], [1] * 700])
@pytest.mark.parametrize("window,sinks,causal", [(10, 3, False), (200, 40, True)])
def test_many_short_sequences(pkg, dev, dtype, d, h, hk, lens, window, sinks, causal):
    """Grids of wide blocks most of whose rows, or most of which, have nothing to do; the first and the last key head."""
    q, k, v, do = _make(lens, lens, h, hk, d, dtype, 89 + len(lens))
    cq = _cu(lens)
    print(f"  window attention short {dtype} D={d} {len(lens)} sequences H={h}/{hk} w={window} {causal}", flush=True)
    got = _run(pkg, dev, q, k, v, do, window, cq, None, sinks=sinks, causal=causal)
    g = h // hk
    ks = [0, hk - 1]
    qs = [x * g + i for x in ks for i in range(g)]
    want = _oracle(q[:, qs], k[:, ks], v[:, ks], do[:, qs], cq, cq, dtype, window, sinks, causal)
    for n in got:
        check(got[n][:, qs if n in ("out", "dq") else ks], want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_tokens_of_several_objects_on_a_cache_with_room(pkg, dev, dtype, d):
    """A cache of three sequences that grow in place: the unused rows behind each one's keys are a sequence without a
    query, and whatever they hold stays out."""
    h, hk, window, sinks, room = 8, 2, 50, 3, (400, 130, 40)
    start = _cu(room)
    _, k, v, _ = _make(room, room, h, hk, d, dtype, 97)
    cache = [torch.full(t.shape, float("nan"), dtype=dtype, device=dev) for t in (k, v)]
    cq = torch.tensor([0, 1, 1, 2, 2, 3, 3], dtype=torch.int32, device=dev)
    for step, lens in enumerate(([1, 1, 1], [64, 129, 40], [399, 130, 0], [400, 0, 33])):
        for a, n in zip(start, lens):
            for to, of in zip(cache, (k, v)):
                to[a:a + n] = of[a:a + n].to(dev)
        q = _make([3], [0], h, hk, d, dtype, 101 + step)[0]
        ck = torch.tensor([0] + [x for a, b, n in zip(start, start[1:], lens) for x in (a + n, b)], dtype=torch.int32, device=dev)
        got = pkg.sparse_window_attention(q.to(dev), *cache, window, cq, ck, sinks=sinks, causal=True, max_seqlen_q=1,
                                          max_seqlen_kv=max(lens))
        keys = [torch.cat([t[a:a + n] for a, n in zip(start, lens)]) for t in (k, v)]
        want = _oracle(q, *keys, torch.zeros_like(q), [0, 1, 2, 3], _cu(lens), dtype, window, sinks, True)["out"]
        check(got, want, f"{lens}")
        for t in cache:
            t.fill_(float("nan"))
