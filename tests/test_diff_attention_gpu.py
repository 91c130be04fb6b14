"""Differential attention and its gradients against the definition in 64 bits on the same inputs.

Tolerances, with u = eps / 2 of the type (half a step), and 2^-25 of absolute error where an fp16
value is below its normal range (half its smallest step):
  scores      a dot product of D/2 terms in fp32: (D/2 + 4) 2^-24 of the sum of its terms' sizes, in
              units of log2; a probability is off by e = twice ln 2 of that (its own and its
              denominator's), and 2^-20 for the exponential and the sums
  P v         each P is rounded to the type once: (u + e) of sum P |v|
  out         that of both maps, and one rounding: u |out|
  dP, r       fp32 dot products of D terms; r = do . (P v) is taken from sums in fp32 of the rounded P over
              the sum of the rounded P: off by sum |do| times (2 u + e) of sum P |v|
  dS          P (error of dP and r) + (u + e) |dS|; dq, dk: their sums against |k|, |q|, one rounding
  dv          (u + e) (P1 + |lambda| P2)^T |do|, one rounding.  The kernel rounds the difference of the
              maps once, or (D = 128 in 16 bits, blocks of 128 keys) P1 and P2 each and takes P2's product
              with do times lambda: relative errors are at most the same, u (P1 + |lambda| P2); below
              fp16's normal range the two are off by up to 2^-25 each, that is (1 + |lambda|) 2^-25
  dlambda     - sum P2 dP, from unrounded fp32 values: e of the sum of P2 |dP|, and dP's error
Sums of fp32 products: 2^-20 of the sum of the sizes (fewer than 16 roundings on a term's way through
the accumulator at equal size; rows here are at most 9000 long)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
ACC = 2.0 ** -20


def _cu(lens):
    return np.cumsum([0] + list(lens)).tolist()


def _make(lq, lkv, h, d, dtype, seed, spread=1.2):
    g = torch.Generator().manual_seed(seed)

    def n(*s):
        return torch.randn(s, generator=g)

    q, k, v, do = n(sum(lq), h, d) * spread, n(sum(lkv), h, d) * spread, n(sum(lkv), h, d), n(sum(lq), h, d)
    lam = 0.2 + 0.6 * torch.rand(h, generator=g)
    return [t.to(dtype) for t in (q, k, v, do)] + [lam]


def _oracle(q, k, v, do, lam, cq, ck, dtype, scale=None):
    """fp64 results and their tolerances: name -> (value, tolerance)."""
    tq, h, d = q.shape
    half = d // 2
    z = scale or 1 / math.sqrt(half)
    f = torch.finfo(dtype)
    u = f.eps / 2
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    # fp64 (H, n, D)
    Q, K, V, DO = (t.double().transpose(0, 1) for t in (q, k, v, do))
    lm = lam.double().view(h, 1, 1)
    al = lm.abs()
    r = {n: torch.zeros_like(t) for n, t in (("out", Q), ("dq", Q), ("dk", K), ("dv", V))}
    t = {n: torch.zeros_like(x) for n, x in r.items()}
    r["dlam"], t["dlam"] = torch.zeros(h, dtype=torch.float64), torch.zeros(h, dtype=torch.float64)
    for b in range(len(cq) - 1):
        a, c = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        if a.start == a.stop or c.start == c.stop:
            continue
        qs, ks, vs, ds = Q[:, a], K[:, c], V[:, c], DO[:, a]
        av, ad = vs.abs(), ds.abs()
        P, E, O, tO = [], [], [], []
        for m in (slice(0, half), slice(half, d)):
            P.append(torch.softmax(qs[..., m] @ ks[..., m].transpose(1, 2) * z, 2))
            size = (qs[..., m].abs() @ ks[..., m].abs().transpose(1, 2)).amax(2, keepdim=True) * z
            E.append(2 * (half + 4) * 2.0 ** -24 * size + ACC)  # log2 units times ln 2 = the score's own
            O.append(P[-1] @ vs)
            tO.append((u + E[-1]) * (P[-1] @ av) + sub * av.sum(1, keepdim=True))
        out = O[0] - lm * O[1]
        r["out"][:, a] = out
        t1 = tO[0] + al * tO[1]
        t["out"][:, a] = t1 + u * out.abs() + sub
        dP = ds @ vs.transpose(1, 2)
        e_dP = (d + 4) * 2.0 ** -24 * (ad @ av.transpose(1, 2))
        r1, r2 = (ds * O[0]).sum(2, keepdim=True), (ds * O[1]).sum(2, keepdim=True)
        e_r1, e_r2 = ((ad * (tO[i] + u * (P[i] @ av) + ACC * O[i].abs())).sum(2, keepdim=True) for i in (0, 1))
        p = P[0] - lm * P[1]
        r["dv"][:, c] = p.transpose(1, 2) @ ds
        ep = (u + E[0]) * P[0] + al * (u + E[1]) * P[1] + (1 + al) * sub
        t["dv"][:, c] = (ep + ACC * (P[0] + al * P[1])).transpose(1, 2) @ ad
        for i, (m, x, e_r, f_) in enumerate(((slice(0, half), r1, e_r1, 1.0), (slice(half, d), r2, e_r2, -lm))):
            dS = P[i] * (dP - x) * f_
            fa = 1.0 if i == 0 else al
            tS = P[i] * (e_dP + e_r) * fa + (u + E[i]) * dS.abs() + sub
            tS = tS + ACC * P[i] * (dP.abs() + x.abs()) * fa
            r["dq"][:, a, m] = dS @ ks[..., m] * z
            t["dq"][:, a, m] = (tS + ACC * dS.abs()) @ ks[..., m].abs() * z
            r["dk"][:, c, m] = dS.transpose(1, 2) @ qs[..., m] * z
            t["dk"][:, c, m] = (tS + ACC * dS.abs()).transpose(1, 2) @ qs[..., m].abs() * z
        r["dlam"] -= r2.sum((1, 2))
        t["dlam"] += (P[1] * (E[1] * dP.abs() + e_dP)).sum((1, 2))
    for n in ("dq", "dk", "dv"):
        t[n] += u * r[n].abs() + sub
    return {n: ((r[n], t[n]) if n == "dlam" else (r[n].transpose(0, 1), t[n].transpose(0, 1))) for n in r}


def _close(got, want, what, rows=None):
    val, tol = want
    if rows is not None:
        got, val, tol = got[rows], val[rows], tol[rows]
    got = got.detach().double().cpu()
    assert got.shape == val.shape
    if not got.numel():
        return
    ratio = ((got - val).abs() / (tol + 1e-30)).max().item()
    print(f"    {what}: worst error {ratio:.3f} of its tolerance", flush=True)
    assert ratio <= 1.0, (what, ratio)


def _run(pkg, dev, q, k, v, do, lam, cq, ck, **kw):
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, lam)]
    o = pkg.sparse_diff_attention(*leaves, cq, ck, **kw)
    grads = torch.autograd.grad(o, leaves, do.to(dev))
    return dict(zip(("out", "dq", "dk", "dv", "dlam"), (o.detach(), *grads)))


SHAPES = [([1], None, 1), ([0, 1, 33, 0, 200, 257], None, 3), ([5], [1], 2), ([128, 129, 127], None, 2),
          ([70, 0, 300, 1, 40], [0, 129, 500, 5, 0], 2), ([31, 32, 33], [65, 64, 63], 9),
          ([17], [95], 8), ([600], [97], 1), ([3, 1], [900, 33], 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv,h", SHAPES)
def test_forward_and_gradients(pkg, dev, dtype, d, lq, lkv, h):
    cq = _cu(lq)
    ck = cq if lkv is None else _cu(lkv)
    q, k, v, do, lam = _make(lq, lkv or lq, h, d, dtype, d + sum(lq))
    print(f"  diff attention {dtype} D={d} H={h} {lq} {lkv}", flush=True)
    want = _oracle(q, k, v, do, lam, cq, ck, dtype)
    plain = pkg.sparse_diff_attention(*(t.to(dev) for t in (q, k, v, lam)), cq, ck)
    got = _run(pkg, dev, q, k, v, do, lam, cq, ck)
    torch.cuda.synchronize()
    assert torch.equal(plain, got["out"])
    for n in got:
        _close(got[n], want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv,h", [([1], [9000], 1), ([1, 1, 1], [3000, 0, 517], 4), ([7, 0, 33], [2000, 40, 5000], 3),
                                      ([100], [4097], 2)])
def test_few_queries_on_many_keys(pkg, dev, dtype, d, lq, lkv, h):
    q, k, v, do, lam = _make(lq, lkv, h, d, dtype, 3 * d + sum(lkv))
    cq, ck = _cu(lq), _cu(lkv)
    print(f"  diff attention few queries {dtype} D={d} {lq} {lkv}", flush=True)
    want = _oracle(q, k, v, do, lam, cq, ck, dtype)
    got = _run(pkg, dev, q, k, v, do, lam, cq, ck)
    plain = pkg.sparse_diff_attention(*(t.to(dev) for t in (q, k, v, lam)), cq, ck)
    assert torch.equal(plain, got["out"])
    for n in got:
        _close(got[n], want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,h", [([1500, 1300], 12), ([2100], 6), ([4000], 1), ([900] * 4, 16)])
def test_larger_self_attention(pkg, dev, dtype, lq, h):
    """Grids past one block per CU and sequences of many tiles; two heads against the definition."""
    d = 128
    q, k, v, do, lam = _make(lq, lq, h, d, dtype, h)
    cq = _cu(lq)
    print(f"  diff attention larger {dtype} {lq} H={h}", flush=True)
    got = _run(pkg, dev, q, k, v, do, lam, cq, None)
    hs = sorted({0, h - 1})
    want = _oracle(*(t[:, hs] for t in (q, k, v, do)), lam[hs], cq, cq, dtype)
    for n in got:
        _close(got[n][hs] if n == "dlam" else got[n][:, hs], want[n], n)


def _two_heads(pkg, dev, lq, lkv, h, d, dtype, seed):
    """Forward and gradients, the first and the last head against the definition."""
    q, k, v, do, lam = _make(lq, lkv or lq, h, d, dtype, seed)
    cq = _cu(lq)
    ck = cq if lkv is None else _cu(lkv)
    got = _run(pkg, dev, q, k, v, do, lam, cq, ck)
    hs = sorted({0, h - 1})
    want = _oracle(*(t[:, hs] for t in (q, k, v, do)), lam[hs], cq, ck, dtype)
    for n in got:
        _close(got[n][hs] if n == "dlam" else got[n][:, hs], want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,n", [(64, 100), (65, 100), (64, 200), (43, 300), (64, 300), (193, 100), (85, 300),
                                 (64, 500), (257, 100), (64, 600), (107, 300), (96, 500), (77, 640), (577, 70)])
def test_grids_on_both_sides_of_each_rule(pkg, dev, dtype, d, h, n):
    """64, 65, 128, 129, 192, 193, 255, 256, 257, 320, 321, 384, 385 and 577 blocks of 128 rows: blocks of 32
    or of 128 rows, in one or more rounds over the CUs, in each of the three passes."""
    print(f"  diff attention grid {dtype} D={d} H={h} n={n}", flush=True)
    _two_heads(pkg, dev, [n], None, h, d, dtype, h + n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,h", [([1500, 1300], 12), ([4000], 16), ([300] * 9 + [1, 2500], 5)])
def test_larger_self_attention_of_64_dimensions(pkg, dev, dtype, lq, h):
    print(f"  diff attention larger {dtype} D=64 {lq} H={h}", flush=True)
    _two_heads(pkg, dev, lq, None, h, 64, dtype, h)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv,h", [([32], [5000], 2), ([33], [5000], 2), ([1] * 12, [3000] + [0, 1, 63, 64, 65] * 2 + [700], 3),
                                      ([1, 0, 2] * 7, [40, 900, 0] * 6 + [5000, 3, 1025], 1)])
def test_parts_of_the_keys_of_many_sequences(pkg, dev, dtype, d, lq, lkv, h):
    """32 and 33 queries (other blocks at 128 dimensions in 16 bits), and more sequences than are ranked by
    their keys, most of them with fewer keys than a part."""
    print(f"  diff attention parts {dtype} D={d} {lq} {lkv}", flush=True)
    ws = pkg.load_library().tsc_diff_attention_workspace_bytes
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    assert ws(code, len(lq), sum(lq), sum(lkv), h, d, max(lq), max(lkv), 0) > 0
    _two_heads(pkg, dev, lq, lkv, h, d, dtype, 23 + h)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv,h", [([64] * 13, [1500] + [41] * 12, 16), ([100] * 28, [3000] + [37] * 27, 8),
                                      ([640] + [10] * 7, None, 5)])
def test_many_uneven_sequences_on_nearly_a_block_per_cu(pkg, dev, dtype, d, lq, lkv, h):
    """193 to 255 blocks of 128 queries, most of the keys in one sequence: whole sequences in fp32,
    parts of them where a type's kernel has those.  The first and the last head against the definition."""
    q, k, v, do, lam = _make(lq, lkv or lq, h, d, dtype, 21 + h)
    cq = _cu(lq)
    ck = cq if lkv is None else _cu(lkv)
    print(f"  diff attention uneven {dtype} D={d} H={h} B={len(lq)}", flush=True)
    got = _run(pkg, dev, q, k, v, do, lam, cq, ck)
    hs = [0, h - 1]
    want = _oracle(*(t[:, hs] for t in (q, k, v, do)), lam[hs], cq, ck, dtype)
    for n in got:
        _close(got[n][hs] if n == "dlam" else got[n][:, hs], want[n], n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
def test_moving_maxima(pkg, dev, dtype, d):
    """Scores that climb along the keys in one map and fall in the other, and one late key far above
    the rest: both running maxima are raised at different steps."""
    n, h = 700, 2
    g = torch.Generator().manual_seed(d)
    q, k, v, do, lam = _make([n], [n], h, d, dtype, d, spread=0.3)
    q[..., 0], q[..., d // 2] = 1.0, 1.0
    ramp = torch.arange(n, dtype=torch.float32)[:, None]
    k[..., 0], k[..., d // 2] = (0.25 * ramp).to(dtype), (-0.25 * ramp).to(dtype)
    k[650, :, d // 2] = 90.0
    print(f"  diff attention moving maxima {dtype} D={d}", flush=True)
    want = _oracle(q, k, v, do, lam, [0, n], [0, n], dtype)
    got = _run(pkg, dev, q, k, v, do, lam, [0, n], None)
    for name in got:
        _close(got[name], want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lkv,h", [([270, 3, 1], [1, 2, 1], 2), ([5000], [1], 16)])
def test_one_key_has_no_gradient_in_its_scores(pkg, dev, dtype, d, lq, lkv, h):
    """The softmax of one score is 1 whatever the score: dq and dk are zeros, not what dP - r rounds to."""
    q, k, v, do, lam = _make(lq, lkv, h, d, dtype, 6)
    cq, ck = _cu(lq), _cu(lkv)
    got = _run(pkg, dev, q, k, v, do, lam, cq, ck)
    for a, b, c, e in zip(cq, cq[1:], ck, ck[1:]):
        one = e - c == 1
        assert bool(got["dq"][a:b].any()) != one and bool(got["dk"][c:e].any()) != one
    assert got["dv"].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_peaked_maps_keep_dq(pkg, dev, dtype, d):
    """Scores of standard deviation 4, where dS = P (dP - r) cancels: an r from rounded outputs would be most of
    dq's error.  A rounding's mean square is at most (u x)^2 / 3, and those of P, dS and dq are independent:
      |dq error|^2 <= u^2 / 3 (dq^2 + z^2 sum_m dS^2 k^2 + z^2 (sum_m P k)^2 sum_j do_j^2 sum_m P^2 (v - P v)^2)
    summed over all values (P's roundings are in the numerator and the denominator of P v, whence v - P v;
    fp32's own errors are 2^-13 of this).  With r from rounded outputs it would be 1.07."""
    n, h, half = 700, 4, d // 2
    q, k, v, do, lam = _make([n], [n], h, d, dtype, 3, spread=2.0)
    got = _run(pkg, dev, q, k, v, do, lam, [0, n], None)["dq"].double().cpu().transpose(0, 1)
    Q, K, V, DO = (t.double().transpose(0, 1) for t in (q, k, v, do))
    z, u = 1 / math.sqrt(half), torch.finfo(dtype).eps / 2
    err = var = 0.0
    for i, f in enumerate((torch.ones(h, 1, 1, dtype=torch.float64), -lam.double().view(h, 1, 1))):
        m = slice(i * half, (i + 1) * half)
        P = torch.softmax(Q[..., m] @ K[..., m].transpose(1, 2) * z, 2)
        O = P @ V
        dS = P * (DO @ V.transpose(1, 2) - (DO * O).sum(2, keepdim=True)) * f
        dq = dS @ K[..., m] * z
        err += (got[..., m] - dq).square().sum()
        p2 = P.square()
        spread = p2 @ V.square() - 2 * O * (p2 @ V) + O.square() * p2.sum(2, keepdim=True)
        r = (DO.square() * spread).sum(2, keepdim=True) * (f * z * (P @ K[..., m])).square()
        var += (dq.square() + z * z * (dS.square() @ K[..., m].square()) + r).sum() * u * u / 3
    ratio = math.sqrt(err / var)
    print(f"    peaked maps {dtype} D={d}: dq error {ratio:.3f} of the roundings' bound", flush=True)
    assert ratio <= 1.0


def test_gradient_against_differences(pkg, dev):
    """Central differences of the definition in 64 bits (step 1e-4; their own error is of order 1e-8)
    along random directions."""
    lq, lkv, h, d, dtype = [9, 20], [31, 7], 2, 64, torch.float32
    q, k, v, do, lam = _make(lq, lkv, h, d, dtype, 1)
    cq, ck = _cu(lq), _cu(lkv)
    want = _oracle(q, k, v, do, lam, cq, ck, dtype)
    got = _run(pkg, dev, q, k, v, do, lam, cq, ck)
    base = [t.double() for t in (q, k, v)]
    g = torch.Generator().manual_seed(2)
    for i, name in enumerate(("dq", "dk", "dv", "dlam")):
        x = lam.double() if name == "dlam" else base[i]
        w = torch.randn(x.shape, generator=g, dtype=torch.float64)
        f = []
        for sign in (1, -1):
            m = list(base) + [lam.double()]
            m[i] = x + sign * 1e-4 * w
            f.append((_oracle(m[0], m[1], m[2], do, m[3], cq, ck, dtype)["out"][0] * do.double()).sum().item())
        diff = (f[0] - f[1]) / 2e-4
        tol = (want[name][1] * w.abs()).sum().item() + 1e-6 * abs(diff)
        dot = (got[name].cpu().double() * w).sum().item()
        print(f"  {name}: {dot:.6f} {diff:.6f}, off by {abs(dot - diff) / tol:.3f} of the tolerance", flush=True)
        assert abs(dot - diff) <= tol


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_of_a_fused_projection(pkg, dev, dtype):
    lens, h, d = [150, 77], 3, 64
    q, k, v, do, lam = _make(lens, lens, h, d, dtype, 5)
    cq = _cu(lens)
    want = _run(pkg, dev, q, k, v, do, lam, cq, None)
    qkv = torch.stack([q, k, v], 1).to(dev).requires_grad_()
    o = pkg.sparse_diff_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], lam.to(dev), cq)
    g, = torch.autograd.grad(o, qkv, do.to(dev))
    assert torch.equal(o, want["out"])
    for i, n in enumerate(("dq", "dk", "dv")):
        assert torch.equal(g[:, i], want[n])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_outside_every_sequence(pkg, dev, dtype):
    """Whatever stands in rows outside the sequences stays out; those rows are zero in new results and
    left alone in a given one."""
    d, h = 64, 2
    q, k, v, do, lam = _make([100], [90], h, d, dtype, 6)
    cq, ck = [5, 5, 40, 83], [3, 8, 60, 71]
    for t, lo, hi in ((q, 5, 83), (k, 3, 71), (v, 3, 71), (do, 5, 83)):
        t[:lo] = float("nan")
        t[hi:] = float("inf")
    clean = [torch.nan_to_num(t, nan=0, posinf=0) for t in (q, k, v, do)]
    want = _oracle(*clean, lam, cq, ck, dtype)
    got = _run(pkg, dev, q, k, v, do, lam, torch.tensor(cq, device=dev), torch.tensor(ck, device=dev))
    for n in got:
        _close(got[n], want[n], n)
    for n, lo, hi in (("out", 5, 83), ("dq", 5, 83), ("dk", 3, 71), ("dv", 3, 71)):
        assert not got[n][:lo].any() and not got[n][hi:].any()
    out = torch.full((100, h, d), 7.0, dtype=dtype, device=dev)
    pkg.sparse_diff_attention(*(t.to(dev) for t in (q, k, v, lam)), cq, ck, out=out)
    assert torch.equal(out[5:83], got["out"][5:83])
    assert bool((out[:5] == 7).all()) and bool((out[83:] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_infinite_values(pkg, dev, dtype, d):
    """An infinite v row of another sequence, past a sequence's last key, does not come in; the last
    key's own does (P1 and P2 both weigh it: infinity or NaN, never a number)."""
    lens = [1, 33, 64, 95]
    q, k, v, do, lam = _make(lens, lens, 2, d, dtype, 8)
    cq = _cu(lens)
    v[34] = float("inf")  # the first key of the third sequence
    out = pkg.sparse_diff_attention(*(t.to(dev) for t in (q, k, v, lam)), cq)
    assert out[:34].isfinite().all() and out[98:].isfinite().all()
    assert not out[34:98].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,h", [([32], 2), ([33, 1, 70], 3), ([700, 900], 16)])
def test_keys_that_no_query_sees(pkg, dev, dtype, d, lens, h):
    """A key of -inf in a dimension where every query is positive has scores of -inf, so P = 0 in that
    map, wherever the queries end in a tile.  One of -30000 there has scores at least 500 below the rest,
    whose exponential is 0 in fp32 too: the same bits, and finite ones, but for dq in that dimension,
    where 0 times infinity is NaN."""
    q, k, v, do, lam = _make(lens, lens, h, d, dtype, 17)
    cq, half = _cu(lens), d // 2
    q[..., 0], q[..., half] = q[..., 0].abs() + 0.2, q[..., half].abs() + 0.2
    rows = [lo + 20 for lo, n in zip(cq, lens) if n > 25]
    k[rows, :, 0], k[[r + 5 for r in rows], :, half] = -30000.0, -30000.0
    want = _run(pkg, dev, q, k, v, do, lam, cq, None)
    k[k == -30000] = -math.inf
    got = _run(pkg, dev, q, k, v, do, lam, cq, None)
    got["dq"][..., 0], got["dq"][..., half] = want["dq"][..., 0], want["dq"][..., half]
    for n in got:
        print(f"  diff attention unseen keys {dtype} D={d} {lens}: {n} has {int(got[n].isnan().sum())} NaN", flush=True)
        assert want[n].isfinite().all() and torch.equal(got[n], want[n]), n
    assert not got["dk"][rows][..., :half].any()


def test_hints_and_offsets(pkg, dev):
    """Too small lengths still cover every row; device offsets give the host offsets' bits and are not
    read back."""
    lens, h, d, dtype = [700, 3, 260], 3, 128, torch.bfloat16
    q, k, v, do, lam = _make(lens, lens, h, d, dtype, 9)
    cq = _cu(lens)
    want = _run(pkg, dev, q, k, v, do, lam, cq, None)
    cd = torch.tensor(cq, dtype=torch.int32, device=dev)
    small = _run(pkg, dev, q, k, v, do, lam, cd, cd, max_seqlen_q=1, max_seqlen_kv=1)
    ref = _oracle(q, k, v, do, lam, cq, cq, dtype)
    for n in want:
        _close(small[n], ref[n], n)
    args = [t.to(dev) for t in (q, k, v, lam)]
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = pkg.sparse_diff_attention(*args, cd)
    finally:
        torch.cuda.set_sync_debug_mode(0)
    assert torch.equal(got, want["out"])


@pytest.mark.parametrize("d,longest", [(64, 200), (128, 200), (128, 100)])
@pytest.mark.parametrize("dtype", TYPES)
def test_hints_below_the_lengths_with_shared_keys(pkg, dev, dtype, d, longest):
    """The parts of the keys reach over sequences far longer than max_seqlen_kv says, with idle parts
    for the short ones; rows behind a wrong max_seqlen_q are still covered."""
    lq, lkv, h = [3, 0, longest, 1], [6000, 100, 2500, 0], 2
    q, k, v, do, lam = _make(lq, lkv, h, d, dtype, 13)
    cq, ck = _cu(lq), _cu(lkv)
    want = _oracle(q, k, v, do, lam, cq, ck, dtype)
    for mq, mk in ((1, 600), (0, 0), (10 ** 6, 10 ** 6), (None, None)):
        got = _run(pkg, dev, q, k, v, do, lam, torch.tensor(cq, device=dev), torch.tensor(ck, device=dev),
                   max_seqlen_q=mq, max_seqlen_kv=mk)
        for n in got:
            _close(got[n], want[n], f"{n} ({mq}, {mk})")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_parts_held_to_the_scratch_there_is(pkg, dev, dtype, d):
    """Many short sequences beside a long one: fewer, longer parts of its keys than blocks could run."""
    lq, lkv, h = [32] * 99 + [1], [97] * 99 + [40000], 1
    q, k, v, do, lam = _make(lq, lkv, h, d, dtype, 19)
    cq, ck = _cu(lq), _cu(lkv)
    got = _run(pkg, dev, q, k, v, do, lam, cq, ck)
    want = _oracle(q, k, v, do, lam, cq, ck, dtype)
    for n in got:
        _close(got[n], want[n], n)


def test_incoming_gradient_at_an_odd_address(pkg, dev):
    """The gradient of a result that was joined to one value is a view 2 bytes into a larger one."""
    lens, h, d, dtype = [40, 9], 2, 64, torch.bfloat16
    q, k, v, do, lam = _make(lens, lens, h, d, dtype, 4)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, lam)]
    o = pkg.sparse_diff_attention(*leaves, _cu(lens))
    w = torch.cat([torch.ones(1, dtype=dtype), do.flatten()]).to(dev)
    got = torch.autograd.grad((torch.cat([o.new_ones(1), o.flatten()]) * w).sum(), leaves)
    want = torch.autograd.grad(pkg.sparse_diff_attention(*leaves, _cu(lens)), leaves, do.to(dev))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_block_without_gradients(pkg, dev):
    p, lam = _block(128, 2, torch.bfloat16, 5)
    d = {k: v.to(dev).requires_grad_() for k, v in p.items()}
    block = pkg.SparseDiffAttentionBlock3d(2, 16, d["nw"], d["nb"], d["wqkv"], d["bqkv"], lam.to(dev),
                                           d["wo"], d["bo"])
    coords = torch.zeros((40, 4), dtype=torch.int32, device=dev)
    assert not block(pkg.SparseTensor(torch.randn(40, 128, device=dev).bfloat16(), coords)).feats.requires_grad


def test_a_saved_input_that_is_written_is_refused(pkg, dev):
    """q, k and v are saved for the gradient: written to through a later call's `out`, it is refused."""
    q, k, v, do, lam = (t.to(dev) for t in _make([30], [30], 2, 64, torch.float32, 2))
    for i in range(3):
        saved = [t.clone() for t in (q, k, v)]
        o = pkg.sparse_diff_attention(*saved, lam.clone().requires_grad_(), [0, 30])
        with torch.no_grad():
            pkg.sparse_diff_attention(q, k, v, lam, [0, 30], out=saved[i])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            o.sum().backward()
    leaf = torch.zeros_like(q).requires_grad_()
    with pytest.raises(pkg.TscError, match="gradients"):
        pkg.sparse_diff_attention(q, k, v, lam, [0, 30], out=leaf)


def test_empty_inputs(pkg, dev):
    z = lambda n: torch.zeros((n, 2, 64), device=dev).requires_grad_()
    lam = torch.ones(2, device=dev).requires_grad_()
    for q, k, cq, ck in ((z(0), z(5), [0, 0], [0, 5]), (z(5), z(0), [0, 5], [0, 0]), (z(4), z(4), [0], [0]),
                         (z(0), z(0), [0], [0])):
        o = pkg.sparse_diff_attention(q, k, k, lam, cq, ck)
        g = torch.autograd.grad(o, (q, k, lam), torch.ones_like(o))
        assert o.shape == q.shape and not o.any() and not any(t.any() for t in g)


def test_c_calls_without_sequences_or_queries(pkg, dev):
    """B = 0: every row is outside, zeroed with zero_rest or left as it was; no queries: dk and dv of the
    sequences' rows are zeros whatever zero_rest is.  dlambda is zero either way."""
    import ctypes
    import sys

    P = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
    lib, hd = sys.modules["trellis2_amd._lib"].stream_handle(0)
    n, h, d = 50, 3, 64
    lam = torch.ones(h, device=dev)
    for code, dtype in ((0, torch.float32), (1, torch.float16), (2, torch.bfloat16)):
        x = torch.ones((n, h, d), dtype=dtype, device=dev)
        for rest in (0, 1):
            o, dq, dk, dv = (torch.full_like(x, 5.0) for _ in range(4))
            dl = torch.full_like(lam, 5.0)
            args = (hd, code, P(x), P(x), P(x), h * d, h * d, h * d, P(lam), None, None, 0, n, n, h, d, 0.0, n, n, rest)
            assert lib.tsc_diff_attention(*args, None, P(o), None, None) == 0
            maps, lse = torch.zeros((n, h, 2, d), device=dev), torch.zeros((2, h, n), device=dev)
            assert lib.tsc_diff_attention_backward(*args, P(maps), P(lse), P(x), None, P(dq), P(dk), P(dv), P(dl)) == 0
            for t in (o, dq, dk, dv):
                assert bool((t == 5 * (1 - rest)).all())
            assert not dl.any()
            cq = torch.zeros(3, dtype=torch.int32, device=dev)
            ck = torch.tensor([4, 20, 41], dtype=torch.int32, device=dev)
            nbytes = lib.tsc_diff_attention_workspace_bytes(code, 2, 0, n, h, d, 0, n, 1)
            ws = torch.full((nbytes // 4,), 7.0, device=dev)
            dk, dv, dl = torch.full_like(x, 5.0), torch.full_like(x, 5.0), torch.full_like(lam, 5.0)
            assert lib.tsc_diff_attention_backward(
                hd, code, None, P(x), P(x), h * d, h * d, h * d, P(lam), P(cq), P(ck), 2, 0, n, h, d, 0.0, 0, n, rest,
                None, None, None, P(ws), None, P(dk), P(dv), P(dl)) == 0
            for t in (dk, dv):
                assert not t[4:41].any() and bool((t[:4] == 5 * (1 - rest)).all())
                assert bool((t[41:] == 5 * (1 - rest)).all())
            assert not dl.any()


def test_c_gradients_over_inputs_are_refused(pkg, dev):
    """dlambda over lambda above all: other blocks still read lambda when dlambda is written."""
    import ctypes
    import sys

    P = lambda t: ctypes.c_void_p(t.data_ptr())
    lib, hd = sys.modules["trellis2_amd._lib"].stream_handle(0)
    n, h, d = 40, 2, 64
    b = {k: torch.ones((n, h, d), device=dev) for k in ("q", "k", "v", "dout", "dq", "dk", "dv")}
    b.update(lam=torch.ones(h, device=dev), dlam=torch.ones(h, device=dev), lse=torch.ones((2, h, n), device=dev),
             maps=torch.ones((n, h, 2, d), device=dev))
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    ws = torch.zeros(1 << 14, device=dev)

    def call(**other):
        x = {k: P(t) for k, t in {**b, **other}.items()}
        ld = h * d
        return lib.tsc_diff_attention_backward(
            hd, 0, x["q"], x["k"], x["v"], ld, ld, ld, x["lam"], P(cu), P(cu), 1, n, n, h, d, 0.0, n, n, 1, x["maps"],
            x["lse"], x["dout"], P(ws), x["dq"], x["dk"], x["dv"], x["dlam"])

    assert call() == 0
    for over in ({"dlam": b["lam"]}, {"dlam": b["lse"]}, {"dlam": b["dq"]}, {"dk": b["lse"]}, {"dlam": b["maps"]},
                 {"dq": b["q"]}, {"dv": b["dk"]}, {"dk": b["dout"]}):
        assert call(**over) == 1 and b"overlap" in lib.tsc_last_error(), list(over)


def test_same_bits_each_time_on_any_stream_and_in_a_graph(pkg, dev):
    """Sums have one order; captured training steps replay to the eager bits with new inputs, with
    eager work in between; two captured graphs share nothing."""
    for lq, lkv in (([500, 260], [500, 260]), ([2, 1], [4000, 700])):
        q, k, v, do, lam = (t.to(dev) for t in _make(lq, lkv, 4, 128, torch.bfloat16, 11))
        cq, ck = (torch.tensor(_cu(x), dtype=torch.int32, device=dev) for x in (lq, lkv))

        def step(q):
            leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
            o = pkg.sparse_diff_attention(*leaves, cq, ck)
            return [o.detach(), *torch.autograd.grad(o, leaves, do)]

        want = step(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(q)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, e) for a, e in zip(got, want))
        graphs = []
        for i in range(2):
            qs = q.clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs = step(qs)
            graphs.append((g, qs, outs))
        for rep in range(3):
            for i, (g, qs, outs) in enumerate(graphs):
                qs.copy_(q * (1 + 0.1 * rep + 0.05 * i))
                g.replay()
            for i, (g, qs, outs) in enumerate(graphs):
                eager = step(q * (1 + 0.1 * rep + 0.05 * i))
                torch.cuda.synchronize()
                assert all(torch.equal(a, e) for a, e in zip(outs, eager)), (rep, i)


def test_calls_of_several_threads_on_streams_of_their_own(pkg, dev):
    """Training steps of both operators from four threads at once give the bits of one after the other."""
    import threading

    cases = []
    for i in range(4):
        lq, lkv = ([3, 1, 9], [2500, 40, 900]) if i % 2 else ([300, 41], [300, 41])
        q, k, v, do, lam = (t.to(dev) for t in _make(lq, lkv, 4, 64, TYPES[i % 3], 30 + i))
        cq, ck = (torch.tensor(_cu(x), dtype=torch.int32, device=dev) for x in (lq, lkv))
        cases.append((q, k, v, do, lam, cq, ck))

    def step(q, k, v, do, lam, cq, ck):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
        o = pkg.sparse_diff_attention(*leaves, cq, ck)
        x = v.detach().flatten(1).requires_grad_()
        y = pkg.group_norm(x, 8, cu_rows=ck, silu=True)
        return [o.detach(), y.detach(), *torch.autograd.grad(o, leaves, do),
                *torch.autograd.grad(y, x, torch.ones_like(y))]

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got[i] = step(*cases[i])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_step_with_other_offsets(pkg, dev, dtype, d):
    """The offsets are read on the device: a replay goes by those of its time, parts of the keys included."""
    tq, tkv, h = 64, 6000, 2
    q, k, v, do, lam = (t.to(dev) for t in _make([tq], [tkv], h, d, dtype, 31))
    offsets = [([0, 1, 30, 64], [0, 5000, 5400, 6000]), ([0, 0, 64, 64], [0, 10, 5990, 6000]),
               ([5, 20, 20, 60], [100, 100, 200, 5999])]
    cq, ck = (torch.tensor(x, dtype=torch.int32, device=dev) for x in offsets[0])

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
        o = pkg.sparse_diff_attention(*leaves, cq, ck, max_seqlen_q=32, max_seqlen_kv=5000)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for a, b in offsets * 2:
        cq.copy_(torch.tensor(a))
        ck.copy_(torch.tensor(b))
        g.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want)), (a, b)
        ref = _oracle(*(t.cpu() for t in (q, k, v, do, lam)), a, b, dtype)
        for n, t in zip(("out", "dq", "dk", "dv", "dlam"), outs):
            _close(t, ref[n], n)


def test_rows_of_different_strides(pkg, dev):
    """q out of a projection with other values beside it, k and v out of one for both."""
    lq, lkv, h, d, dtype = [40, 33], [200, 65], 2, 128, torch.bfloat16
    q, k, v, do, lam = _make(lq, lkv, h, d, dtype, 32)
    cq, ck = _cu(lq), _cu(lkv)
    want = _run(pkg, dev, q, k, v, do, lam, cq, ck)
    wide = torch.full((sum(lq), h * d + 8), float("nan"), dtype=dtype)
    wide[:, 8:] = q.flatten(1)
    wide, kv = wide.to(dev).requires_grad_(), torch.stack([k, v], 1).to(dev).requires_grad_()
    o = pkg.sparse_diff_attention(wide[:, 8:].unflatten(1, (h, d)), kv[:, 0], kv[:, 1], lam.to(dev), cq, ck)
    gq, gkv = torch.autograd.grad(o, (wide, kv), do.to(dev))
    assert torch.equal(o, want["out"]) and torch.equal(gq[:, 8:].unflatten(1, (h, d)), want["dq"])
    assert torch.equal(gkv[:, 0], want["dk"]) and torch.equal(gkv[:, 1], want["dv"]) and not gq[:, :8].any()


def test_more_than_2_31_values(pkg, dev):
    """Keys past the 2^31st element of k and v, their gradients, and zeros before them."""
    h, d, dtype = 16, 128, torch.bfloat16
    n, lq, lk = 2 ** 31 // (h * d) + 3000, 40, 900
    q, ks, vs, do, lam = _make([lq], [lk], h, d, dtype, 12)
    k = torch.zeros((n, h, d), dtype=dtype, device=dev)
    v = torch.zeros_like(k)
    k[n - lk:], v[n - lk:] = ks.to(dev), vs.to(dev)
    got = _run(pkg, dev, q, k, v, do, lam, [0, 0, lq], [0, n - lk, n])
    want = _oracle(q, ks, vs, do, lam, [0, lq], [0, lk], dtype)
    for name in ("out", "dq", "dlam"):
        _close(got[name], want[name], name)
    for name in ("dk", "dv"):
        _close(got[name][n - lk:], want[name], name)
        assert not got[name][:n - lk].any()


def test_refusals_on_the_device(pkg, dev):
    q = torch.zeros((10, 2, 64), device=dev)
    lam = torch.zeros(2, device=dev)
    f = pkg.sparse_diff_attention
    for cu in ([0, 5, 4, 10], [0, 11], [[0, 10]]):
        with pytest.raises(pkg.TscError):
            f(q, q, q, lam, cu)
    with pytest.raises(pkg.TscError, match="differ in length"):
        f(q, q, q, lam, [0, 10], [0, 5, 10])
    with pytest.raises(pkg.TscError, match="cu_seqlens_kv is needed"):
        f(q, q[:7], q[:7], lam, [0, 10])
    with pytest.raises(pkg.TscError, match="GPU"):
        f(q, q, q.cpu(), lam, [0, 10])
    with pytest.raises(pkg.TscError, match="gradients"):
        f(q.clone().requires_grad_(), q, q, lam, [0, 10], out=torch.zeros_like(q))
    with pytest.raises(pkg.TscError, match="overlaps"):
        f(q, q, q, lam, [0, 10], out=q)
    off = torch.zeros(10 * 128 + 1, device=dev)[1:].view(10, 2, 64)
    with pytest.raises(pkg.TscError, match="aligned"):
        f(off, q, q, lam, [0, 10])
    odd = torch.zeros((10, 130), device=dev)[:, :128].unflatten(1, (2, 64))
    with pytest.raises(pkg.TscError, match="row stride"):
        f(odd, q, q, lam, [0, 10])


def _block(c, h, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)
    p = {"nw": 1 + 0.1 * n(c), "nb": 0.1 * n(c), "wqkv": n(3 * c, c) / c ** 0.5, "bqkv": 0.1 * n(3 * c),
         "wo": n(c, c) / c ** 0.5, "bo": 0.1 * n(c)}
    return {k: v.to(dtype) for k, v in p.items()}, 0.2 + 0.6 * torch.rand(h, generator=g)


def _block_ref(x, p, lam, cu, groups, h):
    """The block from its definition, differentiable, in x's type."""
    ys = []
    c = x.shape[1]
    for lo, hi in zip(cu, cu[1:]):
        t = x[lo:hi].view(hi - lo, groups, -1)
        var, mean = torch.var_mean(t, dim=(0, 2), keepdim=True, unbiased=False)
        t = ((t - mean) / (var + 1e-5).sqrt()).view(hi - lo, c) * p["nw"] + p["nb"]
        q, k, v = (t @ p["wqkv"].t() + p["bqkv"]).view(hi - lo, 3, h, c // h).permute(1, 2, 0, 3)
        half = c // h // 2
        a = [torch.softmax(q[..., m] @ k[..., m].transpose(1, 2) / half ** 0.5, 2)
             for m in (slice(0, half), slice(half, None))]
        o = (a[0] - lam.view(-1, 1, 1) * a[1]) @ v
        ys.append(x[lo:hi] + o.transpose(0, 1).reshape(hi - lo, c) @ p["wo"].t() + p["bo"])
    return torch.cat(ys)


@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 2e-2), (torch.float16, 2e-2), (torch.float32, 1e-4)])
def test_block_of_both_operators(pkg, dev, dtype, tol):
    """SparseDiffAttentionBlock3d (group norm, qkv, differential attention, out + x) on a SparseTensor
    of two samples, at the norm-wise tolerance of this library's blocks."""
    c, h, groups, lens = 256, 2, 32, (300, 190)
    p, lam = _block(c, h, dtype, 1)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((sum(lens), c), generator=g).to(dtype)
    coords = torch.cat([torch.cat([torch.full((n, 1), i), torch.randint(0, 64, (n, 3), generator=g)], 1)
                        for i, n in enumerate(lens)]).int()
    d = {k: v.to(dev) for k, v in p.items()}
    block = pkg.SparseDiffAttentionBlock3d(h, groups, d["nw"], d["nb"], d["wqkv"], d["bqkv"], lam.to(dev),
                                           d["wo"], d["bo"])
    y = block(pkg.SparseTensor(x.to(dev), coords.to(dev))).feats
    want = _block_ref(x.double(), {k: v.double() for k, v in p.items()}, lam.double(), _cu(lens), groups, h)
    err = ((y.double().cpu() - want).abs().max() / want.abs().max()).item()
    print(f"  block {dtype}: {err:.2e}", flush=True)
    assert err <= tol


def test_training_step_of_both_operators(pkg, dev):
    """The same block as a training step in fp32: this library's norm and attention around torch's
    linear layers; every gradient at the fp32 norm-wise tolerance."""
    c, h, groups, lens = 128, 2, 16, (200, 131)
    cu = _cu(lens)
    p, lam = _block(c, h, torch.float32, 3)
    g = torch.Generator().manual_seed(4)
    x, dy = torch.randn((sum(lens), c), generator=g), torch.randn((sum(lens), c), generator=g)
    ref = [t.double().requires_grad_() for t in (x, lam, *p.values())]
    yr = _block_ref(ref[0], dict(zip(p, ref[2:])), ref[1], cu, groups, h)
    gr = torch.autograd.grad(yr, ref, dy.double())
    lv = [t.to(dev).requires_grad_() for t in (x, lam, *p.values())]
    w = dict(zip(p, lv[2:]))
    t = pkg.group_norm(lv[0], groups, w["nw"], w["nb"], cu)
    qkv = torch.nn.functional.linear(t, w["wqkv"], w["bqkv"]).view(-1, 3, h, c // h)
    o = pkg.sparse_diff_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], lv[1], cu)
    y = lv[0] + torch.nn.functional.linear(o.reshape(-1, c), w["wo"], w["bo"])
    got = torch.autograd.grad(y, lv, dy.to(dev))
    for name, a, e in zip(("y", "x", "lam", *p), (y, *got), (yr, *gr)):
        err = ((a.detach().double().cpu() - e.detach()).abs().max() / e.detach().abs().max()).item()
        print(f"    {name}: {err:.2e}", flush=True)
        assert err <= 1e-4, name
