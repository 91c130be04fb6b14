"""Performance cases of the normalization and attention operators of a sparse transformer / U-Net
block over active voxels, forward and as training steps, through the package's public entry points.

A case is a dict of plain values; "op" says what one pass is:

  gn       group_norm over the rows of each sample of a (N, C) feature matrix, SiLU fused or not
  gn_step  the same and its gradients (features, weight, bias)
  da       sparse_diff_attention over packed sequences (self: "kv" empty; else cross)
  da_step  the same and its gradients (q, k, v, lambda)

"rows", "q" and "kv" are the samples' lengths.  Features are N(0,1) with an offset and a spread per
channel, as a conv leaves them; norm weights are near 1, biases near 0; q and k make scores of
a spread of 1.4, lambda is in [0.2, 0.8]; output gradients are N(0,1).
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # Two very small objects at the coarsest level: latency.
        {"name": "gn_small_f32", "op": "gn", "rows": "611,397", "c": 64, "groups": 32, "silu": True,
         "dtype": "f32"},
        # The widest blocks of the decoder, two samples.
        {"name": "gn_1024_bf16", "op": "gn", "rows": "33003,31301", "c": 1024, "groups": 32,
         "silu": True, "dtype": "bf16"},
        # The finest level, narrow rows, no activation.
        {"name": "gn_512grid_f16", "op": "gn", "rows": "1514003", "c": 32, "groups": 8,
         "silu": False, "dtype": "f16"},
        # An odd channel count whose groups end inside 16-byte pieces, one sample empty.
        {"name": "gn_odd_bf16", "op": "gn", "rows": "20011,0,31,6007", "c": 100, "groups": 20,
         "silu": True, "dtype": "bf16"},
        # A training step of the middle decoder level, four samples.
        {"name": "gn_step_512_bf16", "op": "gn_step", "rows": "61007,60211,62003,60326", "c": 512,
         "groups": 32, "silu": True, "dtype": "bf16"},
        # A training step of a small fp32 level.
        {"name": "gn_step_64_f32", "op": "gn_step", "rows": "25176", "c": 64, "groups": 32,
         "silu": True, "dtype": "f32"},
        # A few tokens of a few small objects in fp32: latency.
        {"name": "da_small_f32", "op": "da", "q": "311,1,0,150", "kv": "", "heads": 8, "dim": 64,
         "dtype": "f32"},
        # Self-attention of the flow transformer over the active voxels of two samples.
        {"name": "da_self_bf16", "op": "da", "q": "9000,6143", "kv": "", "heads": 12, "dim": 128,
         "dtype": "bf16"},
        # Cross-attention of many small objects to their condition tokens.
        {"name": "da_cross_f16", "op": "da", "q": "5003,4817,5310,5500,5120,5133,5128",
         "kv": "1374,1374,1374,1374,1374,1374,1374", "heads": 16, "dim": 64, "dtype": "f16"},
        # One pooled read-out token per object over all of its voxels.
        {"name": "da_one_bf16", "op": "da", "q": "1,1,1,1", "kv": "9000,6143,12011,4520",
         "heads": 12, "dim": 128, "dtype": "bf16"},
        # A training step of the flow transformer.
        {"name": "da_step_bf16", "op": "da_step", "q": "4700,2907", "kv": "", "heads": 12,
         "dim": 128, "dtype": "bf16"},
        # A training step in fp32, small objects.
        {"name": "da_step_f32", "op": "da_step", "q": "1203,700", "kv": "", "heads": 8, "dim": 64,
         "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _split(rng, total, parts):
    """`total` rows over `parts` samples, uneven; a sample may be empty."""
    w = [rng.choice((0.0, 0.3, 1.0, 1.0, 2.0)) + 1e-3 * rng.random() for _ in range(parts)]
    cut = [int(total * sum(w[:i + 1]) / sum(w)) for i in range(parts)]
    cut[-1] = total
    return [b - a for a, b in zip([0] + cut, cut)]


def _text(lens):
    return ",".join(str(n) for n in lens)


def _lens(text):
    return [int(n) for n in text.split(",")] if text else []


_WIDTHS = ((32, 8), (32, 32), (64, 32), (64, 16), (72, 12), (100, 20), (96, 32), (128, 32),
           (48, 16), (256, 32), (320, 32), (512, 32), (1024, 32), (13, 13), (33, 1))


def draw(rng):
    op = rng.choice(("gn", "gn_step", "da", "da", "da_step"))
    dtype = rng.choice(("bf16", "f16", "f32"))
    if op in ("gn", "gn_step"):
        c, groups = rng.choice(_WIDTHS)
        most = {"gn": 6.0e7, "gn_step": 6.0e7}[op] / (2 if dtype == "f32" else 1) / c
        lens = _split(rng, _log_int(rng, 1, int(min(most, 1500000))), rng.randint(1, 5))
        return {"op": op, "rows": _text(lens), "c": c, "groups": groups,
                "silu": rng.random() < 0.6, "dtype": dtype}
    heads, dim = rng.choice(((12, 128), (16, 64), (8, 128), (24, 64), (8, 64), (3, 128)))
    seqs = rng.randint(1, 6)
    most = {"da": 11000, "da_step": 4500}[op] // (3 if dtype == "f32" else 1)
    form = rng.choice(("self", "cross", "few")) if op == "da" else rng.choice(("self", "cross"))
    if form == "self":
        return {"op": op, "q": _text(_split(rng, _log_int(rng, 1, most), seqs)), "kv": "",
                "heads": heads, "dim": dim, "dtype": dtype}
    if form == "few":
        q = [rng.randint(0 if i else 1, rng.choice((1, 1, 7, 33))) for i in range(seqs)]
        kv = _split(rng, _log_int(rng, 100, 40000), seqs)
    else:
        q = _split(rng, _log_int(rng, 1, most), seqs)
        kv = _split(rng, _log_int(rng, 1, 1600), seqs)
    return {"op": op, "q": _text(q), "kv": _text(kv), "heads": heads, "dim": dim, "dtype": dtype}


# ---- inputs ------------------------------------------------------------------------------------
def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _inputs(case, seed):
    """The case's tensors on the GPU in its type, from the seed alone."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if case["op"] in ("gn", "gn_step"):
        at = _offsets(_lens(case["rows"]))
        c = case["c"]
        x = normal(at[-1], c).mul_(1.0 + 0.3 * normal(c)).add_(0.7 * normal(c)).to(dt)
        s = {"x": x, "w": (1.0 + 0.1 * normal(c)).to(dt), "b": (0.1 * normal(c)).to(dt), "at": at}
        if case["op"] == "gn_step":
            s["dy"] = normal(at[-1], c).to(dt)
        return s
    aq = _offsets(_lens(case["q"]))
    ak = _offsets(_lens(case["kv"])) if case["kv"] else aq
    h, d = case["heads"], case["dim"]
    s = {"q": normal(aq[-1], h, d).mul_(1.2).to(dt), "k": normal(ak[-1], h, d).mul_(1.2).to(dt),
         "v": normal(ak[-1], h, d).to(dt), "aq": aq, "ak": ak,
         "lam": 0.2 + 0.6 * torch.rand((h,), generator=g, device=dev)}
    if case["op"] == "da_step":
        s["do"] = normal(aq[-1], h, d).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    leaves = {"gn_step": ("x", "w", "b"), "da_step": ("q", "k", "v", "lam")}.get(case["op"], ())
    dev = torch.device("cuda")
    for name in ("at", "aq", "ak"):
        if name in s:
            s["cu_" + name] = torch.tensor(s[name], dtype=torch.int32, device=dev)
    if own:
        from __graft_entry__ import load_package

        s["pkg"] = load_package()
        for name in leaves:
            s[name].requires_grad_()
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if c["op"] in ("gn", "gn_step"):
        return _gn_own(s, c) if own else _gn_plain(s, c)
    return _da_own(s, c) if own else _da_plain(s, c)


def _gn_own(s, c):
    y = s["pkg"].group_norm(s["x"], c["groups"], s["w"], s["b"], cu_rows=s["cu_at"], eps=EPS,
                            silu=c["silu"])
    if c["op"] == "gn":
        return y
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _da_own(s, c):
    longest = [max(b - a for a, b in zip(s[n], s[n][1:])) for n in ("aq", "ak")]
    o = s["pkg"].sparse_diff_attention(s["q"], s["k"], s["v"], s["lam"], s["cu_aq"], s["cu_ak"],
                                       max_seqlen_q=longest[0], max_seqlen_kv=longest[1])
    if c["op"] == "da":
        return o
    dq, dk, dv, dlam = torch.autograd.grad(o, (s["q"], s["k"], s["v"], s["lam"]), s["do"])
    return {"out": o.detach(), "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def _gn_plain(s, c):
    x, w, b = s["x"], s["w"].float(), s["b"].float()
    g, ch, dt = c["groups"], c["c"], s["x"].dtype
    step = c["op"] == "gn_step"
    y = torch.empty_like(x)
    if step:
        dx = torch.empty_like(x)
        dw = torch.zeros(ch, dtype=torch.float64, device=x.device)
        db = torch.zeros_like(dw)
    for r0, r1 in zip(s["at"], s["at"][1:]):
        if r0 == r1:
            continue
        n = (r1 - r0) * (ch // g)

        def per_channel(t):  # a value per group -> per channel
            return t.float().repeat_interleave(ch // g)

        xs = x[r0:r1].float()
        mean = xs.sum(0, dtype=torch.float64).view(g, -1).sum(1) / n
        xs = xs - per_channel(mean)
        var = (xs * xs).sum(0, dtype=torch.float64).view(g, -1).sum(1) / n
        rstd = per_channel(1.0 / torch.sqrt(var + EPS))
        xh = xs * rstd
        h = xh * w + b
        if c["silu"]:
            sig = 1.0 / (1.0 + torch.exp(-h))
            y[r0:r1] = (h * sig).to(dt)
        else:
            y[r0:r1] = h.to(dt)
        if step:
            dh = s["dy"][r0:r1].float()
            if c["silu"]:
                dh = dh * (sig * (1.0 + h * (1.0 - sig)))
            sb = dh.sum(0, dtype=torch.float64)
            sw = (dh * xh).sum(0, dtype=torch.float64)
            db += sb
            dw += sw
            ga = per_channel((sb * w).view(g, -1).sum(1) / n)
            gb = per_channel((sw * w).view(g, -1).sum(1) / n)
            dx[r0:r1] = (rstd * (dh * w - ga - xh * gb)).to(dt)
    if not step:
        return y
    return {"y": y, "dx": dx, "dw": dw.to(dt), "db": db.to(dt)}


def _chunk(nk):
    """Queries whose score rows over nk keys come to about 2^26 values."""
    return max(1, (1 << 26) // max(nk, 1))


def _softmax(s):
    e = torch.exp(s - s.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _da_plain(s, c):
    q, k, v, lam = s["q"], s["k"], s["v"], s["lam"]
    dt, d = q.dtype, c["dim"]
    half, sc = d // 2, 1.0 / math.sqrt(d // 2)
    step = c["op"] == "da_step"
    out = torch.zeros_like(q)
    if step:
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dlam = torch.zeros(c["heads"], dtype=torch.float64, device=q.device)
    for (a0, a1), (b0, b1) in zip(zip(s["aq"], s["aq"][1:]), zip(s["ak"], s["ak"][1:])):
        if a0 == a1 or b0 == b1:
            continue
        for h in range(c["heads"]):
            ks, vs = k[b0:b1, h].float(), v[b0:b1, h].float()
            k1, k2 = ks[:, :half], ks[:, half:]
            if step:
                gk = torch.zeros_like(ks)
                gv = torch.zeros_like(vs)
            for i in range(a0, a1, _chunk(b1 - b0)):
                j = min(a1, i + _chunk(b1 - b0))
                qs = q[i:j, h].float()
                p1 = _softmax(qs[:, :half] @ k1.t() * sc)
                p2 = _softmax(qs[:, half:] @ k2.t() * sc)
                p = p1 - lam[h] * p2
                out[i:j, h] = (p @ vs).to(dt)
                if step:
                    do = s["do"][i:j, h].float()
                    dp = do @ vs.t()
                    gv += p.t() @ do
                    r1 = (p1 * dp).sum(1, keepdim=True)
                    r2 = (p2 * dp).sum(1, keepdim=True)
                    dlam[h] -= r2.sum(dtype=torch.float64)
                    d1 = p1 * (dp - r1) * sc
                    d2 = p2 * (dp - r2) * (-lam[h] * sc)
                    dq[i:j, h, :half] = (d1 @ k1).to(dt)
                    dq[i:j, h, half:] = (d2 @ k2).to(dt)
                    gk[:, :half] += d1.t() @ qs[:, :half]
                    gk[:, half:] += d2.t() @ qs[:, half:]
            if step:
                dk[b0:b1, h] = gk.to(dt)
                dv[b0:b1, h] = gv.to(dt)
    if not step:
        return out
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam.float()}


# ---- the definition in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    return _gn_exact(s, case) if case["op"] in ("gn", "gn_step") else _da_exact(s, case)


def _gn_exact(s, c):
    step = c["op"] == "gn_step"
    w, b = s["w"].double().requires_grad_(step), s["b"].double().requires_grad_(step)
    ys, dxs = [], []
    for lo, hi in zip(s["at"], s["at"][1:]):
        x = s["x"][lo:hi].double().requires_grad_(step)
        if hi > lo:
            t = x.view(hi - lo, c["groups"], -1)
            var, mean = torch.var_mean(t, dim=(0, 2), keepdim=True, unbiased=False)
            y = ((t - mean) * (var + EPS).rsqrt()).view(hi - lo, -1) * w + b
            if c["silu"]:
                y = y * torch.sigmoid(y)
        else:
            y = x
        if step:
            if hi > lo:
                y.backward(s["dy"][lo:hi].double())
                dxs.append(x.grad)
            else:
                dxs.append(torch.zeros_like(x))
        ys.append(y.detach())
    if not step:
        return torch.cat(ys)
    return {"y": torch.cat(ys), "dx": torch.cat(dxs),
            "dw": torch.zeros_like(w) if w.grad is None else w.grad,
            "db": torch.zeros_like(b) if b.grad is None else b.grad}


def _da_exact(s, c):
    step = c["op"] == "da_step"
    names = ("q", "k", "v", "lam")
    half = c["dim"] // 2
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    grads = {n: torch.zeros(s[n].shape, dtype=torch.float64, device=out.device) for n in names}
    for b in range(len(s["aq"]) - 1):
        qr, kr = slice(*s["aq"][b:b + 2]), slice(*s["ak"][b:b + 2])
        nk = kr.stop - kr.start
        if qr.stop == qr.start or nk == 0:
            continue
        for h in range(c["heads"]):
            k = s["k"][kr, h].double().requires_grad_(step)
            v = s["v"][kr, h].double().requires_grad_(step)
            lam = s["lam"][h].double().requires_grad_(step)
            for i in range(qr.start, qr.stop, _chunk(2 * nk)):
                rows = slice(i, min(qr.stop, i + _chunk(2 * nk)))
                q = s["q"][rows, h].double().requires_grad_(step)
                a = [torch.softmax(q[:, m] @ k[:, m].t() / half ** 0.5, dim=1)
                     for m in (slice(0, half), slice(half, 2 * half))]
                o = a[0] @ v - lam * (a[1] @ v)
                out[rows, h] = o.detach()
                if step:
                    o.backward(s["do"][rows, h].double())
                    grads["q"][rows, h] = q.grad
            if step:
                grads["k"][kr, h], grads["v"][kr, h] = k.grad, v.grad
                grads["lam"][h] += lam.grad
    if not step:
        return out
    return {"out": out, **{"d" + n: grads[n] for n in names}}


# ---- what a pass cannot do without -------------------------------------------------------------
def work(case):
    es = ES[case["dtype"]]
    if case["op"] in ("gn", "gn_step"):
        c = case["c"]
        values = sum(_lens(case["rows"])) * c
        silu = 4 if case["silu"] else 0
        if case["op"] == "gn":  # x in, y out; mean, variance, normalization, activation
            return {"bytes": es * (2 * values + 2 * c), "flops": (8 + silu) * values}
        # x and dy in, y and dx out
        return {"bytes": es * (4 * values + 4 * c), "flops": (8 + silu + 14 + 2 * silu) * values}
    lq = _lens(case["q"])
    lk = _lens(case["kv"]) if case["kv"] else lq
    hd = case["heads"] * case["dim"]
    pairs = sum(a * b for a, b in zip(lq, lk))
    # both maps' scores and the product of their difference with v: 2 D each per pair and head;
    # the step adds dP, dv, dq and dk
    if case["op"] == "da":
        return {"bytes": es * hd * (2 * sum(lq) + 2 * sum(lk)) + 4 * case["heads"],
                "flops": 4 * hd * pairs}
    return {"bytes": es * hd * (4 * sum(lq) + 4 * sum(lk)) + 8 * case["heads"],
            "flops": 12 * hd * pairs}
