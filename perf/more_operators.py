"""Performance cases of a transformer block over serialized voxels: attention in a sliding window along
the rows of each sample with a few first tokens that stay visible, and the norms before and after a
block with its gate and residual scale, forward and as training steps, through the package's public
entry points.

A case is a dict of plain values; "op" says what one pass is:

  wa        sparse_window_attention over packed sequences
  wa_step   the same and its gradients (q, k, v)
  mn        modulated_norm: each row's norm, scaled and shifted by its sample's modulation
  mn_step   the same and its gradients
  gr        gated_residual: residual_scale x + gate norm(y)
  gr_step   the same and its gradients
  grn       gated_residual_norm: that sum and the next block's modulated norm of it, in one pass
  grn_step  the same and its gradients

Sequences: "q" and "kv" are the lengths ("kv" empty: the queries' own rows), queries stand at the end
of their keys.  "rows" are the samples' lengths.  q and k make scores of a spread of 1.4; x and y are
N(0,1) with an offset and a spread per channel; norm weights are near 1, biases near 0; modulations
are rows of one (B, 6, C) tensor, as one linear layer makes them; output gradients are N(0,1).
"""
import functools
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def listed():
    return [
        # A few tokens of a few small objects in fp32: latency.
        {"name": "wa_small_f32", "op": "wa", "q": "311,1,0,150", "kv": "", "heads": 8, "kv_heads": 8,
         "dim": 64, "window": 64, "sinks": 4, "causal": False, "dtype": "f32"},
        # The flow transformer over the active voxels of two samples, serialized along a curve, with
        # register tokens in front.
        {"name": "wa_self_bf16", "op": "wa", "q": "9000,6143", "kv": "", "heads": 12, "kv_heads": 12,
         "dim": 128, "window": 512, "sinks": 16, "causal": False, "dtype": "bf16"},
        # The prompt of an autoregressive voxel decoder with shared key heads.
        {"name": "wa_causal_f16", "op": "wa", "q": "20011,4097", "kv": "", "heads": 16, "kv_heads": 4,
         "dim": 64, "window": 1023, "sinks": 4, "causal": True, "dtype": "f16"},
        # Its next token, eight objects at once.
        {"name": "wa_token_bf16", "op": "wa", "q": "1,1,1,1,1,1,1,1",
         "kv": "9000,6143,12011,4520,801,20011,7607,33", "heads": 16, "kv_heads": 4, "dim": 128,
         "window": 4095, "sinks": 4, "causal": True, "dtype": "bf16"},
        # A training step of the flow transformer.
        {"name": "wa_step_bf16", "op": "wa_step", "q": "9000,6143", "kv": "", "heads": 12,
         "kv_heads": 12, "dim": 128, "window": 256, "sinks": 16, "causal": False, "dtype": "bf16"},
        # A training step in fp32, small objects, shared key heads.
        {"name": "wa_step_f32", "op": "wa_step", "q": "1203,700", "kv": "", "heads": 8, "kv_heads": 2,
         "dim": 64, "window": 127, "sinks": 4, "causal": True, "dtype": "f32"},
        # Two very small objects at the coarsest level: latency.
        {"name": "mn_small_f32", "op": "mn", "rows": "611,397", "c": 64, "norm": "layer",
         "affine": False, "dtype": "f32"},
        # A training step of the norm before a block at the transformer's width.
        {"name": "mn_step_1536_bf16", "op": "mn_step", "rows": "9000,6143", "c": 1536, "norm": "layer",
         "affine": False, "dtype": "bf16"},
        # The norm after a block on an odd channel count, one sample empty.
        {"name": "gr_odd_f16", "op": "gr", "rows": "20011,0,31,6007", "c": 100, "post": "rms",
         "affine": True, "residual_scale": 0.5, "dtype": "f16"},
        # A training step of a gated residual in fp32.
        {"name": "gr_step_64_f32", "op": "gr_step", "rows": "25176", "c": 64, "post": "layer",
         "affine": True, "residual_scale": 1.0, "dtype": "f32"},
        # From one block into the next at the widest decoder level, two samples.
        {"name": "grn_1024_bf16", "op": "grn", "rows": "33003,31301", "c": 1024, "post": "none",
         "norm": "layer", "affine": False, "residual_scale": 1.0, "dtype": "bf16"},
        # The same as a training step of a middle level, four samples, with a norm after the block.
        {"name": "grn_step_512_bf16", "op": "grn_step", "rows": "61007,60211,62003,60326", "c": 512,
         "post": "rms", "norm": "rms", "affine": True, "residual_scale": 1.0, "dtype": "bf16"},
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


_WIDTHS = (32, 33, 64, 72, 96, 100, 128, 200, 256, 320, 512, 768, 1000, 1024, 1280, 1536, 2048)


def draw(rng):
    op = rng.choice(("wa", "wa", "wa_step", "mn", "mn_step", "gr", "gr_step", "grn", "grn_step"))
    dtype = rng.choice(("bf16", "f16", "f32"))
    if op not in ("wa", "wa_step"):
        c = rng.choice(_WIDTHS)
        most = 6.0e7 / (2 if dtype == "f32" else 1) / c
        lens = _split(rng, _log_int(rng, 1, int(min(most, 500000))), rng.randint(1, 5))
        case = {"op": op, "rows": _text(lens), "c": c, "affine": rng.random() < 0.5, "dtype": dtype}
        if op in ("gr", "gr_step", "grn", "grn_step"):
            case["post"] = rng.choice(("none", "layer", "rms"))
            case["residual_scale"] = rng.choice((1.0, 1.0, 0.5, 0.7071))
        if op not in ("gr", "gr_step"):
            case["norm"] = rng.choice(("layer", "rms"))
        return case
    heads, kv_heads, dim = rng.choice(((12, 12, 128), (16, 4, 64), (8, 1, 128), (24, 8, 64), (8, 8, 64),
                                       (3, 3, 128), (16, 16, 64), (20, 4, 128)))
    window = rng.choice((0, _log_int(rng, 1, 2047), _log_int(rng, 16, 2047), _log_int(rng, 16, 511)))
    sinks, causal = rng.choice((0, 1, 4, 16, 100)), rng.random() < 0.5
    seqs = rng.randint(1, 6)
    if op == "wa" and rng.random() < 0.35:  # the last tokens of long sequences
        q = [rng.randint(0 if i else 1, rng.choice((1, 1, 7, 33))) for i in range(seqs)]
        kv = [n + extra for n, extra in zip(q, _split(rng, _log_int(rng, 100, 60000), seqs))]
    else:
        span = (window if causal else 2 * window) + sinks + 64
        most = {"wa": 2.0e10, "wa_step": 8.0e9}[op] / (6 if dtype == "f32" else 1) / (heads * dim)
        total = _log_int(rng, 1 if op == "wa" else 100, 24000)
        total = max(1, min(total, int(most / min(span, total))))
        q, kv = _split(rng, total, seqs), []
        if op == "wa_step":  # scores have no gradient where a query sees one key
            window = max(window, 1)
    return {"op": op, "q": _text(q), "kv": _text(kv), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window, "sinks": sinks, "causal": causal, "dtype": dtype}


# ---- inputs ------------------------------------------------------------------------------------
_LEAVES = {"wa": ("q", "k", "v"), "mn": ("x", "scale", "shift", "w", "b"),
           "gr": ("x", "y", "gate", "pw", "pb"),
           "grn": ("x", "y", "gate", "pw", "pb", "scale", "shift", "w", "b")}


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
    op = case["op"].replace("_step", "")

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if op == "wa":
        aq = _offsets(_lens(case["q"]))
        ak = _offsets(_lens(case["kv"])) if case["kv"] else aq
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        s = {"q": normal(aq[-1], h, d).mul_(1.2).to(dt), "k": normal(ak[-1], hk, d).mul_(1.2).to(dt),
             "v": normal(ak[-1], hk, d).to(dt), "aq": aq, "ak": ak}
        if case["op"] == "wa_step":
            s["do"] = normal(aq[-1], h, d).to(dt)
        return s
    at = _offsets(_lens(case["rows"]))
    n, c, b = at[-1], case["c"], len(at) - 1

    def rows():
        return normal(n, c).mul_(1.0 + 0.3 * normal(c)).add_(0.7 * normal(c)).to(dt)

    mod = (0.3 * normal(b, 6, c)).to(dt)
    s = {"x": rows(), "at": at}
    if op in ("gr", "grn"):
        s["y"], s["gate"] = rows(), mod[:, 2]
        if case["affine"] and case["post"] != "none":
            s["pw"] = (1.0 + 0.1 * normal(c)).to(dt)
            if case["post"] == "layer":
                s["pb"] = (0.1 * normal(c)).to(dt)
    if op in ("mn", "grn"):
        s["shift"], s["scale"] = mod[:, 3], mod[:, 4]
        if case["affine"]:
            s["w"] = (1.0 + 0.1 * normal(c)).to(dt)
            if case["norm"] == "layer":
                s["b"] = (0.1 * normal(c)).to(dt)
    if case["op"].endswith("_step"):
        for name in {"mn": ("dh",), "gr": ("dr",), "grn": ("dr", "dh")}[op]:
            s[name] = normal(n, c).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["leaves"] = []
    if case["op"].endswith("_step"):
        s["leaves"] = [n for n in _LEAVES[case["op"].replace("_step", "")] if n in s]
        for name in s["leaves"]:
            s[name] = s[name].detach().requires_grad_()
    for name in ("at", "aq", "ak"):
        if name in s:
            s["cu_" + name] = torch.tensor(s[name], dtype=torch.int32, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"].replace("_step", "")
    if own:
        return _own(s, s["case"], op)
    with torch.no_grad():
        return _wa_plain(s, s["case"]) if op == "wa" else _norm_plain(s, s["case"], op)


@functools.lru_cache(maxsize=None)
def _package():
    from __graft_entry__ import load_package

    return load_package()


def _own(s, c, op):
    pkg = _package()
    post = {"post_norm": None if c.get("post", "none") == "none" else c["post"],
            "post_weight": s.get("pw"), "post_bias": s.get("pb")}
    pre = {"norm": c.get("norm"), "weight": s.get("w"), "bias": s.get("b"), "scale": s.get("scale"),
           "shift": s.get("shift")}
    if op == "wa":
        longest = [max(b - a for a, b in zip(s[n], s[n][1:])) for n in ("aq", "ak")]
        outs = {"out": pkg.sparse_window_attention(
            s["q"], s["k"], s["v"], c["window"], s["cu_aq"], s["cu_ak"], sinks=c["sinks"],
            causal=c["causal"], max_seqlen_q=longest[0], max_seqlen_kv=longest[1])}
        d_out = [s.get("do")]
    elif op == "mn":
        outs = {"h": pkg.modulated_norm(s["x"], s["cu_at"], eps=EPS, **pre)}
        d_out = [s.get("dh")]
    elif op == "gr":
        outs = {"r": pkg.gated_residual(s["x"], s["y"], s["cu_at"], gate=s["gate"], eps=EPS,
                                        residual_scale=c["residual_scale"], **post)}
        d_out = [s.get("dr")]
    else:
        r, h = pkg.gated_residual_norm(s["x"], s["y"], s["cu_at"], gate=s["gate"], eps=EPS,
                                       residual_scale=c["residual_scale"], **post, **pre)
        outs, d_out = {"r": r, "h": h}, [s.get("dr"), s.get("dh")]
    if not s["leaves"]:
        return outs
    grads = torch.autograd.grad(list(outs.values()), [s[n] for n in s["leaves"]], d_out)
    return {**{n: t.detach() for n, t in outs.items()},
            **{"d" + n: t for n, t in zip(s["leaves"], grads)}}


def _wa_plain(s, c):
    """Chunks of queries with the keys between the first and the last one that any of them sees, and the
    sinks; all heads at once."""
    q, k, v, w, sinks = s["q"], s["k"], s["v"], c["window"], c["sinks"]
    dt, h, hk, d = q.dtype, c["heads"], c["kv_heads"], c["dim"]
    g, sc = h // hk, 1.0 / math.sqrt(d)
    step = c["op"] == "wa_step"
    out = torch.zeros_like(q)
    if step:
        dq = torch.zeros_like(q)
        gk, gv = (torch.zeros(k.shape, device=k.device) for _ in range(2))

    def by_kv_head(t):  # (n, heads, D) -> (kv_heads, n * g, D)
        n = t.shape[0]
        return t.float().view(n, hk, g, d).permute(1, 0, 2, 3).reshape(hk, n * g, d)

    def rows(t):  # back
        n = t.shape[1] // g
        return t.view(hk, n, g, d).permute(1, 0, 2, 3).reshape(n, h, d)

    for a0, a1, b0, b1 in zip(s["aq"], s["aq"][1:], s["ak"], s["ak"][1:]):
        n, m = a1 - a0, b1 - b0
        per = max(1, min(1024, (1 << 28) // max(1, h * min(m, 2 * w + sinks + 1024))))
        for i in range(0, n, per):
            j = min(n, i + per)
            p = torch.arange(i, j, device=q.device) + (m - n)  # positions of the queries
            lo, hi = max(0, i + m - n - w), min(m, j + m - n + (0 if c["causal"] else w))
            first = min(sinks, m)
            ids = (torch.arange(max(hi, first), device=q.device) if lo <= first else
                   torch.cat([torch.arange(first, device=q.device),
                              torch.arange(lo, max(hi, lo), device=q.device)]))
            if not ids.numel():
                continue
            sees = (ids < sinks) | ((p[:, None] - ids).abs() <= w)
            if c["causal"]:
                sees = sees & (ids <= p[:, None])
            sees = sees.repeat_interleave(g, 0)
            ks, vs = (t[b0 + ids].float().transpose(0, 1).contiguous() for t in (k, v))
            qs = by_kv_head(q[a0 + i:a0 + j])
            e = torch.matmul(qs, ks.transpose(1, 2).contiguous()).mul_(sc).masked_fill_(~sees, -math.inf)
            e = torch.exp(e - e.amax(2, keepdim=True).clamp_min(-3e38))
            e /= e.sum(2, keepdim=True).clamp_min(1e-37)
            o = torch.matmul(e, vs)
            out[a0 + i:a0 + j] = rows(o).to(dt)
            if step:
                do = by_kv_head(s["do"][a0 + i:a0 + j])
                gv[b0 + ids] += torch.matmul(e.transpose(1, 2).contiguous(), do).transpose(0, 1)
                e *= torch.matmul(do, vs.transpose(1, 2).contiguous()) - (do * o).sum(2, keepdim=True)
                e *= sc
                dq[a0 + i:a0 + j] = rows(torch.matmul(e, ks)).to(dt)
                gk[b0 + ids] += torch.matmul(e.transpose(1, 2).contiguous(), qs).transpose(0, 1)
    if not step:
        return {"out": out}
    return {"out": out, "dq": dq, "dk": gk.to(dt), "dv": gv.to(dt)}


def _normalized(x, kind):
    """A row's norm and its 1 / sigma; x itself without a norm."""
    if kind == "none":
        return x, None
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    return x * rstd, rstd


def _through(d, xh, rstd, kind):
    """The gradient of what was normalized from that of its norm xh."""
    if kind == "none":
        return d
    t = d - xh * (d * xh).mean(1, keepdim=True)
    return rstd * (t - d.mean(1, keepdim=True) if kind == "layer" else t)


def _norm_plain(s, c, op):
    dt, at, cu = s["x"].dtype, s["at"], s["cu_at"]
    sample = torch.repeat_interleave(torch.arange(len(at) - 1, device=cu.device), (cu[1:] - cu[:-1]).long(),
                                     output_size=at[-1])

    def f(name):
        return s[name].float() if name in s else None

    def affine(t, w, b):
        t = t if w is None else t * w
        return t if b is None else t + b

    def of_sample(t):  # sums of the samples' rows
        return torch.stack([t[a:b].sum(0, dtype=torch.float64) for a, b in zip(at, at[1:])])

    x, r, o = f("x"), None, {}
    if op in ("gr", "grn"):
        gate, pw, pb = f("gate"), f("pw"), f("pb")
        yh, y_rstd = _normalized(f("y"), c["post"])
        v = affine(yh, pw, pb)
        x = c["residual_scale"] * x + gate[sample] * v
        o["r"] = x.to(dt)
    if op in ("mn", "grn"):
        scale, shift, w, b = f("scale"), f("shift"), f("w"), f("b")
        xh, rstd = _normalized(x, c["norm"])
        u = affine(xh, w, b)
        o["h"] = (u * (1.0 + scale[sample]) + shift[sample]).to(dt)
    if not s["leaves"]:
        return o
    d = f("dr")
    if op in ("mn", "grn"):
        dh = f("dh")
        o["dshift"], o["dscale"] = of_sample(dh), of_sample(dh * u)
        du = dh * (1.0 + scale[sample])
        if w is not None:
            o["dw"] = (du * xh).sum(0, dtype=torch.float64)
            o["db"] = du.sum(0, dtype=torch.float64)
            du = du * w
        d_in = _through(du, xh, rstd, c["norm"])
        d = d_in if d is None else d + d_in
    if op in ("gr", "grn"):
        o["dgate"] = of_sample(d * v)
        dv = d * gate[sample]
        if pw is not None:
            o["dpw"] = (dv * yh).sum(0, dtype=torch.float64)
            o["dpb"] = dv.sum(0, dtype=torch.float64)
            dv = dv * pw
        o["dy"] = _through(dv, yh, y_rstd, c["post"])
        d = d * c["residual_scale"]
    o["dx"] = d
    return {n: o[n].to(dt) for n in (*o,) if n[0] != "d" or n[1:] in s["leaves"]}


# ---- the definition in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"].replace("_step", "")
    return _wa_exact(s, case) if op == "wa" else _norm_exact(s, case, op)


def _wa_exact(s, c):
    step = c["op"] == "wa_step"
    group = c["heads"] // c["kv_heads"]
    o = {n: torch.zeros(s[m].shape, dtype=torch.float64, device="cuda")
         for n, m in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    for b in range(len(s["aq"]) - 1):
        qr, kr = slice(*s["aq"][b:b + 2]), slice(*s["ak"][b:b + 2])
        n, m = qr.stop - qr.start, kr.stop - kr.start
        if n == 0 or m == 0:
            continue
        key = torch.arange(m, device="cuda")
        for hk in range(c["kv_heads"]):
            k = s["k"][kr, hk].double().requires_grad_(step)
            v = s["v"][kr, hk].double().requires_grad_(step)
            for h in range(hk * group, (hk + 1) * group):
                chunk = max(1, (1 << 26) // m)
                for i in range(0, n, chunk):
                    rows = slice(qr.start + i, min(qr.stop, qr.start + i + chunk))
                    pos = torch.arange(i, i + rows.stop - rows.start, device="cuda")[:, None] + m - n
                    hidden = (key >= c["sinks"]) & ((key - pos).abs() > c["window"])
                    if c["causal"]:
                        hidden |= key > pos
                    q = s["q"][rows, h].double().requires_grad_(step)
                    z = (q @ k.t() / c["dim"] ** 0.5).masked_fill(hidden, -1e300)
                    a = torch.softmax(z, 1).masked_fill(hidden, 0.0) @ v
                    o["out"][rows, h] = a.detach()
                    if step:
                        a.backward(s["do"][rows, h].double())
                        o["dq"][rows, h] = q.grad
            if step:
                o["dk"][kr, hk], o["dv"][kr, hk] = k.grad, v.grad
    return o if step else {"out": o["out"]}


def _norm_exact(s, c, op):
    step = c["op"].endswith("_step")
    t = {n: x.double().requires_grad_(step) for n, x in s.items() if n in _LEAVES["grn"]}
    n = torch.tensor([b - a for a, b in zip(s["at"], s["at"][1:])], device="cuda")

    def spread(m):  # a row per sample -> a row per voxel
        return m.repeat_interleave(n, 0)

    def norm(x, kind, w, b):
        if kind == "layer":
            var, mean = torch.var_mean(x, 1, keepdim=True, unbiased=False)
            x = (x - mean) * (var + EPS).rsqrt()
        elif kind == "rms":
            x = x * (x.square().mean(1, keepdim=True) + EPS).rsqrt()
        return (x if w is None else x * w) + (0.0 if b is None else b)

    x, o = t["x"], {}
    if op in ("gr", "grn"):
        x = o["r"] = (c["residual_scale"] * x
                      + spread(t["gate"]) * norm(t["y"], c["post"], t.get("pw"), t.get("pb")))
    if op in ("mn", "grn"):
        o["h"] = norm(x, c["norm"], t.get("w"), t.get("b")) * (1 + spread(t["scale"])) + spread(t["shift"])
    if step:
        names = [m for m in _LEAVES[op] if m in s]
        grads = torch.autograd.grad(list(o.values()), [t[m] for m in names],
                                    [s["d" + m].double() for m in o])
        o.update({"d" + m: g for m, g in zip(names, grads)})
    return {m: x.detach() for m, x in o.items()}


# ---- what a pass cannot do without -------------------------------------------------------------
def work(case):
    es = ES[case["dtype"]]
    op, step = case["op"].replace("_step", ""), case["op"].endswith("_step")
    if op == "wa":
        lq = _lens(case["q"])
        lk = _lens(case["kv"]) if case["kv"] else lq
        w, sinks, right = case["window"], case["sinks"], 0 if case["causal"] else case["window"]
        pairs = keys = 0
        for n, m in zip(lq, lk):
            for p in range(m - n, m):  # keys in the window, and the sinks outside of it
                lo, hi = max(0, p - w), min(m, p + right + 1)
                first = min(sinks, m, p + 1 if case["causal"] else m)
                inside = max(0, min(hi, first) - lo) if hi > lo else 0
                pairs += max(0, hi - lo) + max(0, first) - inside
            keys += min(m, n + w + sinks) if n else 0
        hd = case["heads"] * case["dim"]
        io = 2 * sum(lq) * hd + 2 * keys * case["kv_heads"] * case["dim"]  # q, out; k, v
        # scores and weighted sums; the step adds dP, dv, dq and dk, reads dout and writes dq, dk, dv
        return {"bytes": es * io * (2 if step else 1), "flops": (12 if step else 4) * hd * pairs}
    values = sum(_lens(case["rows"])) * case["c"]
    streams = {"mn": 2, "gr": 3, "grn": 4}[op]            # inputs and outputs of the forward pass
    streams += {"mn": 2, "gr": 3, "grn": 4}[op] if step else 0  # and of the step beyond them
    flops = {"mn": 10, "gr": 10, "grn": 18}[op] * (3 if step else 1)
    rows = {"mn": 2, "gr": 1, "grn": 3}[op] * len(_lens(case["rows"])) * case["c"]
    return {"bytes": es * (streams * values + rows * (2 if step else 1)), "flops": flops * values}
