"""The modulated norms, window attention and gated residuals as they are used together: the block that the
package has of them, and a training step through all of them around torch's linear layers."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _tokens(pkg, dev, lens, c, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    coords = torch.cat([torch.stack([torch.full((n,), b), *(torch.arange(n),) * 3], 1) for b, n in enumerate(lens)])
    feats = torch.randn((sum(lens), c), generator=g).to(dtype)
    x = pkg.SparseTensor(feats.to(dev), coords.int().to(dev), batch_size=len(lens))
    return x, (0.3 * torch.randn((len(lens), 6, c), generator=g)).to(dtype).to(dev), g


def _weight(g, dtype, dev, *shape):
    return (torch.randn(shape, generator=g) / shape[-1] ** 0.5).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,causal,post", [(2, 2, False, None), (4, 1, True, "rms")])
def test_block(pkg, dev, dtype, heads, kv_heads, causal, post):
    """The block has the bits of its parts, called one by one on its intermediate results."""
    lens, d = [150, 61, 0, 9], 64
    c = heads * d
    x, mod, g = _tokens(pkg, dev, lens, c, dtype, heads)
    w = [_weight(g, dtype, dev, (heads + 2 * kv_heads) * d, c), _weight(g, dtype, dev, c, c),
         _weight(g, dtype, dev, 3 * c, c), _weight(g, dtype, dev, c, 3 * c)]
    b = [_weight(g, dtype, dev, t.shape[0]) for t in w]
    block = pkg.SparseModulatedBlock3d(heads, 30, w[0], b[0], w[1], b[1], w[2], b[2], w[3], b[3],
                                       num_kv_heads=kv_heads, sinks=3, causal=causal, post_norm=post)
    before = x.feats.clone()
    got = block(x, mod)
    assert torch.equal(x.feats, before) and got.coords is x.coords
    cu = np.cumsum([0] + lens).tolist()
    h = pkg.modulated_norm(x.feats, cu, mod[:, 1], mod[:, 0])
    qkv = pkg.sparse_linear(h, w[0], b[0]).view(-1, heads + 2 * kv_heads, d)
    q, k, v = (t.contiguous() for t in qkv.split([heads, kv_heads, kv_heads], 1))
    a = pkg.sparse_window_attention(q, k, v, 30, cu, sinks=3, causal=causal)
    a = pkg.sparse_linear(a.view(-1, c), w[1], b[1])
    r = pkg.gated_residual(x.feats, a, cu, mod[:, 2], post_norm=post)
    r2, h = pkg.gated_residual_norm(x.feats, a, cu, mod[:, 2], post_norm=post, scale=mod[:, 4], shift=mod[:, 3])
    assert torch.equal(r, r2)
    f = pkg.sparse_linear(pkg.silu(pkg.sparse_linear(h, w[2], b[2])), w[3], b[3])
    assert torch.equal(got.feats, pkg.gated_residual(r, f, cu, mod[:, 5], post_norm=post))
    with pytest.raises(ValueError, match="mod must be"):
        block(x, mod[:, :5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[0], [0, 0], [1], [0, 1]])
def test_block_of_one_row_or_none(pkg, dev, dtype, lens):
    heads, kv_heads, d = 2, 1, 64
    c = heads * d
    x, mod, g = _tokens(pkg, dev, lens, c, dtype, 3)
    w = [_weight(g, dtype, dev, (heads + 2 * kv_heads) * d, c), _weight(g, dtype, dev, c, c),
         _weight(g, dtype, dev, 2 * c, c), _weight(g, dtype, dev, c, 2 * c)]
    block = pkg.SparseModulatedBlock3d(heads, 30, w[0], None, w[1], None, w[2], None, w[3], None, num_kv_heads=kv_heads)
    got = block(x, mod)
    assert got.feats.shape == x.feats.shape and got.feats.dtype == dtype
    if sum(lens):  # one row attends to itself alone: its v, for both heads
        m = mod[-1:]
        h = pkg.modulated_norm(x.feats, None, m[:, 1], m[:, 0])
        v = pkg.sparse_linear(h, w[0], None)[:, -d:]
        a = pkg.sparse_linear(torch.cat([v, v], 1).contiguous(), w[1], None)
        r, h = pkg.gated_residual_norm(x.feats, a, None, m[:, 2], scale=m[:, 4], shift=m[:, 3])
        f = pkg.sparse_linear(pkg.silu(pkg.sparse_linear(h, w[2], None)), w[3], None)
        assert torch.equal(got.feats, pkg.gated_residual(r, f, None, m[:, 5]))


def _reference(x, mod, w1, w2, cu, heads, window, sinks):
    """The same step in fp64, from its definition."""
    def norm(t):
        return (t - t.mean(1, keepdim=True)) / torch.sqrt(t.var(1, unbiased=False, keepdim=True) + 1e-6)

    n, c = x.shape
    lens = torch.tensor([b - a for a, b in zip(cu, cu[1:])])
    m = mod.repeat_interleave(lens, 0)
    h = norm(x) * (1 + m[:, 1]) + m[:, 0]
    q, k, v = (h @ w1.t()).view(n, 3, heads, c // heads).permute(1, 2, 0, 3)
    sample = torch.repeat_interleave(torch.arange(len(lens)), lens)
    pos = torch.cat([torch.arange(i) for i in lens])
    see = (sample[:, None] == sample) & (((pos[:, None] - pos).abs() <= window) | (pos < sinks))
    p = torch.softmax((q @ k.transpose(1, 2) / (c // heads) ** 0.5).masked_fill(~see, float("-inf")), 2)
    a = (p @ v).transpose(0, 1).reshape(n, c) @ w2.t()
    r = x + m[:, 2] * a
    return r, norm(r) * (1 + m[:, 4]) + m[:, 3]


def test_training_step_through_all_of_them(pkg, dev):
    """fp32 against the definition's autograd in fp64.  An element of a gradient is a sum through two norms, two
    linear layers and a softmax, each of which passes relative errors of 2^-18 of the sizes at most on (their own
    tests' bounds at these lengths) and multiplies them by at most 4 (weights of unit gain, modulations within
    0.5 to 2, norms of rows of unit spread): 5 steps of a factor 4 from 2^-18 of the largest element, 2^-8 of it
    if all were to add up; a wrong factor or a missing term is of its own size."""
    lens, heads, d = [140, 75], 2, 64
    c = heads * d
    x, mod, g = _tokens(pkg, dev, lens, c, torch.float32, 5)
    w = [_weight(g, torch.float32, dev, 3 * c, c), _weight(g, torch.float32, dev, c, c)]
    dr, dh = (torch.randn((sum(lens), c), generator=g).to(dev) for _ in range(2))
    cu = np.cumsum([0] + lens).tolist()
    leaves = [t.detach().clone().requires_grad_() for t in (x.feats, mod, *w)]
    f, m = leaves[:2]
    h = pkg.modulated_norm(f, cu, m[:, 1], m[:, 0])
    qkv = torch.nn.functional.linear(h, leaves[2]).view(-1, 3, heads, d)
    a = pkg.sparse_window_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], 20, cu, sinks=2)
    a = torch.nn.functional.linear(a.flatten(1), leaves[3])
    r, h = pkg.gated_residual_norm(f, a, cu, m[:, 2], scale=m[:, 4], shift=m[:, 3])
    got = [r, h, *torch.autograd.grad([r, h], leaves, [dr, dh])]
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    want = list(_reference(*ref, cu, heads, 20, 2))
    want += torch.autograd.grad(want, ref, [dr.cpu().double(), dh.cpu().double()])
    for name, a, b in zip(("r", "h", "dx", "dmod", "dw1", "dw2"), got, want):
        off = ((a.detach().cpu().double() - b.detach()).abs().max() / b.detach().abs().max()).item()
        print(f"    {name}: off by {off:.2e} of the largest", flush=True)
        assert off <= 2.0 ** -8, (name, off)


def test_several_threads(pkg, dev):
    """Each op from four threads on streams of their own, at once: the bits of the calls one by one."""
    import threading

    def one(seed):
        g = torch.Generator().manual_seed(seed)
        n, c = 200 + 37 * seed, 128
        x, y, dy = (torch.randn((n, c), generator=g).to(dev) for _ in range(3))
        x.requires_grad_()
        cu = [0, 50 + seed, n]
        r, h = pkg.gated_residual_norm(x, y, cu, norm="rms", post_norm="layer")
        o = pkg.sparse_window_attention(h.view(n, 2, 64), x.view(n, 2, 64), y.view(n, 2, 64), 17, cu, sinks=seed)
        return [t.detach() for t in (r, h, o, *torch.autograd.grad(o, x, dy.view(n, 2, 64)))]

    want = [one(i) for i in range(4)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            s = torch.cuda.Stream(dev)
            with torch.cuda.stream(s):
                for _ in range(5):
                    got[i] = one(i)
            s.synchronize()
        except Exception as e:  # reported by the test, not by the thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
