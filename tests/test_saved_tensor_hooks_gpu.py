"""Training steps whose saved tensors are offloaded, or come back in another layout, have the bits of the same
steps without hooks: q, k and v as slices of one projection, the modulation as slices of one (B, 6, C)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _nothing(t):
    return t


def _transposed(t):
    """The last axis outermost."""
    return t.movedim(-1, 0).contiguous().movedim(0, -1) if t.dim() > 1 else t.clone()


def _misaligned(t):
    """Contiguous, q, k, v, out and statistics behind one element (rows of values may be: sums in another order)."""
    if t.dim() != 3:
        return t.clone()
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


HOOKS = {
    "offloaded": lambda: torch.autograd.graph.save_on_cpu(),
    "offloaded to pinned memory": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    "transposed": lambda: torch.autograd.graph.saved_tensors_hooks(_nothing, _transposed),
    "misaligned": lambda: torch.autograd.graph.saved_tensors_hooks(_nothing, _misaligned),
}


def _same(leaves, call, douts, hook):
    want_o = call()
    want = torch.autograd.grad(want_o, leaves, douts)
    with hook():
        got_o = call()
    got = torch.autograd.grad(got_o, leaves, douts)
    for a, b in zip((*got_o, *got), (*want_o, *want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("lens,h,hk,d", [([70, 0, 33], 4, 2, 64), ([300], 3, 3, 128)])
def test_window_attention(pkg, dev, dtype, hook, lens, h, hk, d):
    g = torch.Generator().manual_seed(61)
    n = sum(lens)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    qkv = torch.randn((n, h + 2 * hk, d), generator=g).to(dtype).to(dev).requires_grad_()
    do = torch.randn((n, h, d), generator=g).to(dtype).to(dev)
    _same([qkv], lambda: [pkg.sparse_window_attention(qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:], 20, cu, sinks=2)],
          [do], HOOKS[hook])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("c", [64, 100, 1536])
@pytest.mark.parametrize("op", ["mn", "gr", "grn"])
def test_norms(pkg, dev, dtype, hook, c, op):
    g = torch.Generator().manual_seed(67)
    n = 51
    cu = torch.tensor([0, 20, 51], dtype=torch.int32, device=dev)

    def leaf(*shape):
        return torch.randn(shape, generator=g).to(dtype).to(dev).requires_grad_()

    x, y, w, b, mod = leaf(n, c), leaf(n, c), leaf(c), leaf(c), leaf(2, 6, c)
    d = [leaf(n, c).detach() for _ in range(2)]
    if op == "mn":
        leaves, call = [x, w, b, mod], lambda: [pkg.modulated_norm(x, cu, mod[:, 1], mod[:, 0], weight=w, bias=b)]
    elif op == "gr":
        leaves = [x, y, w, b, mod]

        def call():
            return [pkg.gated_residual(x, y, cu, mod[:, 2], 0.5, "rms", w, b)]
    else:
        leaves = [x, y, w, b, mod]

        def call():
            return pkg.gated_residual_norm(x, y, cu, mod[:, 2], 0.5, "layer", w, b, scale=mod[:, 4], shift=mod[:, 3])
    _same(leaves, call, d[:1 if op != "grn" else 2], HOOKS[hook])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hook", HOOKS)
def test_group_norm_and_diff_attention(pkg, dev, dtype, hook):
    g = torch.Generator().manual_seed(71)
    n, h, d = 51, 2, 64
    cu = torch.tensor([0, 20, 51], dtype=torch.int32, device=dev)

    def leaf(*shape):
        return torch.randn(shape, generator=g).to(dtype).to(dev).requires_grad_()

    x, w, b, dy = leaf(n, 96), leaf(96), leaf(96), leaf(n, 96).detach()
    _same([x, w, b], lambda: [pkg.group_norm(x, 8, w, b, cu, silu=True)], [dy], HOOKS[hook])
    qkv, do = leaf(n, 3, h, d), leaf(n, h, d).detach()
    lam = torch.rand(h, generator=g).to(dev).requires_grad_()
    _same([qkv, lam], lambda: [pkg.sparse_diff_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], lam, cu)], [do], HOOKS[hook])


@pytest.mark.parametrize("dtype", TYPES)
def test_checkpointed_step(pkg, dev, dtype):
    """Recomputed in the backward pass, which hands its tensors to the gradients through hooks."""
    from torch.utils.checkpoint import checkpoint

    g = torch.Generator().manual_seed(73)
    n, h, d = 90, 2, 64
    c = h * d
    cu = torch.tensor([0, 50, 90], dtype=torch.int32, device=dev)

    def leaf(*shape):
        return torch.randn(shape, generator=g).to(dtype).to(dev).requires_grad_()

    x, mod, w = leaf(n, c), leaf(2, 6, c), leaf(3 * c, c)
    dr, dh = leaf(n, c).detach(), leaf(n, c).detach()

    def block(x, mod, w):
        qkv = torch.nn.functional.linear(pkg.modulated_norm(x, cu, mod[:, 1], mod[:, 0]), w / c ** 0.5).view(n, 3, h, d)
        a = pkg.sparse_window_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], 20, cu, sinks=2)
        return pkg.gated_residual_norm(x, a.flatten(1), cu, mod[:, 2], scale=mod[:, 4], shift=mod[:, 3])

    leaves = [x, mod, w]
    want = torch.autograd.grad(block(*leaves), leaves, [dr, dh])
    got = torch.autograd.grad(checkpoint(block, *leaves, use_reentrant=False), leaves, [dr, dh])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
