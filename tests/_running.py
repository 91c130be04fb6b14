"""Values in fp64 with a bound on what fp32 arithmetic makes of them: every operation adds one rounding
of 2^-23 of its result (twice that of round to nearest, for products and sums taken in another order or
fused) to the bounds that come in with its operands, and a sum of many terms `n` of those of the sum of
the terms' sizes."""
import torch

EPS = 2.0 ** -23


class V:
    def __init__(self, val, err=None):
        self.val = val
        self.err = torch.zeros_like(val) if err is None else err

    def _of(self, o):
        return o if isinstance(o, V) else V(torch.as_tensor(o, dtype=torch.float64))

    def __add__(self, o):
        o = self._of(o)
        v = self.val + o.val
        return V(v, self.err + o.err + EPS * v.abs())

    def __sub__(self, o):
        o = self._of(o)
        v = self.val - o.val
        return V(v, self.err + o.err + EPS * v.abs())

    def __mul__(self, o):
        o = self._of(o)
        v = self.val * o.val
        return V(v, self.err * (o.val.abs() + o.err) + self.val.abs() * o.err + EPS * v.abs())

    def sum(self, dim, n, keepdim=False):
        """The sum over dim, of whose terms each passes through at most n additions."""
        return V(self.val.sum(dim, keepdim=keepdim),
                 self.err.sum(dim, keepdim=keepdim) + n * EPS * self.val.abs().sum(dim, keepdim=keepdim))

    def rsqrt(self):
        """1 / sqrt, of a value that is larger than twice its bound: the derivative at the value less the bound."""
        low = self.val - self.err
        v = self.val.rsqrt()
        return V(v, 0.5 * self.err * low.rsqrt() ** 3 + 2 * EPS * v)

    def rows(self, index):
        return V(self.val[index], self.err[index])

    def rounded(self, dtype):
        """(value, bound) after one rounding to dtype; 2^-25 is half fp16's smallest step."""
        f = torch.finfo(dtype)
        return self.val, self.err * (1 + f.eps) + f.eps / 2 * self.val.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def check(got, want, what):
    val, tol = want
    got = got.detach().double().cpu()
    assert got.shape == val.shape, (what, got.shape, val.shape)
    if not got.numel():
        return
    ratio = ((got - val).abs() / (tol + 1e-30)).max().item()
    print(f"    {what}: worst error {ratio:.3f} of its bound", flush=True)
    assert ratio <= 1.0, (what, ratio)
