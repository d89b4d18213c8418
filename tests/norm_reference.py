"""Layer norm in 64 bits, with the bound of what an evaluation in 32 bits may be off by (tests/test_layernorm_gpu.py).

The bounds are those of the arithmetic, element by element: u = 2^-24 is half a step of a float; a sum of n terms whose
longest chain of additions has k of them is off by at most k u sum|terms|.  No kernel forms a longer chain than a quarter of
the terms behind its last split (a block's four waves, or more lanes, share an axis) and a tree of at most 32 levels."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def chain(n):
    return n / 4 + 32


class Reference:
    """x: [outer, n, inner] on the CPU or the GPU, any type; weight / bias (n,) or None -> y and its bound; after backward(dy)
    dx, dw, db and theirs"""

    def __init__(self, x, weight, bias, eps, mean_chain=None):
        self.kind, n = x.dtype, x.shape[1]
        self.x = x.double()
        self.along = (1, n, 1)
        self.w = torch.ones(n, dtype=torch.float64, device=x.device) if weight is None else weight.double()
        b = torch.zeros(n, dtype=torch.float64, device=x.device) if bias is None else bias.double()
        self.w, b = self.w.view(self.along), b.view(self.along)
        mean = self.x.mean(1, keepdim=True)
        xc = self.x - mean
        var = xc.square().mean(1, keepdim=True)
        self.r = (var + eps).rsqrt()
        self.xhat = xc * self.r
        self.y = self.xhat * self.w + b
        k = chain(n)
        self.k = k
        dm = ((k if mean_chain is None else mean_chain) + 2) * U * self.x.abs().mean(1, keepdim=True)
        dvar = (k + 6) * U * var + 2 * dm * xc.abs().mean(1, keepdim=True) + dm * dm
        self.dr = dvar / (var + eps) + 4 * U                                     # relative, of r (twice the first order)
        self.dxhat = self.r * (dm + U * xc.abs()) + self.xhat.abs() * (self.dr + 3 * U)
        self.y_off = self.w.abs() * self.dxhat + 3 * U * (self.xhat * self.w).abs() + 2 * U * b.abs() + 2 * U * self.y.abs()
        self.y_off = self.y_off + half_step(self.kind) * (self.y.abs() + self.y_off) + 1e-40

    def backward(self, dy, param_kind):
        dy = dy.double()
        g = dy * self.w
        gx = g * self.xhat
        c1, c2 = g.mean(1, keepdim=True), gx.mean(1, keepdim=True)
        core = g - c1 - self.xhat * c2
        self.dx = self.r * core
        dc1 = (self.k + 4) * U * g.abs().mean(1, keepdim=True)
        dc2 = (self.k + 6) * U * gx.abs().mean(1, keepdim=True) + (g.abs() * self.dxhat).mean(1, keepdim=True)
        dcore = 2 * U * g.abs() + dc1 + self.xhat.abs() * dc2 + c2.abs() * self.dxhat + 4 * U * (g.abs() + c1.abs() + (self.xhat * c2).abs())
        self.dx_off = self.r * dcore * (1 + self.dr) + self.dx.abs() * (self.dr + 3 * U)
        self.dx_off = self.dx_off + half_step(self.kind) * (self.dx.abs() + self.dx_off) + 1e-40
        rows = dy.shape[0] * dy.shape[2]
        k, p = chain(rows) + 64, half_step(param_kind)
        self.dw, self.db = (dy * self.xhat).sum((0, 2)), dy.sum((0, 2))
        self.dw_off = (k + 2) * U * (dy * self.xhat).abs().sum((0, 2)) + (dy.abs() * self.dxhat).sum((0, 2))
        self.db_off = k * U * dy.abs().sum((0, 2))
        self.dw_off = self.dw_off + p * (self.dw.abs() + self.dw_off) + 1e-40
        self.db_off = self.db_off + p * (self.db.abs() + self.db_off) + 1e-40
        return self


def inside(got, want, off, what):
    """every element of `got` within `off` of `want` (and not finite where `want` is not)"""
    got = got.double().reshape(want.shape)
    bad = ~((got - want).abs() <= off)
    assert not bad.any(), (f'{what}: {int(bad.sum())} of {bad.numel()} elements outside their bound, worst '
                           f'{((got - want).abs() / off)[bad].max().item():.3g} times it at {bad.nonzero()[0].tolist()}')
