"""Layer norm of whole numbers: sums that a float holds exactly, whatever the order they are taken in, so that a result is off by
its last roundings alone and a lost element, row or partial sum shows at every size (tests/test_norm_exact_gpu.py).

Rows x of whole numbers that add up to 0: the mean is exactly 0 and the sum of squares is exact (below 2^24).
Backward passes are given mean 0 and scale 1: xhat = x, and every sum over rows (dweight, dbias) or along one is one of whole numbers."""
import torch

from norm_reference import U, half_step

# (outer, n, inner): beside the sizes of tests/test_layernorm_gpu.py, those that no cache holds
LARGE = [(16_500, 4099, 1), (270_001, 250, 1), (530_001, 260, 1), (4200, 16_390, 1), (32, 129, 16_390), (16, 512, 8200), (33, 100, 41_000)]
EPS = 0.5


def rows_of(shape, kind, device, seed):
    """whole numbers of 1 .. 3 and their negatives (an odd row has 1, 1, -2 as well) in one random order along the axis; of one
    element 0"""
    outer, n, inner = shape
    gen = torch.Generator(device=device).manual_seed(seed)
    pairs = (n - 3) // 2 if n % 2 and n > 1 else n // 2
    v = torch.randint(1, 4, (outer, pairs, inner), generator=gen, device=device).to(kind)
    parts = [v, -v]
    if n % 2:
        rest = [1, 1, -2] if n > 1 else [0]
        parts.append(torch.tensor(rest, device=device).to(kind).view(1, -1, 1).expand(outer, -1, inner))
    return torch.cat(parts, 1).index_select(1, torch.randperm(n, generator=gen, device=device))


def rejects(ok, what):
    assert ok, what


def check_forward(x, forward):
    """forward(x, eps) -> y, mean, rstd (float32, one per row or position).  The scale: n and 1 / n are rounded, the product, the
    sum with eps: 4 u of the variance, half of that of the scale, and 2 u of the root itself."""
    y, mean, rstd = forward(x, EPS)
    n = x.shape[1]
    r = (x.double().square().sum(1) / n + EPS).rsqrt()
    rejects(bool((mean.reshape(-1) == 0).all()), 'mean')
    rejects(bool(((rstd.reshape(r.shape).double() - r).abs() <= 4 * U * r).all()), 'scale')
    want = x.double() * r.unsqueeze(1)
    rejects(bool(((y.double() - want).abs() <= (6 * U + half_step(x.dtype) * (1 + 6 * U)) * want.abs()).all()), 'y')


def check_backward(x, dy, backward):
    """backward(dy, x, mean, rstd) -> dx, dweight, dbias (float32).  dweight and dbias are exact; dx is off by the two roundings
    of each of its means, and four of its own."""
    n = x.shape[1]
    per = x.shape[0] * x.shape[2]
    dx, dw, db = backward(dy, x, torch.zeros(per, device=x.device), torch.ones(per, device=x.device))
    g, h = dy.double(), x.double()
    gh = g * h
    rejects(torch.equal(dw.double(), gh.sum((0, 2))), 'dweight')
    rejects(torch.equal(db.double(), g.sum((0, 2))), 'dbias')
    c1, c2 = g.sum(1, keepdim=True) / n, gh.sum(1, keepdim=True) / n
    want = g - c1 - h * c2
    off = 4 * U * (g.abs() + c1.abs() + (h * c2).abs())
    off = off + half_step(x.dtype) * (want.abs() + off)
    rejects(bool(((dx.double() - want).abs() <= off).all()), 'dx')


def gradients_of(x, seed):
    """[(name, dy)]: 1 .. 3 everywhere, so that every row counts in every sum; and 0 but for one element of each row, the first,
    the middle and the last one, of about n (a power of two): a row's sums are that element"""
    gen = torch.Generator(device=x.device).manual_seed(seed)
    n = x.shape[1]
    yield 'every', torch.randint(1, 4, x.shape, generator=gen, device=x.device).to(x.dtype)
    for at in sorted({0, n // 2, n - 1}):
        dy = torch.zeros_like(x)
        dy[:, at] = 2.0 ** (n - 1).bit_length()
        yield f'element {at}', dy
