"""The checks on whole numbers (norm_exact.py) accept layer norm in 64 bits rounded once, and reject what a kernel that loses
something would return: at every size of the GPU tests that is quickly computed here."""
import pytest
import torch

from norm_exact import EPS, check_backward, check_forward, gradients_of, rows_of
from test_layernorm_gpu import MAPS, ROWS

SHAPES = [s for s in [(r, n, 1) for r, n in ROWS] + MAPS if s[0] * s[1] * s[2] <= 4_000_000]


def forward(x, eps, lost=0, ddof=0):
    """`lost`: the last elements of a row that the sum of squares leaves out"""
    n = x.shape[1]
    part = x.double()[:, :n - lost]
    mean = part.sum(1) / n
    r = (part.square().sum(1) / (n - ddof) + eps).rsqrt()
    y = (x.double() - mean.unsqueeze(1)) * r.unsqueeze(1)
    return y.to(x.dtype), mean.float(), r.float()


def backward(dy, x, mean, rstd, lost=0, block=None, zero=()):
    """`lost`: the last elements that a row's sums leave out; `block`: rows that dweight and dbias leave out; `zero`: gradients
    that nobody has written"""
    n = x.shape[1]
    g, h = dy.double(), x.double()
    gh = g * h
    c1, c2 = g[:, :n - lost].sum(1, keepdim=True) / n, gh[:, :n - lost].sum(1, keepdim=True) / n
    rows = [t.movedim(1, -1).reshape(-1, n) for t in (gh, g)]
    dw, db = (t.sum(0) - (t[block].sum(0) if block else 0) for t in rows)
    out = {'dx': (g - c1 - h * c2).to(x.dtype), 'dw': dw.float(), 'db': db.float()}
    return [torch.zeros_like(v) if k in zero else v for k, v in out.items()]


def refused(what, call):
    with pytest.raises(AssertionError, match=what):
        call()


@pytest.mark.parametrize('kind', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_what_the_checks_tell_apart(shape, kind):
    x = rows_of(shape, kind, 'cpu', 1)
    n, per = shape[1], shape[0] * shape[2]
    assert not x.double().sum(1).any()
    check_forward(x, forward)
    for name, dy in gradients_of(x, 2):
        check_backward(x, dy, backward)
        if name == 'every':
            refused('dbias', lambda: check_backward(x, dy, lambda *a: backward(*a, zero=('db',))))
            for block in (slice(per - 1, per), slice(0, max(1, per // 256)), slice(per // 2, per // 2 + max(1, per // 64))):
                refused('dweight|dbias', lambda: check_backward(x, dy, lambda *a: backward(*a, block=block)))
            if n > 1 and per > 2:
                refused('dweight', lambda: check_backward(x, dy, lambda *a: backward(*a, zero=('dw',))))
        if n > 3:
            refused('dx', lambda: check_backward(x, dy, lambda *a: backward(*a, zero=('dx',))))
            if name == f'element {n - 1}':
                for lost in (1, 4):
                    refused('dx', lambda: check_backward(x, dy, lambda *a: backward(*a, lost=min(lost, n - 1))))
    if n > 3:
        for lost in (1, 4):
            refused('mean|scale', lambda: check_forward(x, lambda x, eps: forward(x, eps, min(lost, n - 1))))
        refused('scale', lambda: check_forward(x, lambda x, eps: forward(x, eps, ddof=1)))

        def only_the_scale(x, eps):                          # (as if the sum of squares alone had lost the last element)
            return forward(x, eps)[0], torch.zeros(per), forward(x, eps, 1)[2]
        refused('scale', lambda: check_forward(x, only_the_scale))
