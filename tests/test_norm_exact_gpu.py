"""Layer norm of whole numbers on the GPU (norm_exact.py): every size that the kernels split differently, with nothing lost."""
import pytest
import torch

from norm_exact import LARGE, check_backward, check_forward, gradients_of, rows_of
from test_layernorm_gpu import DEV, KINDS, MAPS, ROWS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('shape', [(r, n, 1) for r, n in ROWS] + MAPS + LARGE, ids=str)
def test_nothing_is_lost(shape, kind):
    from rtg import ops
    x = rows_of(shape, kind, DEV, 1)
    x = x.squeeze(-1) if shape[2] == 1 else x
    dim = -1 if shape[2] == 1 else 1

    def forward(x3, eps):
        y, mean, rstd = ops.layer_norm_forward(x, eps=eps, dim=dim, keep=True)
        return y.view(shape), mean, rstd

    def backward(dy, x3, mean, rstd):
        dx, dw, db = ops.layer_norm_backward(dy.view(x.shape), x, mean, rstd, dim=dim)
        return dx.view(shape), dw, db
    x3 = x.view(shape)
    check_forward(x3, forward)
    for name, dy in gradients_of(x3, 2):
        check_backward(x3, dy, backward)
