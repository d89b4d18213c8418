"""Calls of layer norm and of the gradient operators that lie beside the ordinary ones, on the GPU."""
import pytest
import torch

from norm_reference import Reference, inside
from test_layernorm_gpu import DEV, KINDS, make, params

pytestmark = pytest.mark.gpu


def three(t, dim):
    return t.detach().reshape(t.shape[:dim].numel(), t.shape[dim], t.shape[dim + 1:].numel())


SAVED = {'time crop': (lambda t: t[:, :, 5:44], 1), 'channel slice': (lambda t: t[:, 7:30], 1), 'row slice': (lambda t: t[:, :, 3:67], 2),
         'last rows': (lambda t: t[:, -1], 1), 'channels last': (lambda t: t.transpose(1, 2), 1), 'whole': (lambda t: t, 1)}


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('view', list(SAVED))
@pytest.mark.parametrize('how', ['on the host', 'dense', 'recomputed'])
def test_saved_tensors_that_leave_and_come_back(view, how, kind):
    """activations that a hook keeps elsewhere (their gaps are gone when they return): the gradients are those of the kept ones,
    and the definition's"""
    from rtg import ops
    cut, dim = SAVED[view]
    base = make((6, 48, 120), kind, 1)
    x = cut(base).detach().requires_grad_(True)
    w, b = (p.requires_grad_(True) for p in params(x.shape[dim], torch.float32, 2))
    dy = make(tuple(x.shape), kind, 3, 0.0)
    want = torch.autograd.grad(ops.layer_norm(x, w, b, dim=dim), (x, w, b), dy)
    if how == 'recomputed':
        y = torch.utils.checkpoint.checkpoint(lambda *a: ops.layer_norm(*a, dim=dim), x, w, b, use_reentrant=False)
    else:
        hooks = (torch.autograd.graph.save_on_cpu() if how == 'on the host' else
                 torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t))
        with hooks:
            y = ops.layer_norm(x, w, b, dim=dim)
    got = torch.autograd.grad(y, (x, w, b), dy)
    ref = Reference(three(x, dim), w.detach(), b.detach(), 1e-5).backward(three(dy, dim), torch.float32)
    inside(three(got[0], dim), ref.dx, ref.dx_off, 'dx')
    inside(got[1], ref.dw, ref.dw_off, 'dweight')
    inside(got[2], ref.db, ref.db_off, 'dbias')
    assert torch.equal(got[0], want[0])                         # (an element's gradient does not go by the layout it is read from)


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    from rtg import ops
    from rtg.lib import RtgError
    x, (w, b) = make((4, 48), torch.float32, 1), params(48, torch.float32, 2)
    want = ops.layer_norm(x, w, b)
    with fw.dual_level():
        assert torch.equal(ops.layer_norm(x, w, b), want)
        for duals in ((fw.make_dual(x, x), w, b), (x, fw.make_dual(w, w), b), (x, w, fw.make_dual(b, b))):
            with pytest.raises(RtgError, match='tangent'):
                ops.layer_norm(*duals)
