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


@pytest.mark.parametrize('clips,n,t', [((1 << 26) + 5, 2, 2), ((1 << 24) + 3, 33, 2)])
def test_more_tiles_than_a_launch_holds(clips, n, t):
    """maps of many short clips: a block of 256 threads for every one or four of them would be 2^32 threads and more"""
    from rtg import ops
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, dy = (torch.empty(clips, n, t, device=DEV, dtype=torch.bfloat16).normal_(m, 1.0, generator=gen) for m in (1.0, 0.0))
    w, b = params(n, torch.float32, 2)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, dim=1, keep=True)
    dx, _, _ = ops.layer_norm_backward(dy, x, mean, rstd, w, dim=1, needs=(True, False, False))
    for at in range(0, clips, 1 << 21):
        cut = slice(at, min(at + (1 << 21), clips))
        ref = Reference(x[cut], w, b, 1e-5).backward(dy[cut], torch.float32)
        inside(y[cut], ref.y, ref.y_off, 'y')
        inside(dx[cut], ref.dx, ref.dx_off, 'dx')


@pytest.mark.parametrize('n', [(1 << 27) + 64, (1 << 30) + 256])
def test_rows_longer_than_a_launch_has_threads(n):
    """One row of +1, -1, ... with the gradient +2, +2, -2, -2, ...: sums of whole numbers that a float holds (n is a multiple of
    its step there), so the mean and both sums of dx are 0, the variance is 1 up to the rounding of 1 / n, and
    y = x, dx = dy, dweight = dy x up to the roundings of that and of the scale (u each, 8 in all)."""
    from norm_reference import U
    from rtg import ops
    x = torch.tensor([1.0, -1.0], device=DEV).repeat(n // 2).view(1, n)
    dy = torch.tensor([2.0, 2.0, -2.0, -2.0], device=DEV).repeat(n // 4).view(1, n)
    y, mean, rstd = ops.layer_norm_forward(x, eps=0.0, keep=True)
    assert mean.item() == 0.0 and abs(rstd.item() - 1.0) <= 4 * U
    assert ((y - x).abs() <= 8 * U).all()
    del y
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd)
    assert torch.equal(db, dy[0])
    assert ((dx - dy).abs() <= 16 * U).all()
    assert (dw.sub_(dy[0] * x[0]).abs_() <= 16 * U).all()
    del dx, dw, db
    empty = x[:0]
    _, dw, db = ops.layer_norm_backward(empty, empty, mean[:0], rstd[:0])
    assert dw.shape == db.shape == (n,) and not dw.any() and not db.any()


@pytest.mark.parametrize('sizes', [[2], [5, 3000], [50] * 40, [5_000_003]])
@pytest.mark.parametrize('scale', [1.0, 1e-3])
def test_an_update_whose_norm_no_float_holds_is_left_out(sizes, scale):
    """two finite gradients of 3e38: their norm is 4.2e38, and inf as a float.  What the caller sees as not finite leaves the
    buffers alone; scaled so that a float holds the norm, it does not"""
    from test_gradnorm_gpu import state, update
    s = state(sizes, 1)
    s['g'][0][:2] = 3e38
    before = {k: [t.clone() for t in s[k]] for k in s}
    norm = update(s, 0.05, grad_scale=scale)
    assert torch.isinf(norm) == (scale == 1.0)
    for k in 'pmvt':
        assert all(torch.equal(a, b) for a, b in zip(s[k], before[k])) == (scale == 1.0), k


def test_clipping_by_a_norm_no_float_holds():
    """the returned norm is inf, the factor that of the norm itself"""
    from rtg import ops
    t = torch.full((4,), 3e38, device=DEV)                      # 6e38
    assert torch.isinf(ops.clip_grads_([t], 60.0)) and torch.isinf(ops.total_norm([torch.full((4,), 3e38, device=DEV)]))
    assert ((t - 30.0).abs() <= 30.0 * 2.0 ** -22).all()        # (3e38 as a float, the factor, the product: half a step each)


@pytest.mark.parametrize('shape,dim', [((300, 1024), -1), ((3, 64, 200), 1)])
def test_training_passes_captured_into_graphs(shape, dim):
    """forward and backward through autograd in two graphs, replayed in turn with new inputs and eager passes between"""
    from rtg import ops
    w, b = params(shape[dim], torch.float32, 1)

    def both(x, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.layer_norm(*leaves, dim=dim)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    ins = [(make(shape, torch.float32, s), make(shape, torch.float32, s + 1, 0.0)) for s in (10, 20)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(*ins[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for x, dy in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both(x, dy)
        graphs.append((g, out))
    for r in range(3):
        for k, ((g, out), (x, dy)) in enumerate(zip(graphs, ins)):
            x.copy_(make(shape, torch.float32, 100 * r + k))
            dy.copy_(make(shape, torch.float32, 100 * r + k + 50, 0.0))
            g.replay()
            want = both(x, dy)
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, want)), (r, k)


def test_training_passes_of_two_threads_and_streams():
    """two threads, each with a stream and layouts of its own, while nobody waits for the other"""
    import threading
    from rtg import ops
    work = []
    for k, (shape, dim, cut) in enumerate((((6, 48, 300), 1, lambda t: t[:, :, 5:270]), ((500, 1100), -1, lambda t: t[:, 3:1003]))):
        x = cut(make(shape, torch.float32, k))
        work.append((x, *params(x.shape[dim], torch.float32, k), make(tuple(x.shape), torch.float32, k + 5, 0.0), dim))

    def one(x, w, b, dy, dim):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.layer_norm(*leaves, dim=dim)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    want = [one(*w) for w in work]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def run(k):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    got[k].append(one(*work[k]))
            st.synchronize()
        except Exception as e:                                  # (shown below: a thread's exception is not the test's)
            failed.append(e)
    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed
    assert all(len(g) == 20 and all(torch.equal(a, c) for out in g for a, c in zip(out, want[k])) for k, g in enumerate(got))


def test_a_map_of_more_positions_than_a_tile_counts():
    """2^24 positions and more: the kernels for any size"""
    from rtg import ops
    shape = (1, 5, (1 << 24) + 70)
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, dy = (torch.empty(shape, device=DEV, dtype=torch.bfloat16).normal_(m, 1.0, generator=gen) for m in (1.0, 0.0))
    w, b = params(5, torch.float32, 2)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, dim=1, keep=True)
    dx, _, _ = ops.layer_norm_backward(dy, x, mean, rstd, w, dim=1)
    ref = Reference(x, w, b, 1e-5).backward(dy, torch.float32)
    inside(y, ref.y, ref.y_off, 'y')
    inside(dx, ref.dx, ref.dx_off, 'dx')
    ones, zeros = torch.ones(shape[2], device=DEV), torch.zeros(shape[2], device=DEV)      # (sums of whole numbers: exact)
    x, dy = (torch.randint(-1, 2, shape, generator=gen, device=DEV).bfloat16() for _ in range(2))
    _, dw, db = ops.layer_norm_backward(dy, x, zeros, ones, w, dim=1)
    assert torch.equal(dw.double(), (dy.double() * x.double()).sum((0, 2))) and torch.equal(db.double(), dy.double().sum((0, 2)))
