"""rtg.ops.layer_norm (rtg_layernorm.hip) against layer norm in 64 bits: every kind of row and map the kernels split
differently, types, strides, alignments, masked-out gradients, values far from zero and not finite, offsets past 32 bits,
streams and captured graphs.  GPU only."""
import pytest
import torch
import torch.nn.functional as F

from norm_reference import Reference, inside

pytestmark = pytest.mark.gpu
DEV = 'cuda'
KINDS = [torch.float32, torch.bfloat16]
# (rows, n): single elements, ends inside a vector / a wave / a block, the longest that registers hold and longer ones
ROWS = [(1, 1), (3, 1), (5, 2), (1, 8), (7, 63), (64, 64), (33, 65), (9, 128), (6, 250), (129, 257), (2, 1000), (4, 1024), (5, 2047),
        (3, 2048), (3, 4096), (3, 4097), (2, 8192), (1, 16384), (2, 16385), (2, 20001), (1, 40000), (1, 70001), (5000, 48), (1500, 512),
        (700, 1111),
        # rows of less than a vector; several rows a block, whatever its tile
        (100_003, 3), (4099, 7), (70_000, 24), (2500, 1500), (600, 4096), (530, 9000), (300, 16384), (1100, 12_289), (70, 33_000)]
# (clips, channels, positions)
MAPS = [(2, 1, 3), (2, 3, 5), (1, 16, 4), (2, 32, 64), (3, 33, 67), (2, 128, 32), (1, 512, 10), (2, 64, 1025), (1, 1024, 33), (1, 1025, 7),
        (1, 2500, 70), (2, 2, 4096), (4, 7, 1), (1, 40, 2048), (16, 8, 300), (2, 256, 515), (40, 20, 2), (1, 600, 129),
        # clips of less than a vector of positions
        (3, 40, 2), (2, 33, 3), (5, 128, 7), (300, 500, 5), (2, 1000, 6), (50, 1024, 4), (1, 2000, 3),
        # no more than two vectors of positions, each cut of the channels
        (9, 100, 8), (7, 250, 11), (5, 500, 16), (3, 1024, 9),
        # every tile for maps that fill the chip, several tiles a block
        (70, 5, 9001), (40, 13, 8200), (33, 30, 8001), (32, 61, 4101), (17, 100, 8003), (9, 200, 8003), (5, 400, 7001), (3, 1000, 5003),
        (3, 1100, 500), (2, 2048, 11), (4, 2049, 130)]


def make(shape, kind, seed, level=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.rand(shape[:1] + (1,) * (len(shape) - 1), generator=gen).mul(2).add(0.1) + level
    return x.to(DEV).to(kind)


def params(n, kind, seed):
    gen = torch.Generator().manual_seed(seed)
    return ((1 + 0.3 * torch.randn(n, generator=gen)).to(DEV).to(kind), (0.3 * torch.randn(n, generator=gen)).to(DEV).to(kind))


def check(x, w, b, dy, dim, eps=1e-5, layout=None):
    """forward and the three gradients of layer_norm(x) over `dim` against the reference; x may be any view"""
    from rtg import ops
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps=eps, dim=dim)
    assert y.shape == x.shape and y.dtype == x.dtype
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    d = dim % x.dim()

    def three(t):
        t = t.detach()
        return t.reshape(t.shape[:d].numel(), t.shape[d], t.shape[d + 1:].numel())
    kind = next((t.dtype for t in (w, b) if t is not None), torch.float32)
    ref = Reference(three(x), w, b, eps).backward(three(dy), kind)
    inside(three(y), ref.y, ref.y_off, 'y')
    got = dict(zip([k for k, t in zip('xwb', leaves) if t is not None], got))
    assert got['x'].shape == x.shape and got['x'].dtype == x.dtype
    inside(three(got['x']), ref.dx, ref.dx_off, 'dx')
    if w is not None:
        assert got['w'].dtype == w.dtype
        inside(got['w'], ref.dw, ref.dw_off, 'dweight')
    if b is not None:
        inside(got['b'], ref.db, ref.db_off, 'dbias')
    with torch.no_grad():                                   # without statistics to keep: the same bits
        assert torch.equal(ops.layer_norm(x, w, b, eps=eps, dim=dim), y)
    return y, got


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('rows,n', ROWS)
def test_rows(rows, n, kind):
    w, b = params(n, kind if rows % 2 else torch.float32, 3)
    check(make((rows, n), kind, rows + n), w, b, make((rows, n), kind, n, 0.0), -1)


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('clips,n,t', MAPS)
def test_maps(clips, n, t, kind):
    w, b = params(n, kind if clips % 2 else torch.float32, 4)
    check(make((clips, n, t), kind, n + t), w, b, make((clips, n, t), kind, t, 0.0), 1)


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('shape,dim', [((6, 300), 1), ((3, 48, 70), 1)])
@pytest.mark.parametrize('has_w,has_b', [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(shape, dim, has_w, has_b, kind):
    w, b = params(shape[1], kind, 5)
    check(make(shape, kind, 1), w if has_w else None, b if has_b else None, make(shape, kind, 2, 0.0), dim)


@pytest.mark.parametrize('shape,dim', [((4, 5, 64), -1), ((2, 3, 4, 96), 3), ((2, 24, 6, 50), 1), ((5, 40, 3), 0), ((7,), 0), ((3, 40, 1), 1)])
def test_any_axis_of_any_shape(shape, dim):
    w, b = params(shape[dim], torch.float32, 6)
    check(make(shape, torch.float32, 3), w, b, make(shape, torch.float32, 4, 0.0), dim)


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('view', ['row slice', 'odd rows', 'last rows', 'time crop', 'channel slice', 'channels last', 'permuted rows',
                                  'expanded rows', 'every second'])
def test_strided_inputs(view, kind):
    base = make((12, 40, 90), kind, 8)
    x, dim = {'row slice': (base[:, :, 3:67], -1), 'odd rows': (base.reshape(-1)[1:1 + 33 * 77].view(33, 77), -1),
              'last rows': (base[:, -1], -1), 'time crop': (base[:, :, 5:44], 1), 'channel slice': (base[:, 7:30], 1),
              'channels last': (base.transpose(1, 2), 1), 'permuted rows': (base.permute(1, 0, 2), -1),
              'expanded rows': (base[:1, :1].expand(6, 40, 90), -1), 'every second': (base[:, :, ::2], 1)}[view]
    w, b = params(x.shape[dim], kind, 9)
    y, got = check(x, w, b, make(tuple(x.shape), kind, 10, 0.0), dim)
    if view == 'channels last':                              # read and written as rows: no copy into another order
        assert y.transpose(1, 2).is_contiguous()


def test_gradient_of_a_broadcast_and_of_a_transposed_output():
    """dy as autograd makes it: expanded (a sum) and transposed"""
    from rtg import ops
    x = make((3, 20, 50), torch.float32, 1).requires_grad_(True)
    w, b = (p.requires_grad_(True) for p in params(20, torch.float32, 2))
    y = ops.layer_norm(x, w, b, dim=1)
    y.sum().backward()
    ref = Reference(x.detach(), w.detach(), b.detach(), 1e-5).backward(torch.ones(3, 20, 50, device=DEV), torch.float32)
    for got, want, off in ((x.grad, ref.dx, ref.dx_off), (w.grad, ref.dw, ref.dw_off), (b.grad, ref.db, ref.db_off)):
        inside(got, want, off, 'broadcast')
    dy = make((3, 50, 20), torch.float32, 3, 0.0)
    got, = torch.autograd.grad((ops.layer_norm(x, w, b, dim=1).transpose(1, 2) * dy).sum(), x)
    ref.backward(dy.transpose(1, 2), torch.float32)
    inside(got, ref.dx, ref.dx_off, 'transposed')


@pytest.mark.parametrize('shape,dim', [((5, 96), -1), ((2, 24, 10), 1)])
def test_gradient_against_differences(shape, dim):
    """the gradient of sum(y * dy) against central differences of the 64-bit definition"""
    from rtg import ops
    x, dy = make(shape, torch.float32, 1), make(shape, torch.float32, 2, 0.0)
    w, b = params(shape[dim], torch.float32, 3)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves, dim=dim), leaves, dy)

    three = (lambda t: t.reshape(-1, t.shape[-1], 1)) if dim == -1 else (lambda t: t)
    ref = Reference(three(x), w, b, 1e-5).backward(three(dy), torch.float32)

    def value(*v):
        v = [t.double() for t in v]
        return (F.layer_norm(v[0].movedim(dim, -1), (shape[dim],), v[1], v[2], 1e-5).movedim(-1, dim) * dy.double()).sum()
    for i, g in enumerate(grads):
        way = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV).double()
        h = 1e-5
        up, down = ([t.detach().double() + (s * h * way if k == i else 0) for k, t in enumerate(leaves)] for s in (1, -1))
        want = (value(*up) - value(*down)) / (2 * h)
        # the gradient within its bound; the differences within h^2 / 6 of a third derivative (r^3 |dy| n < 1e5 at the smallest
        # spread of 0.1) and 1e-16 |value| / h of rounding: 1e-5 covers both
        off = [ref.dx_off, ref.dw_off, ref.db_off][i].reshape(g.shape)
        assert abs((g.double() * way).sum() - want) <= (off * way.abs()).sum() + 1e-5


@pytest.mark.parametrize('shape,dim', [((40, 1000), -1), ((5, 4000), -1), ((6, 33000), -1), ((2, 100, 300), 1), ((1, 3000, 40), 1)])
def test_levels_far_from_zero_keep_their_digits(shape, dim):
    """values around a level of 2^22 / n in steps of a quarter: every sum of them is a multiple of 1/4 below 2^22, exact in a
    float, so the mean is off by its own rounding alone — and a variance taken as E x^2 - mean^2 would have lost its digits"""
    from rtg import ops
    n = shape[dim]
    level = int(4 * 2 ** 22 / n) / 4 - 8
    x = (level + torch.randint(-8, 9, shape, generator=torch.Generator().manual_seed(1)) / 4).to(DEV)
    w, b = params(n, torch.float32, 2)
    y = ops.layer_norm(x, w, b, dim=dim)
    three = (lambda t: t.reshape(-1, n, 1)) if dim == -1 else (lambda t: t)
    ref = Reference(three(x), w, b, 1e-5, mean_chain=1)
    inside(three(y), ref.y, ref.y_off, 'y')


@pytest.mark.parametrize('shape,dim', [((6, 200), -1), ((2, 17000), -1), ((2, 60, 40), 1), ((1, 1100, 12), 1)])
def test_values_that_are_not_finite_stay_in_their_row(shape, dim):
    from rtg import ops
    x = make(shape, torch.float32, 1)
    rows = x.movedim(dim, -1).reshape(-1, shape[dim])
    clean = ops.layer_norm(x, dim=dim).movedim(dim, -1).reshape(rows.shape)
    y = x.clone().movedim(dim, -1)
    y[(0,) * (y.dim() - 1)][3] = float('inf')
    y[(0,) * (y.dim() - 2) + (1,)][5] = float('nan')
    bad = y.movedim(-1, dim).contiguous()
    got = ops.layer_norm(bad, dim=dim).movedim(dim, -1).reshape(rows.shape)
    assert torch.isnan(got[0]).all() and torch.isnan(got[1]).all()
    assert torch.equal(got[2:], clean[2:])


def test_constant_rows_and_zero_gradients():
    from rtg import ops
    for shape, dim in (((4, 300), -1), ((2, 30, 20), 1)):
        x = torch.full(shape, 2.5, device=DEV, requires_grad=True)
        w, b = (p.requires_grad_(True) for p in params(shape[dim], torch.float32, 1))
        y = ops.layer_norm(x, w, b, dim=dim)
        along = (1, -1) + (1,) * (len(shape) - 2)
        assert torch.equal(y, b.view(along).expand(shape))                  # xhat is exactly 0
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(shape, device=DEV))
        assert not dx.any() and not dw.any() and not db.any()


@pytest.mark.parametrize('shape,dim', [((0, 16), -1), ((0, 16, 4), 1), ((3, 16, 0), 1)])
def test_no_rows(shape, dim):
    from rtg import ops
    x = torch.empty(shape, device=DEV, requires_grad=True)
    w, b = (p.requires_grad_(True) for p in params(16, torch.float32, 1))
    y = ops.layer_norm(x, w, b, dim=dim)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(shape, device=DEV))
    assert y.shape == dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize('wanted', [(True, False, False), (False, True, True), (False, True, False), (False, False, True), (True, True, False)])
@pytest.mark.parametrize('shape,dim', [((50, 700), -1), ((3, 17000), -1), ((2, 48, 130), 1), ((1, 1100, 9), 1)])
def test_only_the_gradients_asked_for(shape, dim, wanted):
    from rtg import ops
    x, dy = make(shape, torch.float32, 1), make(shape, torch.float32, 2, 0.0)
    w, b = params(shape[dim], torch.float32, 3)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, dim=dim, keep=True)
    every = ops.layer_norm_backward(dy, x, mean, rstd, w, dim=dim)
    some = ops.layer_norm_backward(dy, x, mean, rstd, w, dim=dim, needs=wanted)
    for a, s, want in zip(every, some, wanted):
        assert torch.equal(a, s) if want else s is None


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('shape,dim', [((3000, 768), -1), ((5, 17000), -1), ((7, 65, 1111), 1), ((2, 1100, 40), 1)])
def test_the_same_call_gives_the_same_bits(shape, dim, kind):
    x, dy = make(shape, kind, 1), make(shape, kind, 2, 0.0)
    w, b = params(shape[dim], torch.float32, 3)
    y, first = check(x, w, b, dy, dim)
    z, again = check(x, w, b, dy, dim)
    assert torch.equal(y, z) and all(torch.equal(first[k], again[k]) for k in first)


def test_memory_around_the_outputs_is_left_alone():
    """outputs cut out of larger buffers, written through the C entry points: nothing in front of or behind them changes"""
    import ctypes as C
    from rtg import lib as L
    from rtg.lib import lib, check as ok, current_stream_ptr
    for kind in KINDS:
        for outer, n, inner in ((5, 77, 1), (3, 4100, 1), (2, 17001, 1), (2, 19, 37), (1, 1030, 5)):
            x, dy = make((outer, n, inner), kind, 1), make((outer, n, inner), kind, 2, 0.0)
            w, b = params(n, torch.float32, 3)
            e, r = outer * n * inner, outer * inner
            d = L.LayerNormDesc(outer, n, inner, n * inner, inner, int(kind == torch.bfloat16), 0, 1e-5)
            big = {k: torch.full((m + 66,), 7.0, device=DEV, dtype=t) for k, m, t in (
                ('y', e, kind), ('dx', e, kind), ('mean', r, torch.float32), ('rstd', r, torch.float32), ('dw', n, torch.float32),
                ('db', n, torch.float32), ('ws', lib.rtg_layernorm_ws(C.byref(d)), torch.float32))}
            at = {k: C.c_void_p(t.data_ptr() + 33 * t.element_size()) for k, t in big.items()}
            p = lambda t: C.c_void_p(t.data_ptr())                                                    # noqa: E731
            ok(lib.rtg_layernorm_forward(C.byref(d), p(x), p(w), p(b), at['y'], at['mean'], at['rstd'], current_stream_ptr()))
            ok(lib.rtg_layernorm_backward(C.byref(d), p(dy), p(x), at['mean'], at['rstd'], p(w), at['dx'], at['dw'], at['db'], at['ws'],
                                          current_stream_ptr()))
            for k, t in big.items():
                assert (t[:33] == 7).all() and (t[-33:] == 7).all(), (k, kind, outer, n, inner)
            ref = Reference(x, w, b, 1e-5).backward(dy, torch.float32)
            inside(big['y'][33:-33], ref.y, ref.y_off, 'y')
            inside(big['dx'][33:-33], ref.dx, ref.dx_off, 'dx')
            inside(big['dw'][33:-33], ref.dw, ref.dw_off, 'dweight')


def test_offsets_past_32_bits():
    """rows of a view that lie more than 2^31 elements apart, and a map whose clips do"""
    step = (1 << 30) + 1025
    base = torch.empty(2 * step + 4096, device=DEV, dtype=torch.bfloat16)
    for size, stride, dim in (((3, 640), (step, 1), -1), ((3, 24, 20), (step, 100, 1), 1)):
        x = base.as_strided(size, stride)
        x.copy_(make(size, torch.bfloat16, 5))
        w, b = params(size[1], torch.float32, 6)
        check(x, w, b, make(size, torch.bfloat16, 7, 0.0), dim)


def test_channels_far_apart():
    """more than 2^24 elements between the channels of a map: the offsets inside a tile would pass 32 bits"""
    for t in (70, 3):
        size, stride = (2, 20, t), (t + 1, (1 << 24) + 3, 1)
        x = torch.empty(20 * stride[1] + 4096, device=DEV, dtype=torch.bfloat16).as_strided(size, stride)
        x.copy_(make(size, torch.bfloat16, 5))
        check(x, *params(20, torch.float32, 6), make(size, torch.bfloat16, 7, 0.0), 1)


@pytest.mark.parametrize('shape,dim,kind', [((16_500, 4099), -1, torch.float32), ((270_001, 250), -1, torch.float32), ((530_001, 260), -1, torch.bfloat16),
                                            ((4200, 16_390), -1, torch.float32), ((32, 129, 16_390), 1, torch.float32), ((16, 512, 8200), 1, torch.float32),
                                            ((33, 100, 41_000), 1, torch.bfloat16)])
def test_activations_that_no_cache_holds(shape, dim, kind):
    """256 MB and more, which are read past the caches"""
    gen = torch.Generator(device=DEV).manual_seed(8)
    x, dy = (torch.randn(shape, generator=gen, device=DEV).add_(level).to(kind) for level in (1.0, 0.0))
    assert x.numel() * x.element_size() >= 256 << 20
    check(x, *params(shape[dim], torch.float32, 9), dy, dim)


def test_another_stream():
    from rtg import ops
    x, w, b = make((64, 1000), torch.float32, 1), *params(1000, torch.float32, 2)
    dy = make((64, 1000), torch.float32, 3, 0.0)
    want = ops.layer_norm_forward(x, w, b, keep=True)
    grads = ops.layer_norm_backward(dy, x, want[1], want[2], w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.layer_norm_forward(x, w, b, keep=True)
        got_grads = ops.layer_norm_backward(dy, x, got[1], got[2], w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want + grads, got + got_grads))


@pytest.mark.parametrize('shape,dim', [((300, 1024), -1), ((3, 64, 200), 1)])
def test_captured_into_graphs(shape, dim):
    """two graphs of forward and backward, replayed in turn with new inputs and eager calls between"""
    from rtg import ops
    w, b = params(shape[dim], torch.float32, 1)
    ins = [(make(shape, torch.float32, s), make(shape, torch.float32, s + 1, 0.0)) for s in (10, 20)]

    def both(x, dy):
        y, mean, rstd = ops.layer_norm_forward(x, w, b, dim=dim, keep=True)
        return (y, *ops.layer_norm_backward(dy, x, mean, rstd, w, dim=dim))
    both(*ins[0])
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


def test_refusals():
    from rtg import ops
    from rtg.lib import RtgError
    x, (w, b) = make((4, 16), torch.float32, 1), params(16, torch.float32, 2)
    for args in ((x.half(), w, b), (x.double(), w, b), (x, w[:8], b), (x, w, b.view(4, 4)), (x, w, b.bfloat16()), (x, w.half(), None),
                 (x, w.cpu(), b), (x.cpu(), w, b)):
        with pytest.raises(RtgError):
            ops.layer_norm(*args)
    for kw in ({'dim': 2}, {'dim': -3}, {'eps': -1.0}, {'eps': float('nan')}):
        with pytest.raises(RtgError):
            ops.layer_norm(x, w, b, **kw)
    with pytest.raises(RtgError):
        ops.layer_norm(torch.empty(4, 0, device=DEV))
    y, mean, rstd = ops.layer_norm_forward(x, w, b, keep=True)
    for args in ((y.bfloat16(), x, mean, rstd, w), (y[:2], x, mean, rstd, w), (y, x, mean[:2], rstd, w), (y, x, mean.double(), rstd, w)):
        with pytest.raises(RtgError):
            ops.layer_norm_backward(*args)
    with pytest.raises(RuntimeError):                          # not differentiable twice: refused, not wrong
        xl = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(ops.layer_norm(xl, w, b).square().sum(), xl, create_graph=True)
        g.sum().backward()


def test_module_is_torch_layer_norm():
    from models.layers import LayerNorm
    from rtg.lib import RtgError
    m, t = LayerNorm(48).to(DEV), torch.nn.LayerNorm(48).to(DEV)
    assert {k: v.shape for k, v in m.state_dict().items()} == {k: v.shape for k, v in t.state_dict().items()}
    t.load_state_dict(m.state_dict())
    x = make((3, 48, 60), torch.float32, 1)
    want = t.double()(x.double().transpose(1, 2)).transpose(1, 2)
    assert (m(x).double() - want).abs().max() < 1e-5
    assert LayerNorm(48, affine=False).to(DEV)(x).shape == x.shape and LayerNorm(48, bias=False).bias is None
    with pytest.raises(RtgError):
        m(x.transpose(1, 2))
