"""rtg.ops.total_norm / clip_grads_ / clipped_adamw_ and what train builds on them, against the same in 64 bits: lists of
every cut, types, alignments and sizes, values at the ends of the float range, refusals, streams and captured graphs.
GPU only.

u = 2^-24 (half a step of a float).  The norm is a sum of doubles, rounded once: u.  A clipped gradient: the factor and the
product are rounded, 2 u, and the result once more to its type."""
import math

import pytest
import torch

from norm_reference import U, half_step, inside

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF = torch.float32, torch.bfloat16
# element counts of a list's tensors: one element, none, ends inside a vector, a chunk and a block's round, more tensors than
# one launch takes, one tensor over many chunks, small beside large
LISTS = {'one': [1], 'three': [5, 0, 3], 'vector ends': [3, 4, 5, 7, 8, 9, 15, 16, 17], 'round ends': [1023, 1024, 1025, 4096, 4097],
         'chunk ends': [4095, 4096, 4097, 8191, 8192, 8193], 'many': [(i * 37) % 300 for i in range(700)], 'one large': [3_000_001],
         'mixed': [7, 2_000_000, 1, 33, 65537], 'table': [64] * 160, 'table and one': [65] * 161}


def gradients(sizes, kinds, seed, flat=False):
    """tensors of these sizes, of the kinds in turn; flat: views of one buffer per kind (any element alignment)"""
    gen = torch.Generator().manual_seed(seed)
    kinds = kinds if isinstance(kinds, list) else [kinds]
    made = [torch.randn(n, generator=gen) * math.exp(i % 7 - 3) for i, n in enumerate(sizes)]
    if not flat:
        return [t.to(DEV).to(kinds[i % len(kinds)]) for i, t in enumerate(made)]
    out = []
    buffers = {k: torch.zeros(1 + sum(sizes), device=DEV, dtype=k) for k in kinds}
    at = dict.fromkeys(kinds, 1)
    for i, t in enumerate(made):
        k = kinds[i % len(kinds)]
        v = buffers[k][at[k]:at[k] + t.numel()]
        v.copy_(t)
        at[k] += t.numel()
        out.append(v)
    return out


def norm64(ts, kind=2):
    vals = [t.double().reshape(-1) for t in ts if t.numel()]
    if not vals:
        return 0.0
    return math.sqrt(math.fsum(float(v.square().sum()) for v in vals)) if kind == 2 else max(float(v.abs().max()) for v in vals)


def close(got, want):
    assert got.dtype == F32 and got.shape == ()
    assert abs(got.item() - want) <= (U + 1e-12) * want, (got.item(), want)


@pytest.mark.parametrize('flat', [False, True])
@pytest.mark.parametrize('kinds', [[F32], [BF], [F32, BF]], ids=['f32', 'bf16', 'both'])
@pytest.mark.parametrize('name', list(LISTS))
def test_norm(name, kinds, flat):
    from rtg import ops
    ts = gradients(LISTS[name], kinds, 1, flat)
    before = [t.clone() for t in ts]
    close(ops.total_norm(ts), norm64(ts))
    top = ops.total_norm(ts, float('inf'))
    assert top.item() == norm64(ts, 'inf')                     # a maximum is exact
    assert all(torch.equal(a, b) for a, b in zip(ts, before))


@pytest.mark.parametrize('flat', [False, True])
@pytest.mark.parametrize('kinds', [[F32], [BF], [F32, BF]], ids=['f32', 'bf16', 'both'])
@pytest.mark.parametrize('name', list(LISTS))
@pytest.mark.parametrize('norm_type', [2, float('inf')])
def test_clip(name, kinds, flat, norm_type):
    from rtg import ops
    ts = gradients(LISTS[name], kinds, 2, flat)
    before, norm = [t.clone() for t in ts], norm64(ts, norm_type)
    got = ops.clip_grads_(ts, 2 * norm + 1, norm_type)          # within the limit: not a bit changes
    close(got, norm)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    limit = 0.3 * norm
    close(ops.clip_grads_(ts, limit, norm_type), norm)
    f = limit / (norm + 1e-6)
    for t, b in zip(ts, before):
        want = b.double() * f
        inside(t, want, (2 * U + half_step(t.dtype) + 1e-9) * want.abs() + 1e-40, 'clipped')


def test_against_torch():
    from rtg import ops
    import train
    shapes = [(64, 3, 5), (7,), (1,), (33, 9)]
    ps = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in shapes] + [torch.nn.Parameter(torch.zeros(3, device=DEV))]
    qs = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in shapes]
    for i, (p, q) in enumerate(zip(ps, qs)):
        p.grad = gradients([p.numel()], F32, i)[0].view(p.shape)
        q.grad = p.grad.clone()
    want = torch.nn.utils.clip_grad_norm_(qs, 0.5)
    versions = [p.grad._version for p in ps[:4]]
    got = train.clip_grad_norm_(iter(ps), 0.5)                   # the last parameter has no gradient
    assert abs(got.item() - want.item()) <= 4e-7 * want.item()   # torch: a norm of norms in float, 6 roundings
    for p, q in zip(ps, qs):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)
    assert all(p.grad._version > v for p, v in zip(ps, versions))
    assert train.clip_grad_norm_(ps[-1], 1.0).item() == 0.0
    close(ops.total_norm(ps[0].grad), norm64([ps[0].grad]))     # a single tensor


def test_permuted_and_gapped_gradients():
    from rtg import ops
    from rtg.lib import RtgError
    base = gradients([6000], F32, 3)[0]
    dense = base.view(20, 30, 10).permute(2, 0, 1)
    gaps = base.view(60, 100)[:, ::2]
    close(ops.total_norm([dense]), norm64([dense]))
    close(ops.total_norm([gaps]), norm64([gaps]))
    want = dense.clone() * (0.5 / (norm64([dense]) + 1e-6))
    ops.clip_grads_([dense], 0.5)
    torch.testing.assert_close(dense, want, rtol=4 * U, atol=0)
    keep = base.clone()
    for bad in (gaps, base[:1].expand(5), base.view(60, 100)[:, :50]):
        with pytest.raises(RtgError):
            ops.clip_grads_([bad], 0.5)
    assert torch.equal(base, keep)


def test_the_ends_of_the_float_range():
    """squares that no float holds, in both directions"""
    from rtg import ops
    for value, n in ((3e38, 1), (1e30, 5000), (1e-30, 5000), (1.4e-45, 1), (1.4e-45, 100)):
        t = torch.full((n,), value, device=DEV)
        want = norm64([t])
        got = ops.total_norm([t]).item()
        assert abs(got - want) <= U * want + 0.75e-45, (value, n, got, want)     # (half a step of the smallest floats)
    big = torch.full((4096,), 1e37, device=DEV)                                     # the norm itself still fits
    ops.clip_grads_([big], 64.0)
    inside(big, torch.ones(4096, device=DEV, dtype=torch.float64), torch.full((4096,), 4 * U, device=DEV, dtype=torch.float64), 'clipped')


@pytest.mark.parametrize('norm_type', [2, float('inf')])
@pytest.mark.parametrize('where', [0, 5000, 99_999])
def test_gradients_that_are_not_finite(where, norm_type):
    from rtg import ops
    ts = gradients([100_000, 17], [F32, BF], 4)
    ts[0][where] = float('-inf')
    assert ops.total_norm(ts, norm_type).item() == float('inf')
    ops.clip_grads_(ts, 1.0, norm_type)                          # torch's: the factor is 0
    assert torch.isnan(ts[0][where]) and ts[0].isnan().sum() == 1 and not ts[0].nan_to_num().any() and not ts[1].any()
    ts = gradients([100_000, 17], [F32, BF], 4)
    ts[0][where] = float('nan')
    assert math.isnan(ops.total_norm(ts, norm_type).item())
    ops.clip_grads_(ts, 1.0, norm_type)
    assert ts[0].isnan().all() and ts[1].isnan().all()


def test_limits_of_zero_and_infinity():
    from rtg import ops
    ts = gradients([1000], F32, 5)
    before = ts[0].clone()
    ops.clip_grads_(ts, float('inf'))
    assert torch.equal(ts[0], before)
    ops.clip_grads_(ts, 0.0)
    assert not ts[0].any()
    assert ops.clip_grads_(ts, 1.0).item() == 0.0


def test_more_elements_than_32_bits_count():
    from rtg import ops
    n = (1 << 31) + 4099
    t = torch.zeros(n, device=DEV, dtype=BF)
    t[0], t[n // 2], t[-1] = 3.0, 4.0, 12.0
    close(ops.total_norm([t]), 13.0)
    ops.clip_grads_([t], 6.5)
    assert (t[0].item(), t[n // 2].item(), t[-1].item()) == (1.5, 2.0, 6.0) and t.count_nonzero().item() == 3


@pytest.mark.parametrize('kind', [F32, BF])
@pytest.mark.parametrize('norm_type', [2, float('inf')])
def test_lists_that_no_cache_holds(norm_type, kind):
    """more than 256 MB, which are read past the caches, with more partials than a workgroup of the scaling reads by itself"""
    from rtg import ops
    flat = torch.randn(150_000_001, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV).to(kind)
    ts = [t for t in flat[1:].split(31_013)]
    assert len(ts) > 4096
    before, norm = flat.clone(), norm64([flat[1:]], norm_type)
    close(ops.total_norm(ts, norm_type), norm)
    close(ops.clip_grads_(ts, 2 * norm, norm_type), norm)
    assert torch.equal(flat, before)
    close(ops.clip_grads_(ts, 0.3 * norm, norm_type), norm)
    want = before[1:].double() * (0.3 * norm / (norm + 1e-6))
    inside(flat[1:], want, (2 * U + half_step(kind) + 1e-9) * want.abs() + 1e-40, 'clipped')
    assert flat[0] == before[0]


def test_many_small_tensors():
    """more partials than a workgroup of the scaling reads by itself, in a list that a cache holds"""
    from rtg import ops
    ts = gradients([50 + i % 11 for i in range(5000)], [F32, BF], 8, True)
    before, norm = [t.clone() for t in ts], norm64(ts)
    close(ops.clip_grads_(ts, 0.3 * norm), norm)
    f = 0.3 * norm / (norm + 1e-6)
    for kind in (F32, BF):
        got, want = (torch.cat([t for t in l if t.dtype == kind]).double() for l in (ts, before))
        inside(got, want * f, (2 * U + half_step(kind) + 1e-9) * want.abs() + 1e-40, 'clipped')


def test_memory_around_the_tensors_is_left_alone():
    from rtg import ops
    for kind in (F32, BF):
        for n in (1, 3, 1000, 4097, 300_003):
            for off in (1, 2, 3, 5):
                big = torch.full((n + 64,), 7.0, device=DEV, dtype=kind)
                mid = big[off:off + n]
                ops.clip_grads_([mid], 1.0)
                assert (big[:off] == 7).all() and (big[off + n:] == 7).all() and (mid != 7).all()


def test_refusals():
    from rtg import ops
    from rtg.lib import RtgError
    t = gradients([100], F32, 6)[0]
    for bad in ([], [t.half()], [t.double()], [t.cpu()], [t, t.cpu()], [torch.sparse_coo_tensor([[0]], [1.0], (4,)).to(DEV)]):
        with pytest.raises(RtgError):
            ops.total_norm(bad)
        with pytest.raises(RtgError):
            ops.clip_grads_(bad, 1.0)
    for limit in (-1.0, float('nan'), t[:1]):
        with pytest.raises(RtgError):
            ops.clip_grads_([t], limit)
    with pytest.raises(RtgError):
        ops.total_norm([t], 3)
    keep = t.clone()
    for overlap in ([t, t], [t[:60], t[50:]], [t[50:], t[:51]]):
        with pytest.raises(RtgError):
            ops.clip_grads_(overlap, 1e-3)
    assert torch.equal(t, keep)
    close(ops.total_norm([t, t]), norm64([t, t]))                # only reading


# ---------------------------------------------------------------------------------------------------------------------
# AdamW with clipped gradients
# ---------------------------------------------------------------------------------------------------------------------
LR, BETAS, EPS, DECAY = 3e-3, (0.8, 0.99), 1e-8, 0.01


def state(sizes, seed, off=0, step=4.0):
    gen = torch.Generator().manual_seed(seed)

    def buf(n, scale, positive=False):
        t = scale * torch.randn(n + off, generator=gen)
        return (t.abs() if positive else t).to(DEV)[off:]
    s = {k: [buf(n, sc, k == 'v') for n in sizes] for k, sc in (('p', 0.5), ('g', 0.1), ('m', 0.05), ('v', 0.01))}
    s['t'] = [torch.full((1,), step, device=DEV) for _ in sizes]
    return s


def update(s, limit, **kw):
    from rtg import ops
    return ops.clipped_adamw_(s['p'], s['g'], s['m'], s['v'], s['t'], limit, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, **kw)


def want64(s, limit, scale=1.0):
    """the update in 64 bits -> (norm, per buffer (p, m, v) and their bounds)"""
    norm = norm64(s['g']) * scale
    f = min(1.0, limit / (norm + 1e-6)) * scale
    out = []
    for p, g, m, v, t in zip(s['p'], s['g'], s['m'], s['v'], s['t']):
        p, g, m, v, t = p.double(), g.double() * f, m.double(), v.double(), t.item() + 1
        m1 = BETAS[0] * m + (1 - BETAS[0]) * g
        v1 = BETAS[1] * v + (1 - BETAS[1]) * g * g
        den = v1.sqrt() / math.sqrt(1 - BETAS[1] ** t) + EPS
        rate = LR / (1 - BETAS[0] ** t)
        p1 = p * (1 - LR * DECAY) - rate * m1 / den
        # the factor: 2 roundings, the product 1; m: difference, weight, product, sum; v: only positive terms, 12 roundings;
        # the quotient: those of m and half of v's, and 6 of its own
        m_off = 8 * U * (m.abs() + g.abs())
        v_off = 12 * U * v1
        p_off = 3 * U * (p.abs() + p1.abs()) + rate / den * m_off + 16 * U * (rate * m1 / den).abs()
        out.append(((p1, p_off), (m1, m_off), (v1, v_off)))
    return norm, out


def verify(s, norm, want, got):
    close(got, norm)
    for p, m, v, w in zip(s['p'], s['m'], s['v'], want):
        for a, (b, off), name in zip((p, m, v), w, ('parameters', 'first moment', 'second moment')):
            inside(a, b, off + 1e-40, name)


@pytest.mark.parametrize('off', [0, 1])
@pytest.mark.parametrize('limit', [0.4, 1e6])
@pytest.mark.parametrize('sizes', [[1], [3, 5], [4096, 4097, 1023], [300_001, 17], [2_748_371], [50] * 40, [5_000_003, 12_000_001], [1000] * 32])
def test_update(sizes, limit, off):
    s = state(sizes, 1, off)
    g = [t.clone() for t in s['g']]
    norm, want = want64(s, limit * norm64(s['g']))
    got = update(s, limit * norm)
    verify(s, norm, want, got)
    assert all(t.item() == 5.0 for t in s['t']) and all(torch.equal(a, b) for a, b in zip(g, s['g']))
    norm, want = want64(s, limit * norm)                        # and once more from there
    verify(s, norm, want, update(s, limit * norm))


def test_update_of_gradients_that_no_cache_holds():
    gen = torch.Generator(device=DEV).manual_seed(9)
    sizes = [70_000_001, 5]
    s = {k: [sc * torch.randn(n, generator=gen, device=DEV) for n in sizes] for k, sc in (('p', 0.5), ('g', 0.1), ('m', 0.05), ('v', 0.01))}
    s['v'] = [t.abs() for t in s['v']]
    s['t'] = [torch.full((1,), 4.0, device=DEV) for _ in sizes]
    limit = 0.4 * norm64(s['g'])
    norm, want = want64(s, limit)
    verify(s, norm, want, update(s, limit))


def test_without_a_limit_it_is_the_update_that_was_there():
    from rtg.lib import lib, check, current_stream_ptr
    from rtg.ops import _p
    a, b = state([100_003], 2), state([100_003], 2)
    update(a, float('inf'), grad_scale=0.5)
    check(lib.rtg_adamw(_p(b['p'][0]), _p(b['g'][0]), _p(b['m'][0]), _p(b['v'][0]), 100_003, _p(b['t'][0]), None, LR, *BETAS, EPS, DECAY, 0.5,
                        current_stream_ptr()))
    for k in 'pmvt':
        torch.testing.assert_close(a[k][0], b[k][0], rtol=4 * U, atol=1e-9)


def test_scaled_gradients_and_first_step():
    s = state([5000, 333], 3, step=0.0)
    for k in 'mv':
        [t.zero_() for t in s[k]]
    norm, want = want64(s, 0.05, 0.25)
    verify(s, norm, want, update(s, 0.05, grad_scale=0.25))


def test_flags_and_norms_that_leave_buffers_alone():
    nan, one = torch.full((), float('nan'), device=DEV), torch.ones(1, device=DEV)
    s = state([5000, 70, 333], 4)
    before = {k: [t.clone() for t in s[k]] for k in s}
    norm, want = want64(s, 0.05)
    close(update(s, 0.05, loss_flags=[one, nan, None]), norm)
    for i, same in enumerate((False, True, False)):
        for k in 'pmvt':
            assert torch.equal(s[k][i], before[k][i]) == same, (k, i)
        if not same:
            for k, (b, off) in zip('pmv', want[i]):
                inside(s[k][i], b, off + 1e-40, k)
    for value in (float('inf'), float('nan')):
        s = state([5000, 70], 4)
        s['g'][1][3] = value
        before = {k: [t.clone() for t in s[k]] for k in s}
        got = update(s, 0.05)
        assert not math.isfinite(got.item())
        assert all(torch.equal(a, b) for k in 'pmvt' for a, b in zip(s[k], before[k]))


def test_adamw_refusals():
    from rtg import ops
    from rtg.lib import RtgError
    s = state([100], 5)
    p, g, m, v, t = (s[k] for k in 'pgmvt')
    for cols in (([], [], [], [], []), (p, g, m, v, []), (p, [g[0][:50]], m, v, t), (p, [g[0].bfloat16()], m, v, t), (p, g, m, v, [t[0].expand(2)]),
                 (p, p, m, v, t), (p, g, m, m, t), (p + p, g + g, m + m, v + v, t + t), (p, g, m, v, [m[0][5:6]]), (p, [g[0].cpu()], m, v, t),
                 (p, [torch.zeros(200, device=DEV)[::2]], m, v, t)):
        with pytest.raises(RtgError):
            ops.clipped_adamw_(*cols, 1.0)
    for kw in ({'grad_scale': 0.0}, {'grad_scale': -1.0}, {'loss_flags': []}, {'loss_flags': [torch.zeros(2, device=DEV)]},
               {'out': torch.zeros(2, device=DEV)}, {'out': t[0]}, {'out': m[0][7:8]}):
        with pytest.raises(RtgError):
            update(s, 1.0, **kw)
    for limit in (-1.0, float('nan')):
        with pytest.raises(RtgError):
            update(s, limit)


# ---------------------------------------------------------------------------------------------------------------------
# streams, graphs
# ---------------------------------------------------------------------------------------------------------------------
def test_two_streams_at_once():
    """calls on two streams side by side: nothing is shared between them"""
    from rtg import ops
    lists = [gradients([1_000_003, 70, 5000], [F32, BF], s) for s in (1, 2)]
    want = [ops.total_norm(ts).item() for ts in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(ops.total_norm(lists[k]))
    torch.cuda.synchronize()
    assert all(x.item() == want[k] for k in range(2) for x in got[k])


def test_captured_into_graphs():
    """a clip and an update in two graphs, replayed in turn with eager calls and new gradients between"""
    from rtg import ops
    sizes = [3000, 5, 100_001]
    ts, s = gradients(sizes, [F32, BF], 1), state([5000, 333], 2)
    ops.clip_grads_([t.clone() for t in ts], 1.0)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        norm_a = ops.clip_grads_(ts, 2.5)
    with torch.cuda.graph(gb):
        norm_b = update(s, 0.1)
    for r in range(3):
        for t, new in zip(ts, gradients(sizes, [F32, BF], 10 + r)):
            t.copy_(new)
        eager = [t.clone() for t in ts]
        ga.replay()
        want = ops.clip_grads_(eager, 2.5)
        twin = {k: [t.clone() for t in s[k]] for k in s}
        gb.replay()
        want_b = update(twin, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(norm_a, want) and all(torch.equal(a, b) for a, b in zip(ts, eager)), r
        assert torch.equal(norm_b, want_b) and all(torch.equal(a, b) for k in s for a, b in zip(s[k], twin[k])), r


def test_the_same_list_gives_the_same_bits():
    from rtg import ops
    ts = gradients(LISTS['many'] + [2_000_003], [F32, BF], 7)
    first = ops.total_norm(ts)
    assert all(torch.equal(first, ops.total_norm(ts)) for _ in range(5))


# ---------------------------------------------------------------------------------------------------------------------
# the set as a training step uses it
# ---------------------------------------------------------------------------------------------------------------------
def small_model():
    from models.layers import BankedModel, LayerNorm, WNConv, conv

    class Net(BankedModel):
        def __init__(self):
            super().__init__()
            self.a = WNConv('conv', 32, 32, 3, pad=1)
            self.norm = LayerNorm(32)
            self.b = WNConv('conv', 32, 32, 3, pad=1)
            self.rows = LayerNorm(50, dim=-1, bias=False)

        def forward(self, x):
            tok = self.token()
            return self.rows(conv(tok, self.b, self.norm(conv(tok, self.a, x))))
    torch.manual_seed(3)
    return Net().to(DEV)


def reference_loss(net, leaves, x, dy):
    import torch.nn.functional as F

    def unit(name):
        return leaves[name + '.weight_v'] / leaves[name + '.weight_v'].flatten(1).norm(dim=1).view(-1, 1, 1)
    wa, wb = (leaves[n + '.weight_g'] * unit(n) for n in 'ab')
    h = F.conv1d(x, wa, leaves['a.bias'], padding=1)
    h = F.layer_norm(h.transpose(1, 2), (32,), leaves['norm.weight'], leaves['norm.bias']).transpose(1, 2)
    h = F.conv1d(h, wb, leaves['b.bias'], padding=1)
    return (F.layer_norm(h, (50,), leaves['rows.weight']) * dy).sum(), h, wb, unit('b')


def test_a_model_with_layer_norms_trains_with_clipped_updates():
    """forward, backward, norm, clipped update of a model of convolutions and layer norms in one flat buffer: gradients against
    the same model in 64 bits (float convolutions of 96 terms: 1e-5 of a gradient's norm), the update against torch's clipping and
    AdamW in 64 bits on these gradients"""
    import train
    net = small_model()
    opt = train.AdamW(net.parameters(), 2e-3, betas=[0.8, 0.99], max_norm=0.5)
    gen = torch.Generator().manual_seed(1)
    names = [n for n, _ in net.named_parameters()]
    ref = None
    for step in range(3):
        x, dy = torch.randn(4, 32, 50, generator=gen), torch.randn(4, 32, 50, generator=gen)
        leaves = {n: p.detach().cpu().double().requires_grad_(True) for n, p in net.named_parameters()}
        loss, h, wb, unit = reference_loss(net, leaves, x.double(), dy.double())
        *want, dh, dwb = torch.autograd.grad(loss, [leaves[n] for n in names] + [h, wb])
        opt.zero_grad()
        (net(x.to(DEV)) * dy.to(DEV)).sum().backward()
        bank = net.bank()
        bank.sync_grads()
        for n, p, w in zip(names, net.parameters(), want):
            # The last layer norm takes a row's level and scale away, so b.bias (a level: the gradient is the sum of dh over a
            # row) and b.weight_g (a scale: the sum of dwb * v / |v| over a row of weights) have gradients of next to nothing: sums
            # that cancel.  What a sum of floats is off by goes by the size of its terms (k u sum|terms|), not of their sum.
            size = {'b.bias': dh.abs().sum((0, 2)), 'b.weight_g': (dwb * unit).abs().sum((1, 2))}.get(n, w)
            assert (p.grad.cpu().double() - w).norm() <= 1e-5 * size.norm(), n
        if ref is None:
            ref = [torch.nn.Parameter(p.detach().cpu().double()) for p in net.parameters()]
            topt = torch.optim.AdamW(ref, 2e-3, betas=(0.8, 0.99))
        for q, p in zip(ref, net.parameters()):
            q.grad = p.grad.cpu().double()
        norm = torch.nn.utils.clip_grad_norm_(ref, 0.5)
        opt.step()
        topt.step()
        assert norm > 0.5 and abs(opt.total_norm.item() - norm.item()) <= 2e-7 * norm.item()
        for n, q, p in zip(names, ref, net.parameters()):
            # a float's rounding per step, and the update's 16 (of at most lr times a few)
            assert (p.detach().cpu().double() - q.detach()).abs().max() <= (step + 1) * (2 * U * q.abs().max() + 64 * U * 2e-3 * 10), n


def test_clip_grad_norm_of_a_banked_model():
    import train
    net = small_model()
    x = torch.randn(2, 32, 50, generator=torch.Generator().manual_seed(2)).to(DEV)
    net(x).square().sum().backward()
    bank = net.bank()
    bank.sync_grads()
    before, want = bank.gflat.clone(), norm64([p.grad for p in net.parameters()])
    close(train.clip_grad_norm_([net, *net.parameters()], 0.25 * want), want)      # a parameter given twice is scaled once
    inside(bank.grads(), before[:-1].double() * 0.25, 4 * U * before[:-1].double().abs() + 1e-7 * before[:-1].double().abs(), 'clipped')
    close(train.clip_grad_norm_(net, 1e9), norm64([p.grad for p in net.parameters()]))


@pytest.mark.parametrize('graphed', [False, True])
@pytest.mark.parametrize('share', [None, 1e-3, 1e3])
def test_trainer_with_a_limit_on_the_gradients(monkeypatch, share, graphed):
    """hparam.grad_clip (a share of a first step's norm): one more step, eager or replayed, from the weights and moments after the
    first ones is, on the gradients that it leaves in the flat buffers, the clipped update in 64 bits; without a limit, the
    update that was there.  (Two trainers cannot be compared: each tunes its own block shapes, and a first AdamW step turns the
    last bits of a gradient next to 0 into up to twice the learning rate.)"""
    import hparam as hp
    import train

    def build(clip):
        monkeypatch.setattr(hp, 'grad_clip', clip)
        torch.manual_seed(0)
        return train.Trainer(use_mpd=False, use_mtd=False, d_train_times=1, dev='cuda:0')
    gen = torch.Generator().manual_seed(5)
    batch = [t.to(DEV) for t in (torch.randn(1, 80, 32, generator=gen), *(torch.rand(1, 1, 8192, generator=gen) * 2 - 1 for _ in range(2)))]
    clip = None
    if share is not None:
        probe = build(1e30)
        probe.train_step(*batch)
        clip = share * min(probe.optim_d.total_norm.item(), probe.optim_g.total_norm.item())
    tr = build(clip)
    step = tr.train_step_graphed if graphed else tr.train_step
    step(*batch)
    pairs = [(tr.optim_g, tr.generator), (tr.optim_d, tr.msd)]

    def now(opt, m):
        s, b = opt._st(m), m.bank()
        return {'p': [b.flat], 'g': [b.grads()], 'm': [s['exp_avg']], 'v': [s['exp_avg_sq']], 't': [s['step']]}
    before = [{k: [t.clone() for t in v] for k, v in now(*pair).items()} for pair in pairs]
    step(*batch)
    torch.cuda.synchronize()
    for (opt, m), old in zip(pairs, before):
        new = now(opt, m)
        monkeypatch.setitem(globals(), 'LR', opt.param_groups[0]['lr'])
        old['g'] = new['g']
        norm, want = want64(old, float('inf') if clip is None else clip)
        assert new['t'][0].item() == old['t'][0].item() + 1
        if clip is None:
            assert opt.total_norm is None
        else:
            close(opt.total_norm, norm)
            assert (norm > clip) == (share < 1)
        for k, (b, off) in zip('pmv', want[0]):
            inside(new[k][0], b, off + 1e-40, (type(m).__name__, k))
