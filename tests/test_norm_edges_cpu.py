"""Calls of layer norm and of the gradient operators that lie beside the ordinary ones, as far as a machine without a GPU shows
them: the launches are replaced by functions that look at what they are given."""
import pytest
import torch


class Launches:
    """stands in for the library: keeps the description and the address of each layer norm backward launch"""

    def __init__(self):
        self.backward = []

    def rtg_layernorm_forward(self, *args):
        return 0

    def rtg_layernorm_ws(self, ref):
        return 16

    def rtg_layernorm_backward(self, ref, dy, x, *args):
        d = ref._obj
        self.backward.append(((d.outer, d.n, d.inner, d.x_outer, d.x_n), x))
        return 0


@pytest.fixture
def launches(monkeypatch):
    from rtg import ops
    fake = Launches()
    monkeypatch.setattr(ops, 'lib', fake)
    monkeypatch.setattr(ops, '_stream', lambda: None)
    monkeypatch.setattr(ops, '_NORM_SEEN', {})
    return fake


def apply(x, w, b, dim):
    from rtg import ops
    return ops.LayerNormFn.apply(x, w, b, 1e-5, ops._norm_plan(x.shape, x.stride(), dim, x.dtype is torch.bfloat16, False, 1e-5))


VIEWS = {'time crop': (lambda t: t[:, :, 5:44], 1), 'channel slice': (lambda t: t[:, 7:30], 1), 'row slice': (lambda t: t[:, :, 3:67], 2),
         'last rows': (lambda t: t[:, -1], 1), 'whole': (lambda t: t, 1), 'every second': (lambda t: t[:, :, ::2], 1)}


@pytest.mark.parametrize('view', list(VIEWS))
def test_saved_activations_that_come_back_in_another_layout(launches, view):
    """a saved-tensor hook may give the values back dense: what the backward launch reads has to lie where the tensor is"""
    cut, dim = VIEWS[view]
    base = torch.randn(4, 64, 200)
    x = cut(base).requires_grad_(True)
    w, b = torch.ones(x.shape[dim], requires_grad=True), torch.zeros(x.shape[dim], requires_grad=True)
    back = []

    def unpack(t):
        back.append(t.float())
        return back[-1]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.double().contiguous(), unpack):
        y = apply(x, w, b, dim)
    torch.autograd.grad(y, (x, w, b), torch.ones(x.shape))
    saved = next(t for t in back if t.shape == x.shape)
    (outer, n, inner, x_outer, x_n), at = launches.backward[-1]
    assert (outer * n * inner, n, at) == (x.numel(), x.shape[dim], saved.data_ptr())
    last = (outer - 1) * x_outer + (n - 1) * x_n + inner - 1
    assert last == saved.numel() - 1 == saved.untyped_storage().nbytes() // 4 - 1, 'the launch reads behind the tensor'
    # ... and without a hook it is read in place, where it can be
    torch.autograd.grad(apply(x, w, b, dim), (x, w, b), torch.ones(x.shape))
    assert (launches.backward[-1][1] == x.data_ptr()) == (view != 'every second')


def test_saved_tensors_that_come_back_as_others_are_refused(launches):
    from rtg.lib import RtgError
    x, w = torch.randn(6, 16, requires_grad=True), torch.ones(16, requires_grad=True)
    for what, other in (('activations', lambda t: t[:3] if t.dim() == 2 else t), ('activations', lambda t: t.double() if t.dim() == 2 else t),
                        ('weight', lambda t: t[:8] if t.shape == (16,) else t), ('weight', lambda t: t.bfloat16() if t.shape == (16,) else t),
                        ('statistics', lambda t: t[:6] if t.shape == (12,) else t)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), other):
            y = apply(x, w, None, 1)
        with pytest.raises(RtgError, match=what):
            torch.autograd.grad(y, (x, w), torch.ones(6, 16))
    assert not launches.backward


@pytest.mark.parametrize('which', [0, 1, 2])
@pytest.mark.parametrize('wants_grad', [False, True])
def test_forward_mode_tangents_are_refused(launches, monkeypatch, which, wants_grad):
    """a dual operand's tangent would be lost without a word"""
    import torch.autograd.forward_ad as fw
    from rtg import ops
    from rtg.lib import RtgError
    monkeypatch.setattr(ops, '_need_here', lambda *a: None)
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: -1)
    ts = [torch.randn(4, 8).requires_grad_(wants_grad), torch.ones(8), torch.zeros(8)]
    with fw.dual_level():
        duals = list(ts)
        duals[which] = fw.make_dual(ts[which], torch.ones_like(ts[which]))
        for call in (ops.layer_norm, ops.layer_norm_forward):
            with pytest.raises(RtgError, match='tangent'):
                call(*duals)
        if which < 2:
            with pytest.raises(RtgError, match='tangent'):
                ops.layer_norm_backward(ts[0], duals[0], torch.zeros(4), torch.ones(4), duals[1])
        assert ops.layer_norm(*ts).shape == (4, 8)              # operands without one are ordinary
    from models.layers import LayerNorm
    with pytest.raises((RtgError, RuntimeError)):
        torch.func.jvp(LayerNorm(8, dim=-1), (torch.randn(4, 8),), (torch.ones(4, 8),))


def test_an_import_leaves_the_threads_of_autograd_alone():
    """unless the program asks for its own thread (RTG_AUTOGRAD_THREADS=0)"""
    import os
    import subprocess
    import sys
    code = ("import torch, importlib; before = torch._C._is_multithreading_enabled(); importlib.import_module('transtacos-retunegan_amd'); "
            "from rtg import ops; import train, models; print(before, torch._C._is_multithreading_enabled())")
    env = {k: v for k, v in os.environ.items() if k != 'RTG_AUTOGRAD_THREADS'}
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, '-c', code], cwd=root, env=env, capture_output=True, text=True, check=True)
    assert out.stdout.split()[-2:] == ['True', 'True']


@pytest.mark.parametrize('name', ['Generator_RefineGAN_small', 'Generator_RefineGAN'])
def test_generators_list_their_layer_norms(name):
    """a layer norm added to a generator joins its flat buffers, beside the parameter that the generator lists itself"""
    from models import generator
    from models.layers import LayerNorm

    class Normed(getattr(generator, name)):
        def __init__(self):
            super().__init__()
            self.norm = LayerNorm(32)
    own = [n for n, _ in getattr(generator, name)()._bank_params()]
    net = Normed()
    assert own == ['noise.w']
    got = dict(net._bank_params())
    assert set(got) == {'norm.weight', 'norm.bias', 'noise.w'} and got['norm.weight'] is net.norm.weight and got['noise.w'] is net.noise.w


def test_a_layer_norm_left_out_of_the_bank_is_refused():
    from models.layers import BankedModel, LayerNorm
    from rtg.lib import RtgError

    class Net(BankedModel):
        def __init__(self):
            super().__init__()
            self.norm, self.scale = LayerNorm(4), torch.nn.Parameter(torch.ones(3))

        def _extra_bank_params(self):
            return [('scale', self.scale), ('norm.weight', self.norm.weight)]
    with pytest.raises(RtgError, match='norm.bias'):
        Net()._bank_params()


def test_a_loss_flag_inside_a_written_buffer_is_refused():
    """flags are read while, or after, other buffers are written: what the update itself writes is none"""
    import ctypes as C
    from rtg.lib import AdamWJob, lib
    one = C.c_void_p(256)

    def adamw(*jobs, out=one):
        return lib.rtg_adamw_clipped(len(jobs), (AdamWJob * len(jobs))(*jobs), 1.0, 1e-3, 0.9, 0.99, 1e-8, 0.01, 1.0, one, out, None)
    # parameters, gradients, moments, step, flag, elements
    first, second = [512, 1024, 1536, 2048, 2560, None, 10], [8512, 81024, 81536, 82048, 82560, None, 10]
    for flag in (512, 548, 1536, 2048 + 36, 2560, 256, 2558):
        assert adamw(tuple(first[:5] + [flag, 10])) == -1, flag
        assert adamw(tuple(first), tuple(second[:5] + [flag, 10])) == -1, flag
        assert adamw(tuple(first[:5] + [1024, 10]), tuple(second[:5] + [flag, 10]), out=one) == -1, flag


def test_a_norm_inside_a_clipped_gradient_is_refused():
    import ctypes as C
    from rtg.lib import lib
    ptrs, counts, bf16 = (C.c_void_p * 2)(4096, 512), (C.c_longlong * 2)(10, 10), (C.c_int * 2)(0, 1)
    for out in (4096, 4132, 512, 516, 528):
        assert lib.rtg_grad_clip(2, ptrs, counts, bf16, 0, 1.0, C.c_void_p(64), C.c_void_p(out), None) == -1, out
