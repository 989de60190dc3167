"""nerf_amd.layers under the modes in which torch watches a call for more than its result -- forward-mode differentiation, torch.func's
transforms, traced programs, graphs of operations -- without a GPU: a stand-in library computes what the entry points' header says of them with numpy,
on the raw addresses that the functions pass, so that whatever reaches a caller has gone the same way as on the GPU."""
import ctypes as C

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from nerf_amd import _lib, layers

FLOATS, INTS = C.c_float, C.c_int64


def at(kind, address, *shape):
    return np.ctypeslib.as_array((kind * int(np.prod(shape))).from_address(address)).reshape(shape)


class StandIn:
    """float32 only; entry points with the library's own argument types."""

    def __init__(self):
        for name in ('nerf_embedding_fwd', 'nerf_rmsnorm_fwd', 'nerf_gated_mlp_fwd'):
            result, args = _lib.SIGNATURES[name]
            setattr(self, name, C.CFUNCTYPE(result, *args)(getattr(self, '_' + name)))
        self.real = _lib.lib()

    def __getattr__(self, name):        # sizes of workspaces: the library's own
        return getattr(self.real, name)

    def _nerf_embedding_fwd(self, table, dtype, entries, dim, index, rows, scale, out, stream):
        at(FLOATS, out, rows, dim)[:] = at(FLOATS, table, entries, dim)[at(INTS, index, rows)] * np.float32(scale)
        return 0

    def _nerf_rmsnorm_fwd(self, x, residual, weight, dtype, weight_dtype, rows, dim, eps, total, y, stream):
        s = at(FLOATS, x, rows, dim)
        if residual:
            s = s + at(FLOATS, residual, rows, dim)
            at(FLOATS, total, rows, dim)[:] = s
        at(FLOATS, y, rows, dim)[:] = s / np.sqrt((s * s).mean(1, keepdims=True) + np.float32(eps)) * at(FLOATS, weight, dim)
        return 0

    def _nerf_gated_mlp_fwd(self, params, x, dtype, rows, k, f, n, act, y, saved, workspace, nbytes, stream):
        p, s = at(FLOATS, params, (2 * k + n) * f), at(FLOATS, x, rows, k)
        g, u = s @ p[:f * k].reshape(f, k).T, s @ p[f * k:2 * f * k].reshape(f, k).T
        at(FLOATS, y, rows, n)[:] = (np.maximum(g, 0) * u) @ p[2 * f * k:].reshape(n, f).T
        return 0


@pytest.fixture
def standin(monkeypatch):
    lib = StandIn()
    monkeypatch.setattr(layers, 'lib', lambda: lib)
    monkeypatch.setattr(layers, '_device', lambda *a: -1)
    monkeypatch.setattr(layers, '_current_device', lambda: -1)
    monkeypatch.setattr(layers, '_current_stream', lambda device: 0)
    return lib


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


W, PARAMS, INDEX = 1 + 0.1 * randn(8, seed=1), randn((2 * 8 + 3) * 5, seed=2), torch.tensor([3, 0, 3, 1, 2, 0])
# name -> (a function of one tensor of 8 columns, what it is in elementary operations)
CALLS = {
    'embedding': (lambda x: layers.embedding(INDEX, x, 0.5), lambda x: x[INDEX] * 0.5),
    'rms_norm': (lambda x: layers.rms_norm(x, W), lambda x: x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * W),
    'rms_norm, residual': (lambda x: layers.rms_norm(x, W, residual=x)[0],
                           lambda x: 2 * x / torch.sqrt((2 * x).square().mean(-1, keepdim=True) + 1e-6) * W),
    'gated_mlp': (lambda x: layers.gated_mlp(x, PARAMS, 5, 3, activation='relu'),
                  lambda x: ((x @ PARAMS[:40].view(5, 8).t()).clamp(min=0) * (x @ PARAMS[40:80].view(5, 8).t())) @ PARAMS[80:].view(3, 5).t()),
}


def close(got, want):
    # sums of 8 products of values up to some 4 in float32, twice, and a square root: 100 roundings are plenty
    return got.shape == want.shape and float((got - want).abs().max()) <= 100 * 2.0 ** -24 * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize('name', list(CALLS))
def test_the_stand_in_computes_the_formula(standin, name):
    call, plain = CALLS[name]
    x = randn(4, 8, seed=3)
    assert close(call(x), plain(x))
    assert close(call(x.clone().requires_grad_(True)).detach(), plain(x))


@pytest.mark.parametrize('name', list(CALLS))
def test_a_tangent_is_refused_not_lost(standin, name):
    """A dual tensor's tangent would not reach the output: also where it needs no gradient, and where none is recorded."""
    call, plain = CALLS[name]
    x = randn(4, 8, seed=3)
    for grad_mode in (True, False):
        with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match='jvp'):
                call(dual)
            assert close(call(x), plain(x))         # without a tangent the value is all there is
    assert close(call(x), plain(x))


@pytest.mark.parametrize('name', list(CALLS))
def test_function_transforms_are_refused(standin, name):
    call, _ = CALLS[name]
    x = randn(4, 8, seed=3)
    for transformed in (lambda: torch.func.jvp(call, (x,), (torch.ones_like(x),)), lambda: torch.func.vjp(call, x),
                        lambda: torch.func.grad(lambda q: call(q).sum())(x), lambda: torch.func.vmap(call)(x[None]),
                        lambda: torch.func.functionalize(call)(x)):
        with pytest.raises(RuntimeError, match='setup_context'):
            transformed()


@pytest.mark.filterwarnings('ignore')
@pytest.mark.parametrize('leaf', [False, True])
@pytest.mark.parametrize('name', list(CALLS))
def test_a_traced_program_makes_the_call(standin, name, leaf):
    """Also on other sizes than those it was traced with; and its arguments are checked on every run."""
    call, plain = CALLS[name]
    traced = torch.jit.trace(call, (randn(4, 8, seed=3).requires_grad_(leaf),), check_trace=False)
    for rows in (4, 7):
        x = randn(rows, 8, seed=4 + rows)
        assert close(traced(x).detach(), plain(x))
    for wrong in (randn(4, 8, seed=6).double(),) + (() if name == 'embedding' else (randn(4, 9, seed=6),)):
        with pytest.raises(RuntimeError, match='must be'):
            traced(wrong)


@pytest.mark.parametrize('mode', ['real', 'fake', 'symbolic'])
@pytest.mark.parametrize('name', list(CALLS))
def test_a_graph_of_operations_is_refused(standin, name, mode):
    """Such a graph would hold the allocation of the result and not the launch.  (Other dispatch modes, which record nothing, may be on.)"""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    call, plain = CALLS[name]
    for leaf in (False, True):
        x = randn(4, 8, seed=3).requires_grad_(leaf)
        with pytest.raises(RuntimeError, match='make_fx|data pointer'):
            make_fx(call, tracing_mode=mode)(x)
        with pytest.raises(RuntimeError, match='make_fx|data pointer'):
            make_fx(call, tracing_mode=mode, pre_dispatch=True)(x)
        with FlopCounterMode(display=False):
            assert close(call(x).detach(), plain(x))


@pytest.mark.filterwarnings('ignore')
@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
@pytest.mark.parametrize('name', list(CALLS))
def test_a_compiled_program_calls_out_of_its_graph(standin, name, backend):
    """torch.compile breaks its graph at the launch and makes the call itself."""
    call, plain = CALLS[name]
    for leaf in (False, True):
        torch._dynamo.reset()
        compiled = torch.compile(lambda q: call(q * 2) + 1, backend=backend)
        for rows in (4, 6):
            x = randn(rows, 8, seed=rows).requires_grad_(leaf)
            assert close(compiled(x).detach(), plain(x.detach() * 2) + 1)
    torch._dynamo.reset()
