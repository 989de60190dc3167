"""nerf_amd.layers under torch's other ways of calling, on the GPU (test_layers_modes_cpu.py covers them with a stand-in library)."""
import threading

import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_layers import Trunk, gated_inputs, randn

pytestmark = pytest.mark.gpu


@pytest.mark.filterwarnings('ignore')
@pytest.mark.parametrize('precision', ['float32', 'bfloat16'])
def test_a_traced_trunk_is_the_trunk(precision):
    net = Trunk(precision)
    index = torch.randint(0, 11, (300,), generator=torch.Generator().manual_seed(3)).cuda()
    feats = randn(300, 48, seed=8).to(torch.bfloat16 if precision == 'bfloat16' else torch.float32)
    frozen = Trunk(precision).requires_grad_(False)
    frozen.load_state_dict(net.state_dict())
    for module in (net, frozen):
        traced = torch.jit.trace(module, (index, feats), check_trace=False)
        for rows in (300, 41):
            torch.full((1 << 20,), float('nan'), device='cuda')        # (what freed memory would show)
            assert torch.equal(traced(index[:rows], feats[:rows]).detach(), module(index[:rows], feats[:rows]).detach())


def test_tangents_and_graphs_of_operations_are_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    from nerf_amd.layers import embedding, gated_mlp, rms_norm
    x, p, _ = gated_inputs(9, 16, 24, 16, torch.float32)
    w, index = torch.ones(16, device='cuda'), torch.arange(9, device='cuda')
    for call in (lambda q: gated_mlp(q, p, 24, 16), lambda q: rms_norm(q, w), lambda q: rms_norm(q, w, residual=q)[1], lambda q: embedding(index, q)):
        with torch.no_grad(), forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match='jvp'):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
            inside = call(x)
        assert torch.equal(inside, call(x))
        with pytest.raises(RuntimeError, match='make_fx'):
            make_fx(call)(x)
        with pytest.raises(RuntimeError, match='setup_context'):
            torch.func.vmap(call)(x[None])


def test_the_sum_kept_for_the_backward_pass_may_not_change():
    from nerf_amd.layers import rms_norm
    x = randn(5, 40, seed=1).requires_grad_(True)
    y, s = rms_norm(x, torch.ones(40, device='cuda'), residual=randn(5, 40, seed=2))
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_calls_of_several_threads():
    """Each on a stream of its own, forward and backward, with workspaces of its own."""
    from nerf_amd.layers import embedding, gated_mlp, rms_norm
    n = 4
    sets = [gated_inputs(700 + 50 * k, 48, 96, 48, torch.bfloat16, seed=10 * k) for k in range(n)]
    index = [torch.randint(0, 50, (len(sets[k][0]),), generator=torch.Generator().manual_seed(k)).cuda() for k in range(n)]
    tables = [randn(50, 48, seed=k).bfloat16() for k in range(n)]
    w = torch.ones(48, device='cuda')

    def one(k):
        x, p, dy = sets[k]
        leaves = [v.detach().clone().requires_grad_(True) for v in (x, p, tables[k])]
        y, s = rms_norm(leaves[0], w, residual=embedding(index[k], leaves[2], 0.5))
        return torch.autograd.grad(s + gated_mlp(y, leaves[1], 96, 48), leaves, dy)

    alone = [one(k) for k in range(n)]
    torch.cuda.synchronize()
    got, failed = [None] * n, []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[k] = one(k)
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # (shown in the main thread)
            failed.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for a, b in zip(alone, got):
        assert all(torch.equal(q, r) for q, r in zip(a, b))


@pytest.mark.filterwarnings('ignore')
@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_a_compiled_trunk_is_the_trunk(backend):
    net = Trunk()
    index = torch.randint(0, 11, (300,), generator=torch.Generator().manual_seed(3)).cuda()
    feats, dy = randn(300, 48, seed=8), randn(300, 3, seed=9)
    params = list(net.parameters())
    torch._dynamo.reset()
    compiled = torch.compile(net, backend=backend)
    for _ in range(2):
        got, want = compiled(index, feats), net(index, feats)
        assert torch.equal(got.detach(), want.detach())
        for a, b in zip(torch.autograd.grad(got, params, dy), torch.autograd.grad(want, params, dy)):
            assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(compiled(index, feats), net(index, feats))
    torch._dynamo.reset()
