"""How exact the gated block's results are as a whole, on the GPU: root-mean-square errors against its definition in 64 bits, beside the
element-by-element bounds of test_gpu_layers.py, which allow the worst case of every sum and so hide a lost product or part."""
import math

import pytest
import torch

from test_gpu_layers import TYPES, act64, gated_inputs

pytestmark = pytest.mark.gpu


def gated64(x, p, f, n_out, dy, act='silu'):
    """y, dx and the three gradients of the weights."""
    k = x.shape[1]
    x, p, dy = x.double(), p.double(), dy.double()
    gate, up, down = p[:f * k].view(f, k), p[f * k:2 * f * k].view(f, k), p[2 * f * k:].view(n_out, f)
    g, u = x @ gate.t(), x @ up.t()
    a, d = act64(g, act)
    dh = dy @ down
    dg, du = dh * u * d, dh * a
    return (a * u) @ down.t(), dg @ gate + du @ up, dg.t() @ x, du.t() @ x, dy.t() @ (a * u)


def rms(v):
    return float(v.double().square().mean().sqrt())


@pytest.mark.parametrize('dtype', ['f16', 'bf16'])
@pytest.mark.parametrize('rows,k,f,n_out', [(1, 2048, 2049, 2048), (1, 2047, 2100, 2047), (2, 1024, 1400, 1050), (1, 4095, 4200, 4100),
                                            (3, 1365, 1500, 1365), (68, 60, 200, 60), (99, 200, 41, 64), (4095, 200, 300, 1)])
def test_a_few_thousand_values_are_as_exact_as_their_rounding(dtype, rows, k, f, n_out):
    """Blocks of 2048 to 4095 values in the smallest of y, h and dx: hidden values in two parts.  An output then errs by its own rounding;
    a hidden value rounded to the type would double the variance (a ratio of 1.41).  The mean square of 2000 and more independent
    roundings is known to 1 / sqrt(2000) = 2 %, its root to 1 %: 1.15 is between the two and over ten deviations from either."""
    from nerf_amd.layers import gated_mlp
    t = TYPES[dtype]
    x, p, dy = gated_inputs(rows, k, f, n_out, t, seed=23)
    xr, pr = x.clone().requires_grad_(True), p.clone().requires_grad_(True)
    y = gated_mlp(xr, pr, f, n_out)
    dx, dp = torch.autograd.grad(y, (xr, pr), dy)
    want = gated64(x, p, f, n_out, dy)
    for got, w, what in ((y.detach(), want[0], 'y'), (gated_mlp(x, p, f, n_out), want[0], 'y alone'), (dx, want[1], 'dx'),
                         (dp, torch.cat([q.reshape(-1) for q in want[2:]]), 'dparams')):
        assert rms(got.double() - w) <= 1.15 * rms(w.to(t).double() - w), what
