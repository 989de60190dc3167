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


# float32 products are those of three bf16 parts of each side, six of nine (gated_mlp.hip).  Leaving one of the six out of one of the
# block's six kinds of product makes some result's relative root-mean-square error 2.4e-6 or more (test_layers_exact_cpu.py emulates that).
# With all of them it is made of roundings: one of a running sum is off by 2^-24 / sqrt(3) of it at the root mean square, and a sum in c
# steps, whose running value grows with the root of the step, by sqrt(c / 2) of those; a matrix instruction takes 16 or 32 of k, the
# low orders' steps are 2^-8 as large, so the longest sums here (4001 rows or 2667 hidden values, in splits) have c < 250: 3.8e-7.
# A result carries up to four such sums (g and u, dh, its own): 2^-20 = 9.5e-7 holds them and is less than half of what a lost product makes.
F32_RMS = 2.0 ** -20
F32_SHAPES = {
    'few rows': (40, 100, 130, 90),
    'narrow, one launch each way': (1000, 40, 100, 30),
    'narrow, two launches each way': (1000, 51, 241, 51),
    'wide, g, u, y and dh in one split': (1200, 72, 96, 80),
    'wide, splits': (700, 100, 130, 90),
    'wide, 256 tiles': (4001, 1001, 2667, 1001),
}


def relative_rms(got, want):
    return [rms(a.double() - b) / rms(b) for a, b in zip(got, want)]


def as_exact_as_float32(got, want):
    return max(relative_rms(got, want)) <= F32_RMS


def parted(dp, k, f, n_out):
    return [q.view(s) for q, s in zip(torch.split(dp, (f * k, f * k, n_out * f)), ((f, k), (f, k), (n_out, f)))]


@pytest.mark.parametrize('what', list(F32_SHAPES))
def test_float32_loses_none_of_its_products(what):
    from nerf_amd.layers import gated_mlp
    rows, k, f, n_out = F32_SHAPES[what]
    x, p, dy = gated_inputs(rows, k, f, n_out, torch.float32, seed=29)
    xr, pr = x.clone().requires_grad_(True), p.clone().requires_grad_(True)
    y = gated_mlp(xr, pr, f, n_out)
    dx, dp = torch.autograd.grad(y, (xr, pr), dy)
    want = gated64(x, p, f, n_out, dy)
    assert as_exact_as_float32([y.detach(), dx] + parted(dp, k, f, n_out), want), relative_rms([y.detach(), dx] + parted(dp, k, f, n_out), want)
    assert as_exact_as_float32([gated_mlp(x, p, f, n_out)], want)
