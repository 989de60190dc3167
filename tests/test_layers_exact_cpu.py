"""The check of test_gpu_layers_exact.py on float32 products, tried on the CPU: it passes the gated block computed with all six products
of three bf16 parts, and fails it with any one of them left out of any one kind of product."""
import pytest
import torch

from test_gpu_layers import act64
from test_gpu_layers_exact import F32_SHAPES, as_exact_as_float32, gated64, relative_rms

PRODUCTS = ((1, 1), (0, 2), (2, 0), (0, 1), (1, 0), (0, 0))
KINDS = ('g and u', 'y', 'dh', 'dx', 'dg and du by x', 'dy by h')


def parts(v):
    out = []
    v = v.float()
    for _ in range(3):
        out.append(v.bfloat16().double())
        v = v - out[-1].float()
    return out


def block(x, gate, up, down, dy, lost=None):
    """lost: (kind, product) that is left out.  Sums in 64 bits, rounded to 32 between the products."""
    def mm(kind, a, b):     # a [i, k] b [j, k]
        a, b = parts(a), parts(b)
        return sum(a[i] @ b[j].t() for i, j in PRODUCTS if (kind, (i, j)) != lost).float()
    g, u = mm('g and u', x, gate), mm('g and u', x, up)
    a, d = (v.float() for v in act64(g.double(), 'silu'))
    h, dh = a * u, mm('dh', dy, down.t())
    dg, du = dh * u * d, dh * a
    return (mm('y', h, down), mm('dx', dg, gate.t()) + mm('dx', du, up.t()), mm('dg and du by x', dg.t(), x.t()), mm('dg and du by x', du.t(), x.t()),
            mm('dy by h', dy.t(), h.t()))


@pytest.mark.parametrize('what', [w for w, s in F32_SHAPES.items() if s[0] < 2000])
def test_the_check_misses_no_lost_product(what):
    rows, k, f, n_out = F32_SHAPES[what]
    r = torch.Generator().manual_seed(7)
    x, dy = torch.randn(rows, k, generator=r), torch.randn(rows, n_out, generator=r)
    gate, up, down = ((torch.rand(o, i, generator=r) * 2 - 1) * (6.0 / (o + i)) ** 0.5 for o, i in ((f, k), (f, k), (n_out, f)))
    want = gated64(x, torch.cat([m.reshape(-1) for m in (gate, up, down)]), f, n_out, dy)
    assert as_exact_as_float32(block(x, gate, up, down, dy), want)
    for kind in KINDS:
        for product in PRODUCTS:
            got = block(x, gate, up, down, dy, (kind, product))
            assert not as_exact_as_float32(got, want), (kind, product)
            assert max(relative_rms(got, want)) >= 2.2e-6, (kind, product)
