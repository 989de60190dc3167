"""rms_norm over the whole range of its types, on the GPU: squares that leave fp32's range must not show."""
import pytest
import torch

from test_gpu_layers import TYPES, norm_reference, randn, within

pytestmark = pytest.mark.gpu


# rows of every kernel: 1 to 64 threads a row, a workgroup a row, rows held in registers forward only, rows read again
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('power,eps', [(70, 1e-6), (100, 1e-6), (122, 0.0), (-60, 0.0), (-100, 0.0), (-118, 0.0), (-60, 1e-30)])
@pytest.mark.parametrize('rows,dim', [(3, 1), (70, 7), (9, 31), (20, 48), (5, 300), (33, 1000), (6, 2048), (300, 4099), (4, 9000), (3, 70001)])
def test_rows_of_any_size(dtype, power, eps, rows, dim):
    """Every other row scaled by a power of two that takes the sum of its squares out of fp32's range; the rows beside it stay as they are."""
    from nerf_amd.layers import rms_norm
    t = TYPES[dtype]
    by = torch.ones(rows, 1, device='cuda')
    by[::2] = 2.0 ** power
    x = (randn(rows, dim, seed=1).to(t).float() * by).to(t).requires_grad_(True)
    res = (randn(rows, dim, seed=5).to(t).float() * by).to(t).requires_grad_(True)
    w = (1 + 0.3 * randn(dim, seed=2)).to(t).requires_grad_(True)
    # (a gradient as large as the row, where its own result would leave the range otherwise)
    dy, ds = (randn(rows, dim, seed=3) * by.clamp(max=1)).to(t), randn(rows, dim, seed=4).to(t)
    eps32 = float(torch.tensor(eps, dtype=torch.float32))
    y = rms_norm(x, w, eps=eps)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wy, wby, wdx, bdx, wdw, bdw = norm_reference(x.detach(), w.detach(), None, dy, None, eps32, t)
    floor = 2.0 ** -126      # results below fp32's smallest normal number keep fewer bits
    within(y.detach(), wy, wby + floor, 'y')
    within(dx, wdx, bdx + floor, 'dx')
    within(dw, wdw, bdw + floor, 'dweight')
    y, s = rms_norm(x, w, residual=res, eps=eps)
    dx, dr, dw = torch.autograd.grad((y, s), (x, res, w), (dy, ds))
    assert torch.equal(s.detach(), (x.detach().float() + res.detach().float()).to(t)) and torch.equal(dx, dr)
    wy, wby, wdx, bdx, wdw, bdw = norm_reference(s.detach(), w.detach(), None, dy, ds, eps32, t)
    within(y.detach(), wy, wby + floor, 'y with a residual')
    within(dx, wdx, bdx + floor, 'dx with a residual')
    within(dw, wdw, bdw + floor, 'dweight with a residual')


@pytest.mark.parametrize('dim', [5, 48, 300, 2048, 5000, 20000])
def test_zeros_infinities_and_nans_stay_what_they_were(dim):
    from nerf_amd.layers import rms_norm
    x, w = randn(8, dim, seed=1), torch.ones(dim, device='cuda')
    x[1], x[2] = 0, 0
    x[3, dim // 2], x[4, 0], x[5] = float('inf'), float('nan'), 2.0 ** 127
    y = rms_norm(x, w, eps=1e-6)
    assert not y[1].any() and not y[2].any() and y[4].isnan().all()
    assert y[3, dim // 2].isnan() and not y[3, :dim // 2].any() and not y[3, dim // 2 + 1:].any()
    assert torch.allclose(y[5], torch.ones(dim, device='cuda'), rtol=0, atol=(dim + 16) * 2.0 ** -24)
    assert torch.isfinite(y[[0, 5, 6, 7]]).all() and torch.equal(y[[0, 6, 7]], rms_norm(x[[0, 6, 7]], w, eps=1e-6))
    assert rms_norm(x[1:3], w, eps=0.0).isnan().all()       # 0 / 0, as in the formula
