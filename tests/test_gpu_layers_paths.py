"""Paths of the layer kernels that sizes alone choose, one case each side of a rule, on the GPU; bounds as in test_gpu_layers.py."""
import pytest
import torch

from test_gpu_layers import TYPES, gated_inputs, gated_reference, within

pytestmark = pytest.mark.gpu

CODES = {'f32': 0, 'f16': 1, 'bf16': 2}


def guarded(nbytes):
    return torch.full((nbytes + 4096,), 0x5a, dtype=torch.uint8, device='cuda')


# runs of the second product's k: 16 bits 256 long for up to 16 rows, 128 beyond and in fp32; as many workgroups as have one
@pytest.mark.parametrize('dtype,rows,k,f,n_out', [
    ('bf16', 1, 64, 2048, 512), ('f16', 16, 200, 2049, 40), ('bf16', 9, 130, 4000, 200), ('f16', 3, 200, 9000, 16), ('bf16', 17, 136, 1024, 100),
    ('f16', 64, 200, 1025, 8), ('f32', 1, 200, 1024, 64), ('f32', 16, 140, 3000, 33), ('f32', 50, 160, 2050, 200), ('bf16', 2, 200, 255, 9)])
def test_few_rows_share_a_tile_among_workgroups(dtype, rows, k, f, n_out):
    from nerf_amd._lib import lib, ptr
    t, code, L = TYPES[dtype], CODES[dtype], lib()
    x, p, dy = gated_inputs(rows, k, f, n_out, t, seed=60)
    n, size = L.nerf_gated_mlp_fwd_workspace_bytes(code, rows, k, f, n_out), rows * n_out * t.itemsize
    ws, y = guarded(n), guarded(size)
    assert L.nerf_gated_mlp_fwd(ptr(p), ptr(x), code, rows, k, f, n_out, 0, ptr(y), None, ptr(ws), n, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert (ws[n:] == 0x5a).all() and (y[size:] == 0x5a).all()
    wy, by = gated_reference(x, p, f, n_out, dy, 'silu', t)[:2]
    within(y[:size].view(t).view(rows, n_out), wy, by, 'y')
