"""Paths of the layer kernels that sizes alone choose, one case each side of a rule, on the GPU; bounds as in test_gpu_layers.py."""
import pytest
import torch

from test_gpu_layers import F32, TYPES, gated_inputs, gated_reference, randn, within

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


# Sort of the table's gradient: tiles of 1024 positions, of 4096 above 2^20 of them; their counts are summed in a launch of their own above 48
# tiles; a pass for every 8 bits of the table's size.
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('rows,entries,dim', [
    (60000, 70000, 5), (49152, 300, 3), (49153, 300, 3), (70000, 70000, 5), (1048576, 300, 1), (1048577, 256, 2), (1100000, 1000, 3),
    (2200000, 20, 1), (1200000, 70000, 2), (100000, 200, 9), (4096, 70000, 4), (4097, 300, 4)])
def test_every_position_reaches_its_entry(dtype, rows, entries, dim):
    """Gradients of small whole numbers: fp32 sums of them are exact below 2^24 in any order, so the table's gradient has to be the whole
    numbers' sum, rounded once -- for the guarded entry point with the workspace it asks for."""
    from nerf_amd._lib import lib, ptr
    t, code, L = TYPES[dtype], CODES[dtype], lib()
    g = torch.Generator().manual_seed(rows + entries)
    index = torch.randint(-2, entries + 2, (rows,), generator=g)        # some outside the table, on both sides
    index[rows // 2:rows // 2 + 5000] = entries // 3                    # and a long stretch of one entry
    whole = torch.randint(-9, 10, (rows, dim), generator=g)
    index, dy = index.cuda(), whole.to(t).cuda()
    ok = (index >= 0) & (index < entries)
    want = torch.zeros(entries, dim, dtype=torch.int64).index_add_(0, index.cpu()[ok.cpu()], whole[ok.cpu()])
    assert int(want.abs().max()) < 1 << 24
    n, size = L.nerf_embedding_bwd_workspace_bytes(code, entries, dim, rows), entries * dim * t.itemsize
    ws, out = guarded(n), guarded(size)
    assert L.nerf_embedding_bwd(ptr(index), ptr(dy), code, rows, entries, dim, 1.0, ptr(out), ptr(ws), n, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert (ws[n:] == 0x5a).all() and (out[size:] == 0x5a).all()
    assert torch.equal(out[:size].view(t).view(entries, dim), want.float().to(t).cuda())
    # and through the layer, with values whose sums do round: the same bits twice
    from nerf_amd.layers import embedding
    table, values = randn(entries, dim, seed=1).to(t).requires_grad_(True), randn(rows, dim, seed=2).to(t)
    once, again = (torch.autograd.grad(embedding(index, table, 0.7), table, values)[0] for _ in range(2))
    assert torch.equal(once, again)
    exact, size_of = (torch.zeros(entries, dim, dtype=torch.float64, device='cuda').index_add_(0, index[ok], v.double()[ok]) * 0.7
                      for v in (values, values.abs()))
    count = torch.bincount(index[ok], minlength=entries).double()[:, None]
    within(once, exact, (count + 8) * F32 * size_of, 'table gradient')      # (8: 0.7 in fp32 and its product among them)


# The wide block in 256 x 256 tiles: every product of it, in whole tiles and in ragged ones.
@pytest.mark.parametrize('dtype,rows,k,f,n_out,act', [
    ('bf16', 3000, 1500, 3000, 2900, 'silu'), ('f16', 3000, 1500, 3000, 2900, 'gelu'), ('bf16', 4096, 4096, 4096, 4096, 'relu'),
    ('f16', 4096, 4096, 4096, 4096, 'silu'), ('f32', 4001, 1001, 2667, 1001, 'gelu'), ('f32', 4096, 2048, 4096, 2048, 'silu')])
def test_large_tiles(dtype, rows, k, f, n_out, act):
    from nerf_amd.layers import gated_mlp
    from test_gpu_layers_exact import F32_RMS, rms
    t = TYPES[dtype]
    x, p, dy = gated_inputs(rows, k, f, n_out, t, seed=70)
    xr, pr = x.clone().requires_grad_(True), p.clone().requires_grad_(True)
    y = gated_mlp(xr, pr, f, n_out, activation=act)
    dx, dp = torch.autograd.grad(y, (xr, pr), dy)
    alone = gated_mlp(x, p, f, n_out, activation=act)
    wy, by, wdx, bdx, wdp, bdp = gated_reference(x, p, f, n_out, dy, act, t)
    for got, want, bound, what in ((y.detach(), wy, by, 'y'), (alone, wy, by, 'y alone'), (dx, wdx, bdx, 'dx'), (dp, wdp, bdp, 'dparams')):
        within(got, want, bound, what)
        # as a whole: 16 bits, the result's own rounding and one of hidden values of the same size (a ratio of 1.41; 1.5 leaves
        # room for fp32); float32: what test_gpu_layers_exact.py derives
        off = rms(got.double() - want)
        assert off <= (F32_RMS * rms(want) if t == torch.float32 else 1.5 * rms(want.to(t).double() - want)), (what, off)


# (weights of 32 hidden values in LDS: 16 KiB beside more than 64 columns of x, and 8 or 4 KiB for those of y: 192 and 256 hidden values in 160 KiB)
@pytest.mark.parametrize('dtype,k,f,n_out', [('bf16', 100, 192, 100), ('bf16', 100, 256, 64), ('f16', 128, 128, 40), ('f32', 50, 200, 60)])
def test_a_narrow_block_alone_allocates_its_result_only(dtype, k, f, n_out):
    from nerf_amd.layers import gated_mlp
    t, rows = TYPES[dtype], 30000
    x, p, dy = gated_inputs(rows, k, f, n_out, t, seed=80)
    gated_mlp(x[:65], p, f, n_out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = gated_mlp(x, p, f, n_out)
    assert torch.cuda.max_memory_allocated() - before <= (y.numel() * t.itemsize + 511) // 512 * 512      # (the allocator's step)
    wy, by = gated_reference(x, p, f, n_out, dy, 'silu', t)[:2]
    within(y, wy, by, 'y')
    kept = gated_mlp(x, p.clone().requires_grad_(True), f, n_out).detach()
    within(kept, wy, by, 'y with a backward pass to follow')
