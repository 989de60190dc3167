"""Rules of the layer entry points that can be seen in the workspaces they ask for, without a GPU."""
import pytest

from nerf_amd import _lib


@pytest.fixture(scope='module')
def lib():
    return _lib.lib()


def up32(n):
    return (n + 31) // 32 * 32


def up256(n):
    return (n + 255) // 256 * 256


@pytest.mark.parametrize('dtype,rows,f,groups', [
    (2, 1, 2048, 1), (1, 16, 2048, 1), (2, 1, 2049, 2), (1, 9, 4096, 2), (2, 17, 1024, 1), (1, 40, 2048, 2), (0, 1, 1024, 1), (0, 30, 1025, 2)])
def test_few_rows_have_no_workgroup_without_work(lib, dtype, rows, f, groups):
    """y of few rows: h (4 bytes a value), and the partial sums of as many workgroups a tile as have a run of k for eight waves.  A run:
    256 of 16 bits for up to 16 rows, 128 otherwise."""
    k, n = 200, 256     # (16 tiles of y: up to 32 workgroups a tile are wanted; rows of 400 and 800 bytes are not laid out anew)
    h = up256(rows * up32(f) * 4)
    assert lib.nerf_gated_mlp_fwd_workspace_bytes(dtype, rows, k, f, n) == h + (up256(groups * rows * n * 4) if groups > 1 else 0)


@pytest.mark.parametrize('dtype,most', [(0, 64), (1, 128), (2, 128)])
def test_a_block_in_one_kernel_needs_no_workspace_where_nothing_is_kept(lib, dtype, most):
    """Narrow widths without a backward pass to follow; with one, those beyond its own narrow kernel keep g and u and need one."""
    for rows in (1000, 786432):
        for k in (17, 64, 65, 128):
            alone = lib.nerf_gated_mlp_alone_workspace_bytes(dtype, rows, k, 128, 64)
            followed = lib.nerf_gated_mlp_fwd_workspace_bytes(dtype, rows, k, 128, 64)
            assert (alone == 0) == (k <= most) and (followed == 0) == (k <= 64) and followed >= alone
    assert lib.nerf_gated_mlp_alone_workspace_bytes(dtype, 4, 0, 8, 8) == -1 and lib.nerf_gated_mlp_alone_workspace_bytes(7, 4, 8, 8, 8) == -1
    for shape in ((5, 200, 264, 200), (900, 200, 264, 200), (0, 40, 64, 16)):
        assert lib.nerf_gated_mlp_alone_workspace_bytes(dtype, *shape) == lib.nerf_gated_mlp_fwd_workspace_bytes(dtype, *shape)
