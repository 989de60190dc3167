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
