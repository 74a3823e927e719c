"""CPU tests (no GPU) of the workspaces of compact rows: what a call asks for is what its kernels write."""
import pytest


@pytest.mark.parametrize("n,da,db", [(1, 40, 5), (700, 4096, 2304), (16384, 4096, 4096), (300, 66000, 100), (0, 70000, 1000)])
def test_gemm_tn_asks_for_no_second_result_where_nothing_is_joined(n, da, db):
    """129 tiles of 256 x 256 and more, or few rows: the product is written where it belongs, there are no partial sums."""
    from vittles_amd import _lib
    nbytes = _lib.load().vt_mx_gemm_tn_workspace_bytes(n, da, db)
    assert 0 < nbytes <= 256         # never 0: callers hand in the address of what they are told to allocate


@pytest.mark.parametrize("n,da,db", [(16384, 1000, 99), (2000, 2560, 2550), (5001, 300, 33)])
def test_gemm_tn_asks_for_every_slab(n, da, db):
    from vittles_amd import _lib
    nbytes = _lib.load().vt_mx_gemm_tn_workspace_bytes(n, da, db)
    assert nbytes % (4 * da * db) == 0 and 2 <= nbytes // (4 * da * db) <= 512
