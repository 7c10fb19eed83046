"""CPU: sizes that a launch of the token operators does not hold are refused on the host."""
import pytest

ARG, WS = 1, 2
P = 0x1000   # never dereferenced: every call below is refused on the host


@pytest.mark.parametrize("n,rows,width", [(10, 1 << 30, 1), (10, (1 << 29) + 64, 2), (0, 0x7ffffffe, 1), (1, 128, 1 << 23), (1, 1, 0x7fffffff)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_gradients_of_large_tables(lib, dtype, n, rows, width):
    assert lib.ligdiff_embed_grad(P, dtype, width, P, 8, n, rows, width, 1.0, P, dtype, width, 0, P, (1 << 62), None) == ARG


@pytest.mark.parametrize("n,rows,width", [(10, 1 << 28, 1), (1, 128, 1 << 21), (1, 2, 1 << 29), (1 << 20, 5000, 1 << 14), (0x7fffffff, 119, 64)])
def test_large_tables_that_fit(lib, n, rows, width):
    """Not refused for their size: the next check, of the workspace, is reached.  (Rows of 2^29 columns are too far apart for the
    tables in LDS and are sorted, in tiles of 256 columns and more.)"""
    assert lib.ligdiff_embed_grad(P, 0, width, P, 8, n, rows, width, 1.0, P, 0, width, 0, P, 0, None) == WS
