"""Scratch sizes of the linear-layer operators for any sizes an int holds.  Runs without a GPU."""
import pytest

from rtatblas_amd import native


@pytest.mark.parametrize("n", [1, 64, 65, 2 ** 30 - 1024, 2 ** 31 - 64, 2 ** 31 - 63, 2 ** 31 - 1])
@pytest.mark.parametrize("m", [1, 1000, 2 ** 31 - 1])
def test_bias_gradient(m, n):
    """Four rows of partial sums to 64 columns, and room to align them."""
    assert native.load().rtat_dbias_workspace_bytes(m, n) == 4 * ((n + 63) // 64) * m * 4 + 256
