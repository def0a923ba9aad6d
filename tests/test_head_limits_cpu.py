"""Sizes that the feature-head layers refuse before anything touches the device."""
import pytest

from tests.test_head_cpu import P, UNSUP, L  # noqa: F401


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_more_rows_than_a_launch_has_threads_for(L, dtype):  # noqa: F811
    """A row count whose tiles need 2^32 threads or more (64 rows a block of 256): refused by size, not by a failed launch."""
    for R in (1 << 33, 1 << 36, 1 << 40):
        assert L.w3d_linear_fwd(P, P, None, 0, None, R, 8, 8, dtype, 0, P, None, P, 4096, None) == UNSUP
        assert L.w3d_gated_linear_fwd(P, P, P, None, None, 0, R, 8, 8, dtype, 3, P, None, P, 4096, None) == UNSUP
    assert L.w3d_linear_fp8_fwd(P, P, P, P, None, 0, None, 1 << 36, 16, 8, 1, 0, P, P, 4096, None) == UNSUP
