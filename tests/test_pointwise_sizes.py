"""Sizes that the library is asked for without a GPU: no argument ends the process."""
import itertools

import pytest

from ss_conv import _ext

SIZES = [-1, 0, 1, 7, 4096]


@pytest.mark.parametrize("n", SIZES)
def test_workspaces_of_any_sizes(n):
    lib = _ext._lib
    for c, clouds, groups in itertools.product(SIZES, SIZES, SIZES):
        bytes_ = lib.ssc_groupnorm_workspace_bytes(n, c, clouds, groups)
        if min(n, c, clouds, groups) > 0:
            assert bytes_ >= 8 * clouds * (2 * c + groups)
    for k, h, dtype in itertools.product(SIZES, SIZES, range(3)):
        made = [lib.ssc_gated_fwd_workspace_bytes(dtype, n, k, h),
                lib.ssc_gated_kept_bytes(dtype, n, h),
                lib.ssc_gated_bwd_workspace_bytes(dtype, n, k, h)]
        assert 0 < min(made) and max(made) < 1 << 40
        if min(n, k, h) > 0:
            assert made[1] >= n * h * (8 if dtype == 0 else 6)
            assert made[2] >= n * h * 2 * (4 if dtype == 0 else 2)
