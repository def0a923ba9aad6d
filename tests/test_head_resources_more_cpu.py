"""Register use of the backward pass's smaller kernels (no GPU needed): nothing spills."""
import re

from tests.test_kernel_resources_cpu import _kernels


def test_backward_kernels_do_not_spill(tmp_path):
    k = _kernels(tmp_path)
    hot = ("dz_kernel", "column_sums_kernel", "rms_norm_wide_kernel", "rms_norm_bwd_wide_kernel", "rms_norm_dw_wide_kernel")
    seen = set()
    for n, v in k.items():
        for h in hot:
            if re.search(r"\d" + h, n):
                seen.add(h)
                assert v["scratch"] == 0, (n, v)
    assert seen == set(hot), set(hot) - seen
