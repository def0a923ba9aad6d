"""Register use of the feature-head kernels, read from the built library's code objects (no GPU needed): nothing spills, and the large tile keeps two waves on every SIMD."""
import re

from tests.test_kernel_resources_cpu import _alloc, _kernels


def test_head_kernels_do_not_spill(tmp_path):
    k = _kernels(tmp_path)
    hot = ("gemm_pipe_kernel", "gemm_kernel", "skinny_kernel", "rms_norm_kernel", "rms_norm_bwd_kernel", "join_slices_kernel", "fold_columns_kernel", "align_rows_kernel")
    seen = set()
    for n, v in k.items():
        for h in hot:
            if re.search(r"\d" + h, n):
                seen.add(h)
                assert v["scratch"] == 0, (n, v)
    assert seen == set(hot), set(hot) - seen
    large = [v for n, v in k.items() if "gemm_pipe_kernel" in n]
    # bf16 and f16: two forward forms, two gradients, dx, dw; fp8: the forward forms
    assert len(large) == 14
    for v in large:
        assert _alloc(v["vgpr"]) + _alloc(v["agpr"]) <= 256, v
