"""Registers and scratch of the paged cache's kernels, read from the built library's metadata."""
from test_kernel_resources import kernels  # noqa: F401  (the fixture)

NAMES = ("block_tables_kernel", "qk_norm_rope_kernel", "page_bounds_kernel", "paged_whole_kernel", "paged_parts_kernel",
         "paged_scan_kernel", "paged_join_kernel", "page_score_kernel", "page_select_kernel")


def test_cache_kernels_keep_their_values_in_registers(kernels):  # noqa: F811
    for want in NAMES:
        found = {k: v for k, v in kernels.items() if want in k}
        assert found, want
        for name, (_, scratch) in found.items():
            assert scratch == 0, (name, scratch)


def test_two_attention_blocks_fit_a_cu(kernels):  # noqa: F811
    """Two blocks of four waves a CU: at most 256 of a lane's 512 registers each."""
    found = {k: v for k, v in kernels.items() if "paged_whole_kernel" in k or "paged_parts_kernel" in k}
    assert len(found) == 6 + 12
    for name, (registers, _) in found.items():
        assert registers <= 256, (name, registers)
