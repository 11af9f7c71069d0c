"""What the compiler gave the kernels of serving over 8-bit pages (no GPU needed)."""
import pytest

from tests.test_kernel_resources import built  # noqa: F401

pytest.importorskip("msgpack")


@pytest.mark.parametrize("name,count", [("paged_q8_few", 6), ("paged_q8_many", 6), ("qk_q8_kernel", 24),
                                        ("values_q8_kernel", 1), ("logprobs_row_kernel", 3), ("logprobs_slice_kernel", 6),
                                        ("logprobs_join_kernel", 6), ("block_norm_kernel", 16)])
def test_no_registers_spill(built, name, count):  # noqa: F811
    """A reload inside attention's key loop would wait for the step's own loads to LDS, which the compiler does not count."""
    mine = {n: k for n, k in built.items() if name in n}
    assert len(mine) == count
    for n, k in mine.items():
        assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] == 0, n
