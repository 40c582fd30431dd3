"""Numbers of rows at the ends of what a selection takes."""
import pytest
import torch


@pytest.mark.parametrize("shape", [(2 ** 31, 1), (2 ** 32 + 5, 1), (2 ** 20, 2 ** 12, 2)])
def test_rows_that_32_bits_do_not_count_are_refused(shape):
    """The number of rows is 32 bits in the kernels: 2^32 + 5 of them were 5."""
    import memory_b200 as M
    with pytest.raises(ValueError, match="rows in one call"):
        M.select_chapters(torch.empty(shape, device="meta", dtype=torch.bfloat16), 1)
    with pytest.raises(ValueError, match="CUDA"):
        M.select_chapters(torch.empty(2 ** 31 - 1, 1, device="meta"), 1)
