"""What the adapters' calls keep in their caller's workspace, by the sizes that nlgpu reports (no device)."""
import pytest

import nlgpu


# (rows, out, cols; the slices of the projection's columns and the tiles they share)
@pytest.mark.parametrize("seq,out,cols,slices,tiles", [(333, 300, 4352, 4, 22), (128, 2560, 6912, 4, 40),
                                                       (512, 2560, 4096, 3, 160), (100, 13824, 4096, 1, 0),
                                                       (333, 300, 2560, 1, 0), (40, 300, 4352, 1, 0)])
def test_the_column_split_is_in_the_workspace(seq, out, cols, slices, tiles):
    """Sums of 256 x 32 values a slice and tile and 256 counters, beside the rows as int8: nothing of a split launch is
    the library's, whose scratch two replayed graphs would share."""
    rest = nlgpu.ternary_linear_lora_workspace(seq, out, cols, 8, 4) - nlgpu.lora_linear_workspace(seq, out, cols, 8, 4)
    rows = seq * cols + 4 * seq
    split = 1024 + slices * tiles * 32768 if slices > 1 else 0
    assert rows + split <= rest <= rows + split + 1024
