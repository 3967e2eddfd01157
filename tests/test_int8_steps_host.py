"""What a cache publishes for a step, on the host."""
import pytest
import torch


def test_row_starts_of_a_step_are_published():
    """The rows of a padded step begin at multiples of its tokens; a step that is refused leaves them as they were."""
    from nkipy_amd.engine import OutOfBlocks, PagedKVCache
    c = PagedKVCache(8, 16, 2, 64, max_seqs=3, max_blocks_per_seq=4, dtype=torch.int8, device="cpu")
    c.begin_step([20, 0, 7], 20)
    assert c.query_starts.tolist() == [0, 20, 40, 60] and c.row_starts.tolist() == [0, 20, 20, 27]
    with pytest.raises(OutOfBlocks):
        c.begin_step([30, 30, 50], 50)
    c.release(1)
    assert c.query_starts.tolist() == [0, 20, 40, 60]
    c.begin_step([0, 5, 3], 5)
    assert c.query_starts.tolist() == [0, 5, 10, 15] and c.row_starts.tolist() == [0, 0, 5, 15]
    assert PagedKVCache(8, 16, 2, 64, max_seqs=3, max_blocks_per_seq=4, device="cpu").query_starts is None
