"""BatchInfo.with_trees looks at its arguments before anything asks for a device."""
import pytest
import torch

from aici_amd import paged


@pytest.mark.parametrize("count", [0, 1, 4, 6, 7])
def test_a_parent_for_every_row(count):
    """Five rows of two trees and a decode row: five parents, not one for all of them, nor one for the decode row."""
    alloc = paged.BlockAllocator(16, 20)
    builder = paged.BatchInfoBuilder(16, 256, 1)
    for sid, n in ((1, 3), (2, 2), (3, 1)):
        alloc.alloc_seq(sid, 20 + n)
        builder.sched_out(alloc, sid, list(range(20 + n)), 20)
    batch = builder.finish()
    assert batch.q_multi == 5 and batch.tokens.numel() == 6
    with pytest.raises(ValueError, match=f"{count} parents for 5 rows"):
        batch.with_trees(torch.full((count,), -1, dtype=torch.int32))
    with pytest.raises(ValueError, match="parents for 5 rows"):
        batch.with_trees(torch.full((5, 1), -1, dtype=torch.int32))
