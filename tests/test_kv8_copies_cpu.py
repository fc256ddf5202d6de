"""Block copies of the 8-bit cache: what they refuse."""
import pytest
import torch

from kharon_b200 import ops


def test_block_copies_refuse_pairs_that_a_kernel_would_misread():
    """Pairs are read as they lie in memory: a strided list would name other blocks.  Either shape of a contiguous one, and pairs out of range."""
    kv = torch.randint(0, 255, (2, 6, 2, ops.kv8_record_bytes(4, 16)), dtype=torch.uint8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    for bad in (i32([[0, 9, 2], [1, 9, 3]])[:, ::2], i32([0, 9, 2, 9, 1, 9, 3, 9])[::2], i32([[0, 1], [2, 3]]).t()):
        with pytest.raises(ValueError):
            ops.copy_blocks8(kv, bad, 2)
    with pytest.raises(ValueError):
        ops.copy_blocks8(kv, i32([0, 2]), -1)
    before = kv.clone()
    for bad in ([0, 6], [-1, 2], [1, 2, 6, 3]):
        with pytest.raises(IndexError):
            ops.copy_blocks8(kv, i32(bad), len(bad) // 2)
    assert torch.equal(kv, before)
    ops.copy_blocks8(kv, i32([[0, 2], [1, 3]]), 2)
    assert torch.equal(kv[:, 2:4], before[:, :2]) and torch.equal(kv[:, 4:], before[:, 4:])
