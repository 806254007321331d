"""`SharedPrefix.load`: what is shared now under a graph that was captured before stays within the page table that the graph reads."""
import pytest
import torch

from qwenforge_b200 import ops


def test_no_more_pages_than_the_page_table_has_room_for():
    share = ops.SharedPrefix([([0, 1], 3)], 2, "cpu", bound_pages=64)
    share.load(ops.SharedPrefix([([0, 1], 20)], 2, "cpu"))   # (no call has read a table with it yet)
    share.load(ops.SharedPrefix([([1, 0], 3)], 2, "cpu"))
    i32 = torch.zeros(3, dtype=torch.int32)
    site = ops.KvSiteArgs(torch.zeros(2, 2, 1, 64, 32), torch.zeros(2, 8, dtype=torch.int32), 1, 32)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.attention_shared(torch.zeros(2, 32), torch.zeros(2, 32), i32, i32[:2], i32[:2], site, 1, 2, 1.0, share, ops.SharedScratch("cpu"), i32[:1])
    with pytest.raises(ops.KernelError, match="page table"):
        share.load(ops.SharedPrefix([([0, 1], 9)], 2, "cpu"))
    assert share.pages.tolist() == [3] and share.members.tolist() == [1, 0]
    share.load(ops.SharedPrefix([([0, 1], 8)], 2, "cpu"))
    assert share.pages.tolist() == [8] and share.entry_pages.tolist() == [8, 8] and share.members.tolist() == [0, 1]
