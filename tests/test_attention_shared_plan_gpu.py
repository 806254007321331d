"""How `ops.attention_shared` cuts a step's work: the parts that it leaves for its join."""
import pytest
import torch

from qwenforge_b200 import ops
from tests.test_attention_shared_gpu import PAGE, TILED, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", TILED)
def test_steps_without_tiles_use_every_sm(shape):
    """A graph's bound asks for the tiles' kernel; what is shared now is too little for them. Every page of a sequence's own is then cut to a part of its own,
    as there are warps for (17 sequences x 11 pages x 2 tiles of rows, or 4 of them with two kv heads, are 374; ten warps an SM are 1,480)."""
    groups, own = [(list(range(10)), 1), ([10, 11, 12], 1)], [10 * PAGE + 7 + e for e in range(17)]
    b = Batch(groups, own, *shape, torch.bfloat16)
    share = ops.SharedPrefix(groups, b.n, "cuda", bound_pages=256)
    b.run(share=share)
    b.check()
    parts = (b.scratch.part_n[:b.n] >> 16).tolist()   # (a page that is shared is a part more)
    assert parts == [12] * 13 + [11] * 4
