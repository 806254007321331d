"""`ops.attention_shared` where members of a group stand inside its pages: what lies behind their own position, whatever it holds, is not theirs."""
import math

import pytest
import torch

from tests.test_attention_shared_gpu import PAGE, TILED, Batch, tiled

pytestmark = pytest.mark.gpu
SMALL = [((14, 2, 64), torch.bfloat16), ((6, 3, 96), torch.bfloat16), ((4, 2, 32), torch.bfloat16), ((16, 2, 128), torch.bfloat16), ((14, 2, 64), torch.float32),
         ((3, 1, 23), torch.bfloat16), ((2, 1, 200), torch.float32)]


def spoil(b, entry, begin, end):
    """Positions begin .. end - 1 of a sequence: keys of NaN, values of NaN and infinity."""
    for p in range(begin, end):
        page = int(b.table_cpu[b.slots_cpu[entry], p // PAGE])
        b.storage[page, 0, :, p % PAGE] = math.nan
        b.storage[page, 1, :, p % PAGE] = math.nan if p % 2 else math.inf


@pytest.mark.parametrize("shape,dtype", SMALL)
def test_members_inside_pages_that_nobody_sees_the_end_of(shape, dtype):
    b = Batch([([0, 1, 2, 3], 5)], [1, 1, 1, 70, 30], *shape, dtype)
    positions = [130, 0, 190, 63]
    b.tok_pos[:4] = torch.tensor(positions, dtype=torch.int32)
    spoil(b, 0, 191, 5 * PAGE)
    b.run()
    b.check()


@pytest.mark.parametrize("shape,dtype", SMALL)
def test_a_member_inside_pages_that_others_see(shape, dtype):
    """Values behind its position that are no numbers: the others' outputs are none either, its own is."""
    b = Batch([([0, 1, 2], 5)], [9, 9, 70], *shape, dtype)
    b.tok_pos[1] = 130
    spoil(b, 0, 131, 140)
    b.run()
    assert torch.isnan(b.out[0].float()).any() and torch.isnan(b.out[2].float()).any()
    assert torch.isfinite(b.out[1]).all()
    b.idle = {0, 2}
    b.out[[0, 2]] = 0
    b.check()


@pytest.mark.parametrize("shape", TILED)
def test_members_inside_the_pages_of_tiles(shape):
    b = tiled(shape)
    inside = {0: 0, 3: 5 * PAGE + 3, 11: 20 * PAGE + 63, 12: 51 * PAGE, 14: 64}
    for e, pos in inside.items():
        b.tok_pos[e] = pos
    spoil(b, 0, 20 * PAGE + 64, 20 * PAGE + 70)   # seen by the first group's others
    spoil(b, 14, 65, 2 * PAGE)                    # seen by sequence 15
    lost = {2, 4, 5, 8, 9, 10, 15}
    b.run()
    for e in lost:
        assert torch.isnan(b.out[e].float()).any()
    b.idle = lost
    b.out[list(lost)] = 0
    b.check()


@pytest.mark.parametrize("shape", TILED)
def test_all_members_inside_the_pages_of_tiles(shape):
    b = tiled(shape, [(list(range(10)), 40)], [1] * 10)
    b.tok_pos.copy_(torch.tensor([30 * PAGE - 1 - 97 * e for e in range(10)], dtype=torch.int32))
    spoil(b, 0, 30 * PAGE, 40 * PAGE)
    b.run()
    b.check()


@pytest.mark.parametrize("shape", TILED)
def test_members_at_the_end_of_the_shared_pages(shape):
    """Nothing of their own: there are no records beside the tiles'."""
    b = tiled(shape, [(list(range(10)), 40)], [1] * 10)
    b.tok_pos.fill_(40 * PAGE - 1)
    b.run()
    b.check()
