"""Workspaces of the attention over a cache in 8 bits."""
import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.engine import Model
from tests import helpers
from tests.test_attention_e4m3_gpu import check, query, run
from tests.test_cache_e4m3_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_longer_sequences_and_larger_batches_need_no_more(tokens, dtype):
    """What the first call allocates serves every other of its head size and rows."""
    scratch = ops.E4m3Scratch("cuda")
    held = None
    for entries in ([(10, tokens)], [(300, tokens)], [(700, tokens)], [(5000, tokens)], [(5000, tokens), (20, tokens)], [(900, tokens)] * 30, [(3000, tokens)] * 8):
        c = Case(entries, 14, 2, 64, dtype, seed=3)
        q = query(c)
        check(c, q, run(c, q, scratch=scratch))
        now = (scratch.part_o, scratch.part_ml, scratch.tickets)
        held = held or now
        assert all(a is b for a, b in zip(held, now)) and not scratch.outgrown


def test_a_sequence_that_grows_launch_by_launch():
    """A model's memory stays where it is while its sequences grow."""
    folder, _ = helpers.make_model_dir(helpers.SMALL_64, 5)
    with torch.inference_mode():
        model = Model.from_dir(folder, "bfloat16", "cuda", cache_dtype="float8_e4m3")
        cache = model.new_cache(4096, 4)
        slot = cache.open()
        model.step(cache, [(slot, helpers.random_tokens(1000, 30, 1))])   # (too long a span to attend over codes)
        model.step(cache, [(slot, [5])])
        scratch = model.codes_scratch
        held, sizes = len(scratch.outgrown), (scratch.part_o.numel(), scratch.part_ml.numel())
        for n in (250, 1, 250, 1, 250, 1, 250, 1, 250, 1):
            model.step(cache, [(slot, helpers.random_tokens(1000, n, n))])
        model.raise_on_kernel_error()
        assert (len(scratch.outgrown), scratch.part_o.numel(), scratch.part_ml.numel()) == (held, *sizes)
