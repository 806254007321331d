"""Steps of several tokens replayed from graphs over a cache in 8 bits: a graph serves every length of its shape."""
import pytest
import torch

from qwenforge_b200.engine import Model
from tests import helpers

pytestmark = pytest.mark.gpu
CONFIGS = {"tiny_a": helpers.TINY_A, "tiny_w": helpers.TINY_W, "small_64": helpers.SMALL_64, "small_128": helpers.SMALL_128}


def in_pieces(model, config, first, spans, seed=3):
    """Logits of every span's tokens behind a prompt of `first`, two sequences a step (the second one 11 tokens behind the first)."""
    tokens = helpers.random_tokens(config["vocab_size"], first + sum(spans), seed)
    got = []
    with torch.inference_mode():
        cache = model.new_cache(4096, 4)
        a, b = cache.open(), cache.open()
        model.step(cache, [(a, tokens[:first]), (b, tokens[:first - 11])])
        at = first
        for n in spans:
            got.append(model.step(cache, [(a, tokens[at:at + n]), (b, tokens[at - 11:at - 11 + n])], [list(range(n))] * 2).cpu())
            at += n
            model.raise_on_kernel_error()
    return got


# Both runs are the same sums in other orders, over pages that hold the same but for codes next to a rounding border: a key's or value's last bit of bfloat16 (2^-8) moves
# one code in some hundreds by 2^-3 of itself. Together below a hundredth of the logits' size; a page left out changes them by their whole size.
SHARE = 2.0 ** -5


@pytest.mark.parametrize("name", list(CONFIGS))
def test_continuations_past_many_page_borders(name):
    """Thirty tokens at a time, always the same rounded shape: what was captured at a few pages is replayed at more, past the bound on the lengths, too."""
    config = CONFIGS[name]
    folder, _ = helpers.make_model_dir(config, 5)
    first = 70
    spans = [30] * min(19, (config["max_position_embeddings"] - first) // 30)
    logits = []
    for graphs in (False, True):
        with torch.inference_mode():
            model = Model.from_dir(folder, "bfloat16", "cuda", cache_dtype="float8_e4m3")
        model.enable_prefill_graphs(graphs)
        logits.append(in_pieces(model, config, first, spans))
    assert model.prefill_graphs.replays >= len(spans) - 4   # (a shape of each bound on the lengths runs launch by launch once)
    for at, (want, got) in enumerate(zip(*logits)):
        assert helpers.max_err(got, want) <= SHARE * float(want.abs().max()), f"span {at}"
