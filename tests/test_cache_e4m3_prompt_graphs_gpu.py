"""Steps of several tokens replayed from graphs over a cache in 8 bits: a graph serves every length of its shape."""
import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.engine import Model
from tests import helpers
from tests.test_cache_e4m3_gpu import Case

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


@pytest.mark.parametrize("name,spans", [("small_64", [5] * 12), ("small_64", [2, 3, 4, 5, 6, 9, 17, 18] * 4), ("small_64", [19, 30, 31] * 4), ("small_128", [5, 4] * 8), ("small_128", [33, 60] * 4),
                                        ("tiny_a", [3, 7] * 8), ("tiny_w", [3, 7] * 8)])
def test_short_spans_go_the_same_way(monkeypatch, name, spans):
    """A replayed step attends over codes where the step itself does, and reads them back where it does: what fills its shape up decides nothing."""
    config = CONFIGS[name]
    folder, _ = helpers.make_model_dir(config, 5)
    ways = []
    for entry in ("attention_e4m3", "cache_read_e4m3"):
        def watched(*args, entry=entry, run=getattr(ops, entry), **more):
            ways.append(entry)
            return run(*args, **more)
        monkeypatch.setattr(ops, entry, watched)
    logits, taken = [], []
    for graphs in (False, True):
        with torch.inference_mode():
            model = Model.from_dir(folder, "bfloat16", "cuda", cache_dtype="float8_e4m3")
        model.enable_prefill_graphs(graphs)
        ways.clear()
        logits.append(in_pieces(model, config, 70, spans))
        taken.append(set(ways[config["num_hidden_layers"]:]))   # (behind the prompt's)
    assert taken[0] == taken[1] and model.prefill_graphs.replays > 0
    group = config["num_attention_heads"] // config["num_key_value_heads"]
    assert taken[0] == {"attention_e4m3" if ops.attention_e4m3_pays(torch.bfloat16, n, group) else "cache_read_e4m3" for n in spans}
    for at, (want, got) in enumerate(zip(*logits)):
        assert helpers.max_err(got, want) <= SHARE * float(want.abs().max()), f"span {at}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("most", [2, 5, 16, 20])
def test_a_padding_entry_longer_than_the_spans(most, dtype):
    """It changes no result, is not reported, and is attended to as zeros."""
    live = [(60, most), (3, 1), (200, 2)]
    with_padding, without = Case(live + [(0, 120, True)], 14, 2, 64, dtype, seed=3), Case(live, 14, 2, 64, dtype, seed=3)
    outs = []
    for c in (with_padding, without):
        c.most = most
        n = without.cu_q[-1]
        qkv = torch.zeros((c.cu_q[-1], c.qkv.shape[1]), dtype=dtype)
        qkv[:n] = without.qkv
        c.bias = without.bias
        # the same pages under the same sequences
        for s in range(len(live)):
            for p in range(-(-sum(live[s]) // 64)):
                a, b = int(c.table[c.slots[s], p]), int(without.table[without.slots[s], p])
                c.storage[a] = without.codes[b].cuda()
                c.held_scales[a] = without.scales[b].cuda()
        q = c.write(qkv.cuda())
        out = torch.full_like(q, 9.0)
        ops.attention_e4m3(q, out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, c.heads, c.n, most, 0.125, 0, ops.E4m3Scratch("cuda"), c.err)
        assert int(c.err) == 0
        pages = torch.cat([c.storage[int(c.table[c.slots[s], p])].float() for s in range(len(live)) for p in range(-(-sum(live[s]) // 64))])
        outs.append((q[:n].clone(), out[:n].clone(), pages))
        assert not bool(out[n:].any())
    for a, b in zip(*outs):
        assert torch.equal(a, b)
