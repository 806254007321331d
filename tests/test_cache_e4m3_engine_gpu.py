"""A model whose sequence cache is in 8 bits: its logits against the plain model on rounded keys and values, and every way of running it
against the others."""
import pytest
import torch

from qwenforge_b200.engine import Model, StudentEngine
from tests import e4m3_refs as ref
from tests import helpers
from tests import plain_qwen2 as plain

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
CONFIGS = {"tiny_a": helpers.TINY_A, "tiny_w": helpers.TINY_W, "small_64": helpers.SMALL_64, "small_128": helpers.SMALL_128}


def model_of(name, dtype, seed=5, **more):
    folder, weights = helpers.make_model_dir(CONFIGS[name], seed)
    with torch.inference_mode():
        return Model.from_dir(folder, dtype, "cuda", cache_dtype="float8_e4m3", **more), weights


def rounded_rows(rows: torch.Tensor) -> torch.Tensor:
    """[kv heads, positions, dim] in 64 bits -> what a cache holds of them that got them all at once."""
    out = torch.empty_like(rows)
    for h in range(len(rows)):
        for p in range(0, rows.shape[1], 64):
            e = ref.exponent(rows[h, p:p + 64])
            out[h, p:p + 64] = ref.round_code(rows[h, p:p + 64] * 2.0 ** -e) * 2.0 ** e
    return out


@pytest.fixture
def rounding_plain_model(monkeypatch):
    """The plain model with keys and values rounded as the cache rounds them."""
    attention = plain.attention
    monkeypatch.setattr(plain, "attention", lambda q, k, v, window=0: attention(q, rounded_rows(k), rounded_rows(v), window))


@pytest.mark.parametrize("name", list(CONFIGS))
def test_prompts_against_the_plain_model(name, rounding_plain_model):
    """float32: what differs is where a key or value lies next to a rounding border (a step of 2^-3 of it, rarely), beside float32's own error."""
    model, weights = model_of(name, "float32")
    prompts = [helpers.random_tokens(CONFIGS[name]["vocab_size"], n, n) for n in (130, 7, 64)]
    with torch.inference_mode():
        cache = model.new_cache(1024, 4)
        entries = [(cache.open(), p) for p in prompts]
        got = model.step(cache, entries, [list(range(len(p))) for p in prompts]).cpu()
        model.raise_on_kernel_error()
    base = 0
    for p in prompts:
        want = plain.forward_logits(CONFIGS[name], weights, p)
        # a border is met by about 1e-6 / 2^-4 of the elements, some thousands here: at most a few flips, each a change of one element by 2^-3 of
        # itself among the dozens of a head and the positions of a softmax. A hundredth of the logits' size is far above that, and far below
        # what unrounded keys and values give
        bound = 1e-2 * float(want.abs().max())
        assert helpers.max_err(got[base:base + len(p)], want) <= bound
        base += len(p)


@BOTH
@pytest.mark.parametrize("name", list(CONFIGS))
def test_a_sequence_in_pieces(name, dtype):
    """A prompt at once, and the same in spans and single tokens: the same pages but for what growing scales round again, so logits as close as
    8 bits make them."""
    model, _ = model_of(name, dtype)
    tokens = helpers.random_tokens(CONFIGS[name]["vocab_size"], 150, 3)
    with torch.inference_mode():
        cache = model.new_cache(2048, 8)
        whole = model.step(cache, [(cache.open(), tokens)], [[149]]).cpu()
        slot, at = cache.open(), 0
        for n in (100, 3, 1, 1, 30, 9, 1, 1, 1, 1, 1, 1):
            pieces = model.step(cache, [(slot, tokens[at:at + n])]).cpu()
            at += n
        assert at == 150
        model.raise_on_kernel_error()
    # two halves of e4m3's step of 2^-3, each against the logits' size
    assert helpers.max_err(pieces, whole) <= 2.0 ** -3 * float(whole.abs().max())
    plain_model = Model.from_dir(helpers.make_model_dir(CONFIGS[name], 5)[0], dtype, "cuda")
    with torch.inference_mode():
        cache16 = plain_model.new_cache(2048, 8)
        exact = plain_model.step(cache16, [(cache16.open(), tokens)], [[149]]).cpu()
    assert helpers.max_err(whole, exact) <= 2.0 ** -3 * float(exact.abs().max())
    assert cache.kv_groups[0].storage.element_size() == 1 and cache.storage_bytes() > 0
    assert cache.read_bytes([100]) * cache16.kv_groups[0].storage.element_size() == cache16.read_bytes([100])


@BOTH
def test_generation_with_and_without_graphs(dtype):
    folder, _ = helpers.make_model_dir(helpers.SMALL_64, 5)
    prompts = [helpers.random_tokens(1000, n, n) for n in (70, 5, 200)]
    results = []
    for graphs in (True, False):
        engine = StudentEngine(str(folder), device="cuda", dtype=dtype, cuda_graphs=graphs, cache_dtype="float8_e4m3")
        results.append([engine.generate_ids(prompts, 40, batch_size=3, ignore_eos=True) for _ in range(3)])   # (prompt graphs replay from the third on)
        assert engine.cache.kv_dtype is torch.float8_e4m3fn
    assert results[0][0] == results[0][1] == results[0][2] == results[1][0] == results[1][1]
    assert all(len(t) == 40 for t in results[0][0])


@BOTH
def test_continuations_of_a_prompt(dtype):
    """Forks take their page's scales with them: greedy continuations are those of the prompt alone."""
    folder, _ = helpers.make_model_dir(helpers.SMALL_64, 5)
    engine = StudentEngine(str(folder), device="cuda", dtype=dtype, cache_dtype="float8_e4m3")
    prompt = helpers.random_tokens(1000, 400, 9)
    got = engine.generate_ids([prompt], 30, continuations=5, ignore_eos=True)
    assert got == [got[0]] * 5
    drawn = engine.generate_ids([prompt], 12, continuations=5, ignore_eos=True, temperature=1.0, seed=3)
    assert len({tuple(t) for t in drawn}) == 5


def test_forked_rewound_and_compacted():
    model, _ = model_of("small_64", "float32")
    tokens = helpers.random_tokens(1000, 300, 3)
    with torch.inference_mode():
        cache = model.new_cache(4096, 8)
        other, slot = cache.open(), cache.open()
        model.step(cache, [(other, tokens[:130]), (slot, tokens[:100])])
        want_cache = model.new_cache(4096, 8)
        want_slot = want_cache.open()
        model.step(want_cache, [(want_slot, tokens[:100])])
        fork, = cache.fork(slot)
        model.step(cache, [(slot, tokens[200:220])])      # the forked page is the slot's own: the fork's stays
        cache.close(other)
        assert cache.compact() > 0
        model.step(cache, [(fork, tokens[100:103])])
        cache.rewind(fork, 100)
        # the page may keep a larger scale from the tokens that were dropped: those alone decide what the next ones add
        got = model.step(cache, [(fork, tokens[100:101])]).cpu()
        want = model.step(want_cache, [(want_slot, tokens[100:101])]).cpu()
        model.raise_on_kernel_error()
    assert helpers.max_err(got, want) <= 2.0 ** -3 * float(want.abs().max())


def test_the_simt_kernel_and_the_fast_ones():
    tokens = helpers.random_tokens(777, 140, 3)
    logits = []
    for attention in ("auto", "generic"):
        model, _ = model_of("small_128", "float32", attention=attention)
        with torch.inference_mode():
            cache = model.new_cache(2048, 8)
            slot = cache.open()
            model.step(cache, [(slot, tokens[:130])])
            logits.append(torch.cat([model.step(cache, [(slot, tokens[t:t + 2])]).cpu() for t in range(130, 140, 2)]))
    helpers.assert_logits_close(logits[0], logits[1].double(), torch.float32)


def test_a_trace_replayed(tmp_path):
    """`trace_run --cache-dtype`: logits near those of a cache in the model's own type, and not the same."""
    import json
    import numpy as np
    from qwenforge_b200.engine import replay
    folder, _ = helpers.make_model_dir(helpers.SMALL_64, 5)
    lines = [json.dumps({"step": 0, "entries": [{"id": "a", "tokens": helpers.random_tokens(1000, 70, 1), "want": [69]}]}),
             json.dumps({"step": 1, "entries": [{"id": "a", "tokens": [5], "want": [0]}], "end": ["a"]})]
    got = {}
    for dtype in ("auto", "float8_e4m3"):
        args = replay.parse_args(["--model", str(folder), "--dtype", "float32", "--out", str(tmp_path), "--max-tokens", "128", "--cache-dtype", dtype])
        with torch.inference_mode():
            model = Model.from_dir(args.model, args.dtype, args.device, "auto", args.cache_dtype)
            replay.replay(model, model.new_cache(1024, 4), lines, tmp_path, report=lambda text: None)
        got[dtype] = np.fromfile(tmp_path / "1.f32", dtype="<f4")
    off = np.abs(got["auto"] - got["float8_e4m3"]).max()
    assert 0 < off <= 2.0 ** -3 * np.abs(got["auto"]).max()
