"""Continuations of one prompt through the model: forks, steps that read shared pages once, drafted tokens verified and rewound, captured
decoding. What is compared: the same sequences run apart from one another, with logits within the tolerance of the type."""
import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.config.presets import preset_config
from qwenforge_b200.engine.engine import StudentEngine
from qwenforge_b200.engine.model import Model
from qwenforge_b200.sampling import Sampler, SamplingParams
from tests.helpers import CONFIGS, SMALL_64, SMALL_128, assert_logits_close, make_model_dir, random_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def always_shared(monkeypatch):
    """These batches are small: they would mostly be faster apart."""
    monkeypatch.setattr(ops.branches, "SHARED_PAYS_BYTES", 0)
    monkeypatch.setattr(ops.branches, "SHARED_PAYS_PAGES", 0)


def model_of(config, dtype, seed=1):
    folder, _ = make_model_dir(config, seed)
    return Model.from_dir(folder, dtype, "cuda"), folder


@pytest.mark.parametrize("config,dtype", [(SMALL_64, torch.bfloat16), (SMALL_128, torch.bfloat16), (SMALL_64, torch.float32), (CONFIGS["tiny_b"], torch.float32),
                                          (CONFIGS["tiny_w"], torch.float32), (CONFIGS["tiny_w"], torch.bfloat16)])
def test_forked_sequences_step_as_their_own(config, dtype):
    """Forks stepped together, in a shuffled batch with a stranger and a padding entry, against every sequence run by itself."""
    model, _ = model_of(config, dtype)
    vocab = config["vocab_size"]
    prompt, other = random_tokens(vocab, 150, 3), random_tokens(vocab, 40, 4)
    tails = [random_tokens(vocab, 9, 10 + i) for i in range(4)]
    cache = model.new_cache(4096, 8)
    slot, stranger = cache.open(), cache.open()
    model.step(cache, [(slot, prompt), (stranger, other)])
    forks = [slot] + cache.fork(slot, 3)
    shared = cache.shared_prefix([forks[2], -1, stranger, forks[0], forks[3], forks[1]])
    assert shared is not None and shared.groups == [([0, 3, 4, 5], 2)]
    got = {}
    for i in range(9):
        logits = model.step(cache, [(forks[2], [tails[2][i]]), (-1, [0]), (stranger, [tails[0][i]]), (forks[0], [tails[0][i]]), (forks[3], [tails[3][i]]),
                                    (forks[1], [tails[1][i]])])
        for who, row in zip((2, "s", 0, 3, 1), logits):
            got[who, i] = row.clone()
    for who, start, tail in [(f, prompt, tails[f]) for f in range(4)] + [("s", other, tails[0])]:
        alone = model.new_cache(512, 1)
        s = alone.open()
        model.step(alone, [(s, start)])
        for i in range(9):
            assert_logits_close(got[who, i], model.step(alone, [(s, [tail[i]])])[0], dtype, f"sequence {who}, token {i}")
    model.raise_on_kernel_error()


def test_the_layers_run_the_shared_kernel(monkeypatch):
    model, _ = model_of(SMALL_64, torch.bfloat16)
    calls = []
    real = ops.attention_shared
    monkeypatch.setattr(ops, "attention_shared", lambda *a, **k: (calls.append(1), real(*a, **k)))
    cache = model.new_cache(2048, 4)
    slot = cache.open()
    model.step(cache, [(slot, random_tokens(1000, 200, 1))])
    model.step(cache, [(slot, [5])])
    assert not calls
    forks = cache.fork(slot, 2)
    model.step(cache, [(s, [6]) for s in [slot] + forks])
    assert len(calls) == SMALL_64["num_hidden_layers"]
    model.step(cache, [(forks[0], [7])])   # alone it shares nothing with the batch
    assert len(calls) == SMALL_64["num_hidden_layers"]
    monkeypatch.setattr(ops.branches, "SHARED_PAYS_BYTES", 10 ** 9)
    model.step(cache, [(s, [8]) for s in forks])
    assert len(calls) == SMALL_64["num_hidden_layers"]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [True, False])
def test_continuations(dtype, graphs):
    """Every continuation is a draw of its own, and each is the run of its own prompt with its own key; greedy ones are all the same."""
    folder, _ = make_model_dir(SMALL_64, 2)
    engine = StudentEngine(str(folder), dtype=dtype, seed=7, cuda_graphs=graphs)
    prompts = [random_tokens(1000, 140, 5), random_tokens(1000, 33, 6), random_tokens(1000, 64, 8)]
    budgets = [20, 0, 12]
    greedy = engine.generate_ids(prompts, budgets, batch_size=2, ignore_eos=True, continuations=3)
    assert [len(t) for t in greedy] == [20] * 3 + [0] * 3 + [12] * 3
    if dtype == "float32":
        alone = engine.generate_ids(prompts, budgets, batch_size=3, ignore_eos=True)
        assert all(greedy[3 * i + c] == alone[i] for i in range(3) for c in range(3))
        drawn = engine.generate_ids(prompts, budgets, batch_size=3, temperature=0.9, ignore_eos=True, continuations=3)
        many = engine.generate_ids([p for p in prompts for _ in range(3)], [b for b in budgets for _ in range(3)], batch_size=9, temperature=0.9, ignore_eos=True)
        assert drawn == many and len({tuple(t) for t in drawn[:3]}) > 1
    assert not engine.cache.live_slots() and engine.cache.pages_used() == [0] * len(engine.cache.kv_groups)
    if graphs and dtype == "float32":   # another prompt of the same shape replays the graph with its own pages
        kept = dict(engine.graph_decoder.graphs)
        again = [random_tokens(1000, 150, 9)]
        first = engine.generate_ids(again, 20, temperature=0.9, ignore_eos=True, continuations=9)
        many = engine.generate_ids(again * 9, 20, batch_size=9, temperature=0.9, ignore_eos=True)
        assert first == many and len(engine.graph_decoder.graphs) >= len(kept)


def test_continuations_that_do_not_fit_leave_nothing_behind():
    folder, _ = make_model_dir(SMALL_64, 2)
    engine = StudentEngine(str(folder), dtype="bfloat16", max_cache_tokens=1024)
    from qwenforge_b200.cache import CacheFull
    with pytest.raises(CacheFull):
        engine.generate_ids([random_tokens(1000, 300, 5)], 200, ignore_eos=True, continuations=6)
    engine.generate_ids([random_tokens(1000, 300, 5)], 100, ignore_eos=True, continuations=3)
    with pytest.raises(ValueError):
        engine.generate_ids([[1, 2]], 3, continuations=0)
    assert not engine.cache.live_slots()


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_drafted_steps_are_the_same_draws(temperature):
    """Prompt, fork, drafts of unequal counts in one step, verification, rewind, over and over: greedily the tokens are those of plain decoding;
    drawn ones without drafts are the sampler's. The cache stands where the kept tokens end."""
    model, _ = model_of(SMALL_64, torch.float32)
    vocab, prompt, n_new = 1000, random_tokens(1000, 130, 3), 24
    sampler = Sampler(SamplingParams(temperature, 11))
    dev = dict(device="cuda")

    def plain(seq_id):
        cache = model.new_cache(512, 1)
        slot, tokens = cache.open(), []
        logits = model.step(cache, [(slot, prompt)])
        while len(tokens) < n_new:
            out = sampler(logits, torch.tensor([seq_id], **dev), torch.tensor([len(tokens)], dtype=torch.int32, **dev))
            tokens.append(int(out))
            logits = model.step(cache, [(slot, [tokens[-1]])])
        return tokens
    want = [plain(s) for s in range(3)]
    cache = model.new_cache(4096, 4)
    slot = cache.open()
    model.step(cache, [(slot, prompt[:-1])])
    slots = [slot] + cache.fork(slot, 2)
    made, last = [[], [], []], [prompt[-1]] * 3
    turn = 0
    while any(len(m) < n_new for m in made):
        drafts = []
        for s in range(3):
            ahead = want[s][len(made[s]):len(made[s]) + (turn + s) % 4]
            if ahead and (turn + s) % 3 == 0:
                ahead[-1] = (ahead[-1] + 1) % vocab   # a draft that is wrong
            drafts.append(ahead if temperature <= 0 else [])
        logits = model.step(cache, [(slots[s], [last[s]] + drafts[s]) for s in range(3)], want=[range(len(drafts[s]) + 1) for s in range(3)])
        first = torch.tensor([0] + torch.tensor([len(d) + 1 for d in drafts]).cumsum(0).tolist(), dtype=torch.int32, **dev)
        accepted, tokens = sampler.verify(logits, torch.tensor(sum(drafts, []), dtype=torch.int32, **dev), first, 4,
                                          torch.zeros(sum(map(len, drafts)), **dev), None, torch.arange(3, **dev),
                                          torch.tensor([len(m) for m in made], dtype=torch.int32, **dev))
        for s, (kept, row) in enumerate(zip(accepted.tolist(), tokens.tolist())):
            new = [t for t in row if t >= 0]
            assert len(new) == kept + 1 and new[:kept] == drafts[s][:kept]
            made[s] += new
            last[s] = new[-1]
            cache.rewind(slots[s], cache.lengths[slots[s]] - (len(drafts[s]) - kept))
            assert cache.lengths[slots[s]] == len(prompt) + len(made[s]) - 1
        turn += 1
    assert [m[:n_new] for m in made] == want
    model.raise_on_kernel_error()


def test_a_rewound_branch_does_not_touch_the_others():
    model, _ = model_of(SMALL_64, torch.float32)
    cache = model.new_cache(2048, 4)
    slot = cache.open()
    prompt = random_tokens(1000, 100, 1)
    model.step(cache, [(slot, prompt)])
    a, b = cache.fork(slot, 2)
    cache.rewind(a, 70)                       # into the page that all three hold
    model.step(cache, [(a, random_tokens(1000, 60, 2))])
    moved = cache.compact()
    logits = model.step(cache, [(b, [3]), (slot, [3])])
    alone = model.new_cache(512, 1)
    s = alone.open()
    model.step(alone, [(s, prompt)])
    want = model.step(alone, [(s, [3])])[0]
    assert moved >= 0
    for row in logits:
        assert_logits_close(row, want, torch.float32)


def test_a_model_with_a_state_forks_it():
    """Recurrent layers: a fork continues from its parent's state, and neither disturbs the other."""
    model = Model.from_random(preset_config("gatosun-tiny"), 3, "float32")
    vocab = model.spec.vocab_size
    prompt, tails = random_tokens(vocab, 70, 1), [random_tokens(vocab, 5, 2), random_tokens(vocab, 5, 3)]
    cache = model.new_cache(1024, 4)
    slot = cache.open()
    model.step(cache, [(slot, prompt)])
    fork = cache.fork(slot)[0]
    got = [model.step(cache, [(slot, [tails[0][i]]), (fork, [tails[1][i]])]).clone() for i in range(5)]
    for who in (0, 1):
        alone = model.new_cache(256, 1)
        s = alone.open()
        model.step(alone, [(s, prompt)])
        for i in range(5):
            assert_logits_close(got[i][who], model.step(alone, [(s, [tails[who][i]])])[0], torch.float32, f"{who} {i}")
