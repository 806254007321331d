"""The calls as a model's step makes them (`constants`): kernels that begin while the one ahead still runs read lengths, tables and older pages then, and the rest
behind it. Bit by bit what the same calls give one after another."""
import pytest
import torch

from qwenforge_b200 import ops
from tests.test_attention_e4m3_gpu import SPANS, TOKENS
from tests.test_cache_e4m3_gpu import ENTRIES, Case

pytestmark = pytest.mark.gpu
LONG = [(4000, 1), (63, 1), (2111, 1), (64, 1)]
CALLS = {"tokens": TOKENS, "spans": SPANS, "prompts": ENTRIES["prompts"], "long": LONG, "many": [(7 * s, 1) for s in range(90)], "long spans": [(3000, 5), (126, 40), (640, 3)]}


def step(c, qkv, bias, freq, q, out, scratch, window, constants):
    """What a layer does behind its product: queries, keys and values written, attention over them. The keys and values are far larger than what the pages
    hold, so that a page with older rows gets another scale just before it is read."""
    ops.rope_cache_write_e4m3(qkv, c.dev["cu_q"], c.dev["tok_seq"], c.dev["tok_pos"], c.dev["slots"], freq, c.rot_dim, c.heads, q, c.site, c.most, c.err, bias=bias,
                              constants=constants)
    ops.attention_e4m3(q, out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, c.heads, c.n, c.most, c.dim ** -0.5, window, scratch, c.err, constants=constants)


@pytest.mark.parametrize("entries", list(CALLS))
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (16, 2, 128), (6, 3, 96), (4, 2, 16)])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_a_step_with_and_without_constants(entries, heads, kv_heads, dim, window, dtype):
    c = Case(CALLS[entries], heads, kv_heads, dim, dtype, seed=dim, spread=500.0)
    raw, scales = c.raw.clone(), c.held_scales.clone()
    qkv, bias, freq = c.qkv.cuda(), c.bias.cuda(), c.inv_freq.cuda()
    scratch = ops.E4m3Scratch("cuda")
    results = []
    for constants in (False,) + (True,) * 6:
        q, out = torch.empty((len(qkv), heads * dim), dtype=dtype, device="cuda"), torch.full((len(qkv), heads * dim), 9.0, dtype=dtype, device="cuda")
        c.raw.copy_(raw)
        c.held_scales.copy_(scales)
        source = qkv.clone()
        torch.cuda.synchronize()
        if constants:
            torch.cuda._sleep(300_000)   # (both calls wait in the stream, so that the second one begins as soon as the first lets it)
        step(c, source, bias, freq, q, out, scratch, window, constants)
        torch.cuda.synchronize()
        results.append((q, out, c.raw.clone(), c.held_scales.clone()))
    assert bool((results[0][3] > scales).any()) and int(c.err) == 0
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_layers_behind_one_another(dtype):
    """Captured: product, write, attention, product, ..., over the same tokens, each layer with a cache of its own and one workspace for all."""
    layers, dim, heads = 6, 64, 8
    cases = [Case([(500, 1), (63, 1), (64, 1), (1300, 1)], heads, 2, dim, dtype, seed=i, spread=500.0) for i in range(layers)]
    for c in cases[1:]:   # (one set of lengths, as a step has)
        assert c.cu_q == cases[0].cu_q
    scratch, g = ops.E4m3Scratch("cuda"), torch.Generator().manual_seed(0)
    products = [torch.randn((heads * dim, 12 * dim), generator=g).to(device="cuda", dtype=dtype) for _ in cases]
    start, freq = cases[0].qkv[:, :heads * dim].cuda().contiguous(), cases[0].inv_freq.cuda()
    held = [(c.raw.clone(), c.held_scales.clone()) for c in cases]
    biases = [c.bias.cuda() for c in cases]

    def run(constants):
        x = start
        for c, w, b in zip(cases, products, biases):
            qkv, q, out = x @ w, torch.empty_like(x), torch.empty_like(x)
            step(c, qkv, b, freq, q, out, scratch, 0, constants)
            x = out
        return x

    def reset():
        for c, (raw, scales) in zip(cases, held):
            c.raw.copy_(raw)
            c.held_scales.copy_(scales)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):   # (the workspaces, and the library's)
        run(False)
    torch.cuda.synchronize()
    reset()
    want = run(False).clone()
    pages = [(c.raw.clone(), c.held_scales.clone()) for c in cases]
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = run(True)
    for _ in range(10):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert all(torch.equal(c.raw, raw) and torch.equal(c.held_scales, scales) for c, (raw, scales) in zip(cases, pages))
    assert all(int(c.err) == 0 for c in cases)
