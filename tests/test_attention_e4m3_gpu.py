"""Attention over a sequence cache in 8 bits against the plain implementation in 64 bits, with the tolerance of `e4m3_refs.attend_tolerance`."""
import numpy as np
import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.ops import KernelError
from tests import e4m3_refs as ref
from tests.test_cache_e4m3_gpu import PAGE, Case

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])


def query(c, spread=0.4, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn((c.cu_q[-1], c.heads * c.dim), generator=g)).to(c.dtype)


def run(c, q, window=0, scratch=None, max_kv_len=None, out=None):
    out = torch.full(q.shape, 9.0, dtype=c.dtype, device="cuda") if out is None else out
    scratch = scratch or ops.E4m3Scratch("cuda")
    ops.attention_e4m3(q.cuda(), out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, c.heads, c.n, c.most, c.dim ** -0.5, window, scratch, c.err, max_kv_len)
    assert scratch.tickets is None or not bool(scratch.tickets.any())
    return out


def check(c, q, got, window=0):
    values = c.storage.cpu().double() * c.held_scales.cpu().double()[..., None, None]
    want, size, far = ref.attend(q, c.cu_q, c.tok_pos, c.slots, values, c.table, c.heads, c.dim ** -0.5, window)
    off = (got.cpu().double().view(want.shape) - want).abs() - ref.attend_tolerance(want, size, far, c.dtype)
    assert bool((off <= 0).all()), f"{float(off.max())} beyond the tolerance"
    assert int(c.err) == 0


SHAPES = [(14, 2, 64), (28, 4, 128), (16, 2, 128), (4, 2, 16), (6, 3, 96), (5, 5, 80), (3, 1, 48), (2, 1, 112), (8, 1, 32), (40, 2, 64), (33, 1, 32)]
TOKENS = [(0, 1), (63, 1), (64, 1), (500, 1), (1, 1), (0, 1, True), (1300, 1), (127, 1), (31, 1), (32, 1)]
SPANS = [(0, 5), (62, 4), (700, 3), (3, 1), (120, 9), (0, 2, True), (191, 2)]


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@BOTH
def test_single_tokens(heads, kv_heads, dim, dtype):
    c = Case(TOKENS, heads, kv_heads, dim, dtype, seed=dim + heads)
    q = query(c)
    got = run(c, q)
    check(c, q, got)
    assert torch.equal(run(c, q, max_kv_len=1301), got)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@BOTH
def test_spans(heads, kv_heads, dim, dtype):
    c = Case(SPANS, heads, kv_heads, dim, dtype, seed=dim + heads)
    q = query(c)
    check(c, q, run(c, q))


@pytest.mark.parametrize("window", [1, 5, 37, 64, 100, 1000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (4, 2, 128), (6, 3, 16)])
@BOTH
def test_windows(window, heads, kv_heads, dim, dtype):
    for entries in (TOKENS, SPANS):
        c = Case(entries, heads, kv_heads, dim, dtype, seed=window)
        for s, slot in enumerate(c.slots):   # pages that have left the window are not held
            if slot >= 0 and c.cu_q[s + 1] > c.cu_q[s]:
                c.dev["table"][slot, :max(0, int(c.tok_pos[c.cu_q[s]]) - window + 1) // PAGE] = -1
        q = query(c)
        check(c, q, run(c, q, window), window)


@pytest.mark.parametrize("length", [4096, 20000])
@pytest.mark.parametrize("alone", [True, False])
@BOTH
def test_a_long_sequence(length, alone, dtype):
    """One of many runs, beside short ones or by itself."""
    c = Case([(length, 1)] + ([] if alone else [(s, 1) for s in range(0, 150, 10)]), 4, 2, 64, dtype, seed=6)
    q = query(c)
    got = run(c, q)
    check(c, q, got)
    for _ in range(5):
        assert torch.equal(run(c, q), got)   # runs are joined in their order, whichever block ends last


def test_more_sequences_than_blocks():
    c = Case([(int(x), 1) for x in np.random.default_rng(0).integers(0, 200, 600)], 8, 4, 32, torch.bfloat16, seed=6)
    q = query(c)
    check(c, q, run(c, q))


def test_entries_without_tokens():
    c = Case([(0, 1), (30, 0), (70, 2), (0, 0), (5, 1)], 4, 2, 64, torch.bfloat16, seed=6)
    q = query(c)
    check(c, q, run(c, q))


@pytest.mark.parametrize("tokens", [TOKENS, SPANS], ids=["tokens", "spans"])
@BOTH
def test_what_lies_behind_a_sequence_is_not_read(tokens, dtype):
    """NaN codes behind the last position, and before the window, of pages that are read."""
    for window in (0, 37):
        c = Case(tokens, 4, 2, 64, dtype, seed=8)
        q = query(c)
        got = run(c, q, window)
        raw = c.storage.view(torch.uint8)
        for s, slot in enumerate(c.slots):
            if slot < 0:
                continue
            first, last = int(c.tok_pos[c.cu_q[s]]), int(c.tok_pos[c.cu_q[s + 1] - 1])
            raw[int(c.table[slot, last // PAGE]), :, :, last % PAGE + 1:] = 0x7f
            lo = max(0, first - window + 1) if window else 0
            raw[int(c.table[slot, lo // PAGE]), :, :, :lo % PAGE] = 0xff
        assert torch.equal(run(c, q, window), got)


@BOTH
def test_a_token_of_a_span_does_not_see_the_next_ones_nan(dtype):
    c = Case([(60, 8), (3, 5), (0, 1)], 10, 2, 64, dtype, seed=8)
    q = query(c)
    for window in (0, 3):
        clean = run(c, q, window)
        raw = c.storage.view(torch.uint8)
        keep = raw.clone()
        page = int(c.table[c.slots[0], 1])
        raw[page, 1, 1, 1] = 0x7f                # position 65, values of the second kv head: tokens 5 and later of the first entry see it
        raw[int(c.table[c.slots[1], 0]), 0, 0, 6] = 0xff   # position 6, keys of the first: tokens 3 and later of the second
        got = run(c, q, window).view(-1, 2, 5, 64)
        raw.copy_(keep)
        clean = clean.view(got.shape)
        seen = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
        seen[5:8, 1] = seen[11:13, 0] = True     # (all of them within a window of 3)
        assert bool(torch.isnan(got[seen]).all()) and torch.equal(got[~seen], clean[~seen])


@BOTH
def test_scales_far_apart(dtype):
    """A page of huge values that no query looks at beside one of tiny values that all of them do, and the other way round."""
    for low, high in ((-100, 20), (20, -100), (-112, 60), (-112, 119), (119, -112)):
        c = Case([(200, 1), (400, 2)], 4, 2, 64, dtype, seed=3, low=-10)
        for s in range(2):
            for p in range(4):
                page = int(c.table[c.slots[s], p])
                c.held_scales[page, 1] = 2.0 ** (low if p % 2 else high)
        q = query(c)
        check(c, q, run(c, q))


@pytest.mark.parametrize("spread", [0.0, 1e-20, 50.0, 1e15])
@BOTH
def test_queries_of_any_size(spread, dtype):
    c = Case(TOKENS[:5], 4, 2, 64, dtype, seed=3)
    if spread == 1e15:   # (scores as always, from keys as small as queries are large)
        c.held_scales[:, 0] = 2.0 ** -56
    q = query(c, spread)
    check(c, q, run(c, q))


def test_a_query_that_is_not_finite_stays_alone():
    c = Case(TOKENS[:5], 4, 2, 64, torch.bfloat16, seed=3)
    q = query(c)
    want = run(c, q).view(-1, 4, 64)
    q[1, 64] = float("nan")
    got = run(c, q).view(-1, 4, 64)
    assert bool(torch.isnan(got[1, 1]).all())
    got[1, 1] = want[1, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [0.0, -0.125])
@BOTH
def test_a_scale_of_zero_or_less(scale, dtype):
    c = Case(TOKENS[:5], 4, 2, 64, dtype, seed=3)
    q = query(c)
    out = torch.empty_like(q, device="cuda")
    ops.attention_e4m3(q.cuda(), out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, 4, c.n, 1, scale, 0, ops.E4m3Scratch("cuda"), c.err)
    values = c.storage.cpu().double() * c.held_scales.cpu().double()[..., None, None]
    want, size, far = ref.attend(q, c.cu_q, c.tok_pos, c.slots, values, c.table, 4, scale, 0)
    assert bool(((out.cpu().double().view(want.shape) - want).abs() <= ref.attend_tolerance(want, size, far.abs(), dtype)).all()) and int(c.err) == 0


def test_entries_longer_than_the_call_says():
    c = Case([(10, 9), (30, 2)], 10, 2, 64, torch.bfloat16, seed=3)
    c.most = 3
    run(c, query(c))
    assert int(c.err) == ops.ERR_ROW_RANGE
    c = Case([(10, 2), (30, 0)], 10, 2, 64, torch.bfloat16, seed=3)   # two tokens of two entries, but not one each
    c.most = 1
    run(c, query(c))
    assert int(c.err) & ops.ERR_ROW_RANGE


def test_pages_that_are_not_held_and_lengths_beyond_the_bound():
    c = Case([(200, 1), (10, 1)], 4, 2, 64, torch.bfloat16, seed=3)
    q = query(c)
    c.dev["table"][c.slots[0], 1] = -1
    run(c, q)
    assert int(c.err) == ops.ERR_NO_PAGE
    c = Case([(200, 1), (10, 1)], 4, 2, 64, torch.bfloat16, seed=3)
    run(c, q, max_kv_len=70)
    assert int(c.err) == ops.ERR_POSITION_RANGE
    c = Case([(200, 1), (10, 1)], 4, 2, 64, torch.bfloat16, seed=3)
    c.dev["tok_pos"][0] = 64 * c.table.shape[1] + 5   # behind the page table's last column
    run(c, q)
    assert int(c.err) & (ops.ERR_NO_PAGE | 32)


@BOTH
def test_as_many_rows_as_entries_but_not_one_each(dtype):
    """An entry without a token, and a row behind the last entry, which stays as it is."""
    c = Case([(700, 1), (90, 0), (300, 1), (20, 1, True)], 14, 2, 64, dtype, seed=3)
    q = torch.cat((query(Case([(0, 3)], 14, 2, 64, dtype)), torch.full((1, 14 * 64), 3.0, dtype=dtype)))
    out = torch.full((4, 14 * 64), 9.0, dtype=dtype, device="cuda")
    tok_pos = torch.cat((c.dev["tok_pos"], c.dev["tok_pos"].new_tensor([5])))
    ops.attention_e4m3(q.cuda(), out, c.dev["cu_q"], tok_pos, c.dev["slots"], c.site, 14, 4, 1, 64 ** -0.5, 0, ops.E4m3Scratch("cuda"), c.err)
    check(c, q[:3], out[:3])
    assert bool((out[3] == 9).all()) and not bool(out[2].any())


def test_a_captured_call_replayed_with_other_lengths():
    """The launch is the same whatever the lengths: runs are cut on the device."""
    c = Case([(900, 1), (40, 1), (3000, 1)], 14, 2, 64, torch.bfloat16, seed=3)
    q, out, scratch = query(c).cuda(), torch.empty((3, 14 * 64), dtype=torch.bfloat16, device="cuda"), ops.E4m3Scratch("cuda")
    run(c, q, scratch=scratch, max_kv_len=4000, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_e4m3(q, out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, 14, 3, 1, 64 ** -0.5, 0, scratch, c.err, 4000)
    for lengths in ([900, 40, 3000], [0, 0, 0], [5, 39, 2999], [899, 1, 64]):
        c.tok_pos = np.array(lengths)
        c.dev["tok_pos"].copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        check(c, q.cpu(), out)
    c.dev["slots"][1] = -1   # an entry that has ended
    graph.replay()
    assert not bool(out[1].any())


def test_a_workspace_that_a_captured_call_shares_with_larger_ones():
    """A larger call replaces buffers whose address the graph holds: the replay finds them still there, and nobody else in them."""
    small, large = Case([(900, 1), (40, 1)], 4, 2, 64, torch.bfloat16, seed=3), Case([(3000, 1)] * 12, 28, 4, 128, torch.bfloat16, seed=4)
    q, out, scratch = query(small).cuda(), torch.empty((2, 4 * 64), dtype=torch.bfloat16, device="cuda"), ops.E4m3Scratch("cuda")
    want = run(small, q, scratch=scratch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_e4m3(q, out, small.dev["cu_q"], small.dev["tok_pos"], small.dev["slots"], small.site, 4, 2, 1, 64 ** -0.5, 0, scratch, small.err)
    before = scratch.part_o.numel()
    check(large, query(large), run(large, query(large), scratch=scratch))
    assert scratch.part_o.numel() > before
    others = [torch.full((before,), 5.0, device="cuda") for _ in range(8)]   # (would get the buffer, were it given back)
    graph.replay()
    assert torch.equal(out, want) and all(bool((o == 5).all()) for o in others)
    check(large, query(large), run(large, query(large), scratch=scratch))


def test_a_workspace_that_grows_under_a_capture():
    """A call behind the capture and before any replay finds its counters zero."""
    c = Case([(900, 1), (4000, 1)], 14, 2, 64, torch.bfloat16, seed=3)
    q = query(c).cuda()
    want, out, scratch = run(c, q), torch.empty((2, 14 * 64), dtype=torch.bfloat16, device="cuda"), ops.E4m3Scratch("cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_e4m3(q, out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, 14, 2, 1, 64 ** -0.5, 0, scratch, c.err)
    assert torch.equal(run(c, q, scratch=scratch), want)
    graph.replay()
    assert torch.equal(out, want)
    assert torch.equal(run(c, q, scratch=scratch), want)


def test_calls_on_two_streams():
    """Each with a scratch of its own, at once."""
    cases = [Case([(3000 + 7 * i, 1), (100, 1)], 14, 2, 64, torch.bfloat16, seed=i) for i in range(2)]
    qs = [query(c, seed=i).cuda() for i, c in enumerate(cases)]
    want = [run(c, q) for c, q in zip(cases, qs)]
    scratches, streams = [ops.E4m3Scratch("cuda") for _ in cases], [torch.cuda.Stream() for _ in cases]
    outs = [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(50):
        for c, q, out, scratch, stream in zip(cases, qs, outs, scratches, streams):
            with torch.cuda.stream(stream):
                ops.attention_e4m3(q, out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, 14, 2, 1, 64 ** -0.5, 0, scratch, c.err)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_offsets_beyond_32_bits():
    """A storage of 5 GB whose last pages hold the sequence."""
    kv_heads, dim, pages = 4, 128, 80000
    storage = torch.empty((pages, 2, kv_heads, PAGE, dim), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.full((pages, 2, kv_heads), 2.0 ** -8, device="cuda")
    c = Case([(100, 1), (150, 2)], 8, kv_heads, dim, torch.bfloat16, seed=3, low=-8)
    far = torch.arange(len(c.codes), device="cuda") + pages - len(c.codes)
    storage[far] = c.storage
    scales[far] = c.held_scales
    q = query(c)
    want = run(c, q)
    c.dev["table"][c.dev["table"] >= 0] += pages - len(c.codes)
    near, c.site = c.site, ops.E4m3SiteArgs(storage, scales, c.dev["table"], kv_heads, dim)
    assert torch.equal(run(c, q), want)
    wrote = c.write()
    out = torch.empty(storage.shape, dtype=torch.bfloat16, device="cuda")
    ops.cache_read_e4m3(out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, 2, 152, c.err)
    c.dev["table"][c.dev["table"] >= 0] -= pages - len(c.codes)
    c.site = near
    assert torch.equal(c.write(), wrote)
    assert torch.equal(storage[far].view(torch.uint8), c.storage.view(torch.uint8)) and torch.equal(scales[far], c.held_scales)
    close = torch.empty(c.storage.shape, dtype=torch.bfloat16, device="cuda")
    ops.cache_read_e4m3(close, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, 2, 152, c.err)
    for s, slot in enumerate(c.slots):
        for p in range(int(c.tok_pos[c.cu_q[s + 1] - 1]) + 1):
            page = int(c.table[slot, p // PAGE])
            assert torch.equal(out[far[page], :, :, p % PAGE], close[page, :, :, p % PAGE])


@BOTH
def test_written_read_and_attended_over(dtype):
    """A prompt, a continuation of a few tokens and single tokens, as a model's layer runs them: attention over the written codes against
    attention over what is read back."""
    c = Case([(0, 200), (0, 77)], 8, 2, 64, dtype, seed=13)
    c.held_scales.fill_(2.0 ** 40)
    scratch = ops.E4m3Scratch("cuda")
    back = torch.zeros(c.codes.shape, dtype=dtype, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    at = [0, 0]
    base = c.qkv.cuda()
    for tokens in ([190, 70], [4, 1], [1, 1], [5, 5]):
        cu = [0, tokens[0], sum(tokens)]
        pos = list(range(at[0], at[0] + tokens[0])) + list(range(at[1], at[1] + tokens[1]))
        rows = torch.cat((base[at[0]:at[0] + tokens[0]], base[200 + at[1]:200 + at[1] + tokens[1]]))
        q = torch.empty((sum(tokens), 8 * 64), dtype=dtype, device="cuda")
        ops.rope_cache_write_e4m3(rows, i32(cu), i32([0] * tokens[0] + [1] * tokens[1]), i32(pos), c.dev["slots"], c.inv_freq.cuda(), 64, 8, q, c.site, max(tokens), c.err,
                                  bias=c.bias.cuda())
        at = [a + t for a, t in zip(at, tokens)]
        ops.cache_read_e4m3(back, i32(cu), i32(pos), c.dev["slots"], c.site, 2, max(at), c.err)
        out = torch.empty_like(q)
        ops.attention_e4m3(q, out, i32(cu), i32(pos), c.dev["slots"], c.site, 8, 2, max(tokens), 64 ** -0.5, 0, scratch, c.err, max(at))
        want, size, far = ref.attend(q.cpu(), cu, pos, c.slots, back.cpu().double(), c.table, 8, 64 ** -0.5, 0)
        off = (out.cpu().double().view(want.shape) - want).abs() - ref.attend_tolerance(want, size, far, dtype)
        assert bool((off <= 0).all()) and int(c.err) == 0


def test_refusals():
    c = Case([(0, 3)], 4, 2, 64, torch.bfloat16)
    d, q = c.dev, query(c).cuda()
    out, scratch = torch.empty_like(q), ops.E4m3Scratch("cuda")

    def attend(**change):
        a = dict(q=q, out=out, cu_q=d["cu_q"], tok_pos=d["tok_pos"], slots=d["slots"], site=c.site, n_heads=4, n_seqs=1, max_q_len=3, scale=0.125, window=0,
                 scratch=scratch, err=c.err, max_kv_len=3)
        a.update(change)
        ops.attention_e4m3(**a)
    for change in (dict(q=q.half()), dict(q=q.cpu()), dict(q=q[:, :-64]), dict(q=q.t().contiguous().t()), dict(out=out.float()), dict(out=out[:2]), dict(n_heads=3),
                   dict(n_heads=0), dict(n_heads=8), dict(n_seqs=2), dict(max_q_len=0), dict(max_kv_len=0), dict(window=-1), dict(cu_q=d["cu_q"].long()),
                   dict(tok_pos=d["tok_pos"][:2]), dict(q=torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)), dict(slots=d["slots"].cpu()), dict(err=c.err.long())):
        with pytest.raises(KernelError):
            attend(**change)
    attend()
