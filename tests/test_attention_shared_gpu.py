"""`ops.attention_shared` against softmax attention in float64 and against the library's own decode attention.

Tolerances. Scores are sums of D products in float32: each of the D additions rounds by 2^-24 of the partial sum, which is at most
sum |q k|, so a score is off by D 2^-24 max sum |q k| scale (natural units), and a weight by as much relatively; the hardware's 2^x
adds 2^-22 per factor of a weight (weight, rescaling, joining: fewer than 8). A row's value is a mean of v under the weights, so it is off
by twice that times max |v|. In bfloat16 each weight is rounded before the second product (2^-8 of it, half a step by eps / 2) while the
sum of weights is not, and the output is rounded (2^-8 of it): 2^-8 (max |v| + max |out|) bounds both."""
import math

import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.ops import branches

pytestmark = pytest.mark.gpu
PAGE = 64


class Batch:
    """Sequences with `own` tokens behind the pages that `groups` ((entries, pages)) share; pages shuffled over the storage."""

    def __init__(self, groups, own, heads, kv_heads, dim, dtype, seed=0, idle=(), extra_columns=0, gap=0):
        n = len(own)
        g = torch.Generator().manual_seed(seed)
        prefix = [0] * n
        for entries, pages in groups:
            for e in entries:
                prefix[e] = pages
        self.lengths = [p * PAGE + t for p, t in zip(prefix, own)]
        columns = max(-(-x // PAGE) for x in self.lengths) + extra_columns
        n_pages = sum(p for _, p in groups) + sum(-(-t // PAGE) for t in own) + 1
        ids = torch.randperm(n_pages, generator=g).tolist()
        slots = torch.randperm(n + 3, generator=g)[:n].tolist()
        table = torch.full((n + 3, columns), -1, dtype=torch.int32)
        for entries, pages in groups:
            common = torch.tensor([ids.pop() for _ in range(pages)], dtype=torch.int32)
            for e in entries:
                table[slots[e], :pages] = common
        for e in range(n):
            for p in range(prefix[e], -(-self.lengths[e] // PAGE)):
                table[slots[e], p] = ids.pop()
        dev = dict(device="cuda")
        self.table_cpu, self.slots_cpu = table, slots
        page = 2 * kv_heads * PAGE * dim
        raw = torch.randn((n_pages, page + gap), generator=g).to(dtype).cuda()
        self.storage = raw.as_strided((n_pages, 2, kv_heads, PAGE, dim), (page + gap, kv_heads * PAGE * dim, PAGE * dim, dim, 1))
        self.q = (1.3 * torch.randn((n, heads * dim), generator=g)).to(dtype).cuda()
        self.out = torch.full_like(self.q, 7.0)
        self.table = table.cuda()
        self.idle = set(idle)
        self.slots = torch.tensor([-1 if e in self.idle else s for e, s in enumerate(slots)], dtype=torch.int32, **dev)
        self.cu_q = torch.arange(n + 1, dtype=torch.int32, **dev)
        self.tok_pos = torch.tensor([x - 1 for x in self.lengths], dtype=torch.int32, **dev)
        self.err = torch.zeros(1, dtype=torch.int32, **dev)
        self.groups, self.n, self.heads, self.kv_heads, self.dim, self.dtype, self.scale = groups, n, heads, kv_heads, dim, dtype, dim ** -0.5
        self.share, self.scratch = ops.SharedPrefix(groups, n, "cuda"), ops.SharedScratch("cuda")
        self.site = ops.KvSiteArgs(self.storage, self.table, kv_heads, dim)

    def run(self, **kw):
        kw = {"max_kv_len": max(self.lengths), **kw}
        share = kw.pop("share", self.share)
        ops.attention_shared(self.q, self.out, self.cu_q, self.tok_pos, self.slots, self.site, self.heads, self.n, self.scale, share, self.scratch,
                             self.err, **kw)
        return self.out

    def check(self, out=None, sinks=None):
        out = self.out if out is None else out
        group = self.heads // self.kv_heads
        for e in range(self.n):
            got = out[e].view(self.heads, self.dim).double()
            if e in self.idle:
                assert (got == 0).all()
                continue
            length = int(self.tok_pos[e]) + 1
            pages = self.table_cpu[self.slots_cpu[e], :-(-length // PAGE)].long().cuda()
            kv = self.storage[pages].double().permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :length]   # [2, kv_heads, length, dim]
            k, v = (x.repeat_interleave(group, 0) for x in kv)
            q = self.q[e].view(self.heads, 1, self.dim).double()
            score = (q * k).sum(-1) * self.scale
            spread = float((q * k).abs().sum(-1).max()) * abs(self.scale)
            if sinks is not None:
                score = torch.cat((score, sinks.double()[:, None]), 1)
                v = torch.cat((v, torch.zeros_like(v[:, :1])), 1)
            weight = torch.softmax(score, -1)
            want = torch.einsum("hk,hkd->hd", weight, v)
            big = float(v.abs().max())
            bound = 2 * big * (self.dim * 2.0 ** -24 * spread + 8 * 2.0 ** -22)
            if self.dtype == torch.bfloat16:
                bound += 2.0 ** -8 * (big + float(want.abs().max()))
            off = float((got - want).abs().max())
            assert off <= bound, (e, off, bound)
        assert int(self.err) == 0


SHAPES = [(14, 2, 64), (16, 2, 128), (28, 4, 128), (6, 3, 96), (5, 1, 32), (20, 1, 64), (40, 2, 32), (3, 3, 128)]
CASES = {
    "one token each": ([([0, 1], 1)], [1, 1]),
    "a group of one": ([([1], 3)], [5, 64, 70]),
    "one group": ([(list(range(9)), 5)], [1, 63, 64, 65, 128, 129, 200, 31, 33]),
    "groups and loners": ([([0, 7, 3, 4], 9), ([2, 6], 17)], [1, 300, 64, 65, 2, 7, 33, 1000]),
    "nothing shared": ([], [1, 64, 65, 700]),
    "many": ([(list(range(1, 70)), 33)], [1 + 7 * i % 90 for i in range(71)]),
    "long and short": ([([0, 1, 2], 150), ([3, 4], 1)], [4000, 1, 2, 3, 4]),
}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("case", list(CASES))
def test_bfloat16(shape, case):
    b = Batch(*CASES[case], *shape, torch.bfloat16, seed=len(case))
    b.run()
    b.check()


@pytest.mark.parametrize("shape,dtype", [((14, 2, 64), torch.float32), ((4, 2, 128), torch.float32), ((20, 1, 32), torch.float32),
                                         ((3, 1, 23), torch.float32), ((2, 1, 256), torch.float32), ((1, 1, 1), torch.float32),
                                         ((3, 1, 23), torch.bfloat16), ((2, 1, 256), torch.bfloat16), ((1, 1, 1), torch.bfloat16)])
@pytest.mark.parametrize("case", [c for c in CASES if c != "long and short"])
def test_any_size(shape, case, dtype):
    b = Batch(*CASES[case], *shape, dtype, seed=len(case))
    b.run()
    b.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_it_is_the_decode_attention(dtype):
    """The same rows by the library's own kernel for single tokens; both within the same bounds of the formula, so within twice of each other."""
    b = Batch([([0, 1, 2, 5], 20)], [100, 1, 64, 700, 5, 6], 14, 2, 64, dtype)
    b.run()
    out = torch.empty_like(b.out)
    if dtype == torch.bfloat16:
        ops.attention_decode(b.q, out, b.cu_q, b.tok_pos, b.slots, b.site, 14, b.n, b.scale, 0, 8, ops.DecodeScratch("cuda"), b.err)
    else:
        ops.attention_generic(b.q, out, b.cu_q, b.tok_pos, b.slots, b.site, 14, b.n, 1, b.scale, 0, b.err)
    b.check()
    b.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ended_sequences_are_padding(dtype):
    """A slot of -1: zeros, whatever its group does; a group whose first member has ended, and one whose members all have."""
    groups, own = [([0, 1, 2, 3], 6), ([4, 5], 3), ([6, 7], 2)], [5, 6, 70, 8, 9, 10, 1, 64, 12]
    b = Batch(groups, own, 14, 2, 64, dtype, idle=(0, 3, 4, 5, 8))
    b.run()
    b.check()
    b = Batch(groups, own, 14, 2, 64, dtype, idle=range(9))
    b.run()
    b.check()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.bfloat16, 96), (torch.float32, 64)])
def test_what_lies_behind_the_last_position_is_not_read(dtype, dim):
    b = Batch([([0, 1, 2], 2)], [1, 40, 97, 31], 6, 3, dim, dtype, extra_columns=3)
    for e in range(b.n):
        length = b.lengths[e]
        page = int(b.table_cpu[b.slots_cpu[e], (length - 1) // PAGE])
        if length % PAGE:
            b.storage[page, 0, :, length % PAGE:] = math.nan
            b.storage[page, 1, :, length % PAGE:] = math.inf
    free = set(range(b.storage.shape[0])) - set(b.table_cpu.flatten().tolist())
    b.storage[list(free)] = math.nan
    b.run()
    b.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_member_that_stands_inside_the_shared_pages(dtype):
    """Keys behind its own position are not visible to it, though its group shares them; it has no own part."""
    b = Batch([([0, 1, 2], 5)], [9, 9, 70], 14, 2, 64, dtype)
    b.tok_pos[1] = 130
    b.tok_pos[0] = 0
    b.run()
    b.check()


def test_sinks():
    for dtype in (torch.bfloat16, torch.float32):
        b = Batch([([0, 2], 4)], [5, 6, 70], 14, 2, 64, dtype)
        sinks = torch.linspace(-3, 9, 14, device="cuda")
        b.run(sinks=sinks)
        b.check(sinks=sinks)


def test_extreme_scores():
    """Large queries: one key takes all the weight; scores of about +-1e4 stay finite, whichever part holds the largest."""
    for dtype in (torch.bfloat16, torch.float32):
        b = Batch([([0, 1], 3)], [70, 2], 4, 2, 64, dtype)
        b.q.mul_(300.0)
        b.run()
        assert torch.isfinite(b.out).all()
        for e in range(2):
            length = b.lengths[e]
            pages = b.table_cpu[b.slots_cpu[e], :-(-length // PAGE)].long().cuda()
            kv = b.storage[pages].double().permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :length].repeat_interleave(2, 1)
            score = (b.q[e].view(4, 1, 64).double() * kv[0]).sum(-1) * b.scale
            two = score.topk(2).values
            for h in range(4):
                if float(two[h, 0] - two[h, 1]) > 60:   # the others' weights are below 2^-80
                    assert torch.equal(b.out[e].view(4, 64)[h], kv[1, h, int(score[h].argmax())].to(dtype))


@pytest.mark.parametrize("gap", [64, 4096])
def test_pages_with_gaps(gap):
    for dtype in (torch.bfloat16, torch.float32):
        b = Batch([([0, 2], 4)], [5, 6, 70], 14, 2, 64, dtype, gap=gap)
        b.run()
        b.check()


def test_a_page_that_is_not_held_is_reported():
    for dtype in (torch.bfloat16, torch.float32):
        b = Batch([([0, 2], 4)], [5, 6, 70], 14, 2, 64, dtype)
        b.table[b.slots.long()[1], 0] = -1
        b.run()
        assert int(b.err) == ops.ERR_NO_PAGE
        b.err.zero_()
        b.idle = {1}   # (its own row is not compared; the others' are whole)
        b.out[1] = 0
        b.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bounds(dtype):
    """A loose or tight bound on the lengths, workspaces that grow: within the same bounds of the formula."""
    b = Batch([([0, 1, 2, 5], 20)], [100, 1, 64, 700, 5, 6], 14, 2, 64, dtype, extra_columns=40)
    b.run(max_kv_len=None)
    b.check()
    b.run(max_kv_len=1)   # (fewer runs: slower, not wrong)
    b.check()
    b.run()
    first = b.out.clone()
    b.run()
    assert torch.equal(first, b.out)   # no sum depends on the order in which blocks end
    b.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_and_replayed_with_other_lengths(dtype):
    b = Batch([([0, 1, 3], 6)], [100, 30, 64, 200], 14, 2, 64, dtype)
    b.run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.run()
    for lengths, idle in (([b.lengths[0], 6 * PAGE + 1, 3, 6 * PAGE + 129], ()), ([6 * PAGE + 7, 1, 64, b.lengths[3]], (1, 0))):
        b.tok_pos.copy_(torch.tensor([x - 1 for x in lengths], dtype=torch.int32))
        b.slots.copy_(torch.tensor([-1 if e in idle else s for e, s in enumerate(b.slots_cpu)], dtype=torch.int32))
        if lengths[1] == 1:
            b.tok_pos[1] = 6 * PAGE
        b.idle = set(idle)
        b.out.fill_(3.0)
        graph.replay()
        b.check()


def test_on_another_stream():
    b = Batch([([0, 1, 3], 6)], [100, 30, 64, 200], 14, 2, 64, torch.bfloat16)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        b.run()
        torch.cuda.current_stream().synchronize()
    b.check()


def test_refusals():
    b = Batch([([0, 2], 4)], [5, 6, 70], 14, 2, 64, torch.bfloat16)
    good = dict(q=b.q, out=b.out, site=b.site, share=b.share, heads=14)

    def run(**kw):
        a = {**good, **kw}
        ops.attention_shared(a["q"], a["out"], a.get("cu_q", b.cu_q), a.get("tok_pos", b.tok_pos), a.get("slots", b.slots), a["site"], a["heads"], b.n, b.scale,
                             a["share"], b.scratch, b.err, **{k: v for k, v in kw.items() if k == "sinks"})
    run()
    for bad in (dict(q=b.q.half()), dict(q=b.q[:, :64]), dict(out=b.out[:2]), dict(out=b.out.float()), dict(heads=13), dict(heads=15), dict(cu_q=b.cu_q[:3]),
                dict(share=ops.SharedPrefix([], 2, "cuda")), dict(share=ops.SharedPrefix([([0, 1], 50)], 3, "cuda")), dict(slots=b.slots.long()),
                dict(sinks=torch.zeros(13, device="cuda")), dict(share=ops.SharedPrefix([([0, 2], 4)], 3, "cpu")),
                dict(site=ops.KvSiteArgs(b.storage.float(), b.table, 2, 64)), dict(site=ops.KvSiteArgs(b.storage, b.table, 2, 32)),
                dict(site=ops.KvSiteArgs(b.storage[:, :1], b.table, 2, 64)), dict(site=ops.KvSiteArgs(b.storage, b.table.t(), 2, 64)),
                dict(q=torch.empty(3 * 14 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, -1))):
        with pytest.raises(ops.KernelError):
            run(**bad)
    wide = Batch([([0, 1], 1)], [2, 3], 2, 1, 257, torch.float32)
    with pytest.raises(ops.KernelError, match="257"):
        wide.run()
    b.check()


def test_offsets_beyond_32_bits():
    """Pages whose first element lies beyond 2^32 elements of the storage."""
    kv_heads, dim, n_pages = 4, 128, 2 ** 32 // (2 * 4 * PAGE * 128) + 9
    storage = torch.empty((n_pages, 2, kv_heads, PAGE, dim), dtype=torch.bfloat16, device="cuda")
    b = Batch([([0, 1], 3)], [5, 70], 8, kv_heads, dim, torch.bfloat16)
    shift = n_pages - b.storage.shape[0]
    storage[shift:] = b.storage
    b.storage, b.table_cpu = storage, torch.where(b.table_cpu >= 0, b.table_cpu + shift, b.table_cpu)
    b.table = b.table_cpu.cuda()
    b.site = ops.KvSiteArgs(storage, b.table, kv_heads, dim)
    b.run()
    b.check()


TILED = [(32, 1, 64), (32, 2, 128)]   # shapes whose groups of nine sequences behind 33 pages go to the tensor-core tiles


def tiled(shape, groups=None, own=None, **kw):
    """Two groups on tiles (288 and 160 or 320 rows, odd and even page counts), a small one on warps, and sequences that share nothing."""
    groups = groups or [([0, 2, 3, 4, 5, 8, 9, 10, 11], 33), ([1, 6, 7, 12, 13], 52), ([14, 15], 2)]
    own = own or [1, 63, 64, 65, 130, 7, 200, 31, 500, 2, 33, 64, 128, 129, 70, 1, 300]
    b = Batch(groups, own, *shape, torch.bfloat16, **kw)
    tiles = branches._shared_sizes(torch.bfloat16, b.dim, b.kv_heads, b.heads, b.share, branches._own_pages(max(b.lengths), b.table, b.share))[1]
    assert tiles > 0
    return b


@pytest.mark.parametrize("shape", TILED)
@pytest.mark.parametrize("gap", [0, 128])
def test_tiles(shape, gap):
    b = tiled(shape, gap=gap)
    b.run()
    b.check()
    first = b.out.clone()
    b.run(max_kv_len=None)
    b.check()
    b.run()
    assert torch.equal(b.out, first)


@pytest.mark.parametrize("shape", TILED)
@pytest.mark.parametrize("idle", [(0, 4), (1, 6, 7, 12, 13), tuple(range(14)), tuple(range(17))])
def test_tiles_of_ended_sequences(shape, idle):
    b = tiled(shape, idle=idle)
    b.run()
    b.check()


@pytest.mark.parametrize("shape", TILED)
def test_tiles_of_members_inside_the_shared_pages(shape):
    b = tiled(shape)
    b.tok_pos[torch.tensor([0, 3, 12, 14])] = torch.tensor([0, 5 * PAGE + 3, 51 * PAGE, 64], dtype=torch.int32, device="cuda")
    b.run()
    b.check()


@pytest.mark.parametrize("shape", TILED)
def test_tiles_with_nothing_beside_them(shape):
    """Every sequence stands inside what it shares: there are no other records."""
    b = tiled(shape, [(list(range(10)), 40)], [1] * 10)
    b.tok_pos.copy_(torch.tensor([40 * PAGE - 1 - 97 * e for e in range(10)], dtype=torch.int32))
    b.run()
    b.check()


@pytest.mark.parametrize("shape", TILED)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.5])
def test_tiles_with_sinks_and_any_scale(shape, scale):
    b = tiled(shape)
    b.scale = scale
    sinks = torch.linspace(-5, 9, shape[0], device="cuda")
    b.run(sinks=sinks)
    b.check(sinks=sinks)


@pytest.mark.parametrize("shape", TILED)
def test_tiles_read_nothing_behind_the_last_position(shape):
    b = tiled(shape)
    for e in range(b.n):
        length = b.lengths[e]
        page = int(b.table_cpu[b.slots_cpu[e], (length - 1) // PAGE])
        if length % PAGE:
            b.storage[page, 0, :, length % PAGE:] = math.nan
            b.storage[page, 1, :, length % PAGE:] = math.inf
    free = set(range(b.storage.shape[0])) - set(b.table_cpu.flatten().tolist())
    b.storage[list(free)] = math.nan
    b.run()
    b.check()


@pytest.mark.parametrize("shape", TILED)
def test_tiles_report_a_page_that_is_not_held(shape):
    b = tiled(shape)
    b.table[b.slots.long()[[1, 6, 7, 12, 13]], 3] = -1
    b.run()
    assert int(b.err) == ops.ERR_NO_PAGE
    b.err.zero_()
    b.idle = {1, 6, 7, 12, 13}   # (their rows are not compared; the others' are whole)
    b.out[list(b.idle)] = 0
    b.check()


@pytest.mark.parametrize("shape", TILED)
def test_what_is_shared_is_replaced_under_a_graph(shape):
    """Within the bound it was captured with: fewer pages are shared, too few for the tiles, then as many as there may be."""
    b = tiled(shape)
    share = ops.SharedPrefix(b.groups, b.n, "cuda", bound_pages=64)
    b.run(share=share)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.run(share=share)
    for pages in (1, 20, None):
        share.load(ops.SharedPrefix([(e, min(p, pages) if pages else p) for e, p in b.groups], b.n, "cuda"))
        b.out.fill_(3.0)
        graph.replay()
        b.check()
    with pytest.raises(ops.KernelError):
        share.load(ops.SharedPrefix([(e, 65) for e, _ in b.groups], b.n, "cuda"))
    with pytest.raises(ops.KernelError):
        share.load(ops.SharedPrefix(b.groups[:2], b.n, "cuda"))


@pytest.mark.parametrize("shape,groups", [((4, 1, 32), [(range(0, 1000), 2)] + [(range(1000 + 5 * i, 1005 + 5 * i), 3) for i in range(200)]),
                                          ((8, 1, 64), [(range(3, 2048), 2)]), ((2, 1, 20), [(range(0, 2048, 2), 1)])])
def test_the_largest_batch(shape, groups):
    b = Batch([(list(e), p) for e, p in groups], [1 + i % 67 for i in range(2048)], *shape, torch.bfloat16)
    b.run()
    b.check()


def test_two_graphs_on_two_streams():
    """With workspaces of their own."""
    runs = []
    for seed, shape in ((1, (14, 2, 64)), (2, (16, 2, 128)), (3, (32, 1, 64))):
        b = Batch(*CASES["many"], *shape, torch.bfloat16, seed=seed)
        b.run()
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            b.run()
        b.out.fill_(3.0)
        runs.append((b, graph, stream))
    torch.cuda.synchronize()
    for _ in range(20):
        for _, graph, stream in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for b, _, _ in runs:
        b.check()
