"""Attention over a sequence cache in 8 bits where a warp takes many pages of a sequence one after another: batches that fill the device, over a few pages that the
sequences share. Against the formula in 64 bits (on the device), with the tolerance of `e4m3_refs.attend_tolerance`."""
import math

import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.ops import cache_e4m3
from tests import e4m3_refs as ref

pytestmark = pytest.mark.gpu
PAGE = 64
BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])


class Batch:
    """Sequences over `pages` [sequences, columns] (page numbers) of `lengths` after the step, the last `tokens` of each its new ones."""

    def __init__(self, pages, lengths, tokens, heads, kv_heads, dim, dtype, seed=0, pool=40):
        self.heads, self.kv_heads, self.dim, self.dtype, self.lengths, self.tokens = heads, kv_heads, dim, dtype, lengths, tokens
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = self.n = len(lengths)
        self.codes = torch.randn((pool, 2, kv_heads, PAGE, dim), generator=g, device="cuda").mul(100).clamp(-448, 448).to(torch.float8_e4m3fn)
        self.scales = torch.full((pool, 2, kv_heads), 2.0 ** -8, device="cuda")
        self.table = pages.to(device="cuda", dtype=torch.int32).contiguous()
        i32 = dict(dtype=torch.int32, device="cuda")
        self.cu_q = [0]
        for t in tokens:
            self.cu_q.append(self.cu_q[-1] + t)
        self.dev_cu = torch.tensor(self.cu_q, **i32)
        self.tok_pos = torch.cat([torch.arange(x - t, x) for x, t in zip(lengths, tokens)]).to(**i32)
        self.slots = torch.arange(n, **i32)
        self.err = torch.zeros(1, **i32)
        self.q = (0.4 * torch.randn((self.cu_q[-1], heads * dim), generator=g, device="cuda")).to(dtype)

    def warp_pages(self):
        """The least pages that a warp of this batch has on average."""
        rows = max(self.tokens) * (self.heads // self.kv_heads)
        block_rows = 8 if rows <= 8 else 16
        slots = cache_e4m3._slots_of(self.dtype == torch.bfloat16, self.dim, block_rows)
        return sum(-(-x // PAGE) for x in self.lengths) * self.kv_heads / slots / 4

    def run(self, window=0, scale=None):
        site = ops.E4m3SiteArgs(self.codes, self.scales, self.table, self.kv_heads, self.dim)
        out = torch.full_like(self.q, 9.0)
        ops.attention_e4m3(self.q, out, self.dev_cu, self.tok_pos, self.slots, site, self.heads, self.n, max(self.tokens), self.dim ** -0.5 if scale is None else scale,
                           window, ops.E4m3Scratch("cuda"), self.err, max(self.lengths))
        assert int(self.err) == 0
        return out

    def plain(self, window=0, scale=None):
        """(output, sum of weights times |value|, largest sum of |q k| times scale) in 64 bits, [T, heads, dim], the last [T, heads, 1]."""
        scale = self.dim ** -0.5 if scale is None else scale
        values = self.codes.double() * self.scales.double()[..., None, None]
        out = torch.empty((self.cu_q[-1], self.heads, self.dim), dtype=torch.float64, device="cuda")
        size, far = torch.empty_like(out), out.new_empty((self.cu_q[-1], self.heads, 1))
        group = self.heads // self.kv_heads
        for s, (length, t) in enumerate(zip(self.lengths, self.tokens)):
            columns = -(-length // PAGE)
            k, v = values[self.table[s, :columns].long()].permute(1, 2, 0, 3, 4).reshape(2, self.kv_heads, columns * PAGE, self.dim)[:, :, :length]
            rows = slice(self.cu_q[s], self.cu_q[s + 1])
            q = self.q[rows].double().view(t, self.kv_heads, group, self.dim)
            at, key = self.tok_pos[rows].long()[:, None], torch.arange(length, device="cuda")
            seen = ((key <= at) & (key > at - window if window > 0 else key >= 0))[:, None, None]
            x = torch.where(seen, torch.einsum("tkgd,kjd->tkgj", q, k) * scale, -math.inf)
            w = torch.softmax(x, -1)
            out[rows] = torch.einsum("tkgj,kjd->tkgd", w, v).reshape(t, self.heads, self.dim)
            size[rows] = torch.einsum("tkgj,kjd->tkgd", w, v.abs()).reshape(t, self.heads, self.dim)
            reach = torch.where(seen, torch.einsum("tkgd,kjd->tkgj", q.abs(), k.abs()), 0.0)
            far[rows] = (reach.amax(-1) * abs(scale)).reshape(t, self.heads, 1)
        return out, size, far

    def check(self, window=0, scale=None, same_scores=False, floor=False):
        """`same_scores`: what differs between scores is so large that it leaves weights of 0, or nothing at all.
        `floor`: components may come from weights alone that are far below the row's largest, where the others' values are zero. A weight is a float16 number (or two)
        that is 2^14 where it is the largest; float16's smallest step is 2^-24, so a weight is off by 2^-25 / 2^14 = 2^-39 of the largest one however small it is
        itself, the largest is at most 1, and the sum of all is no less than it: 2^-39 of every value that a row sees."""
        got, (want, size, far) = self.run(window, scale), self.plain(window, scale)
        if same_scores:
            far.zero_()
        off = (got.double().view(want.shape) - want).abs() - ref.attend_tolerance(want, size, far, self.dtype)
        if floor:
            values = (self.codes[:, 1].double().abs() * self.scales[:, 1].double()[..., None, None]).amax((0, 2))   # [kv heads, dim]
            counts = (self.tok_pos + 1).double()[:, None, None]
            off -= 2.0 ** -39 * counts * values.repeat_interleave(self.heads // self.kv_heads, 0)
        assert bool((off <= 0).all()), f"{float(off.max())} beyond the tolerance"
        assert torch.equal(self.run(window, scale), got)


def scattered(n, longest, seed, pool=40, even=False):
    """Page numbers and lengths: a sequence's pages are any of the pool, lengths up to `longest`, or nearly that."""
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(longest - 40 if even else 1, longest + 1, (n,), generator=g).tolist()
    return torch.randint(0, pool, (n, -(-longest // PAGE)), generator=g), lengths


# heads, kv heads, head size, sequences, longest, most tokens: blocks of 8 rows and of 16, ragged and even, parts of pairs
MANY = [(8, 4, 128, 64, 8000, 1), (14, 2, 64, 150, 6000, 1), (8, 8, 32, 64, 6000, 1), (12, 4, 96, 64, 5000, 4), (28, 4, 64, 40, 6000, 3), (16, 2, 128, 80, 5000, 2)]


@pytest.mark.parametrize("apart", [0, 3, 25])
@pytest.mark.parametrize("heads,kv_heads,dim,n,longest,tokens", MANY)
@BOTH
def test_many_pages_to_a_warp(heads, kv_heads, dim, n, longest, tokens, dtype, apart):
    """Values' scales up to 2^-apart .. 2^apart, another one on every page."""
    pages, lengths = scattered(n, longest, seed=dim)
    b = Batch(pages, lengths, [min(x, 1 + i % tokens) for i, x in enumerate(lengths)], heads, kv_heads, dim, dtype, seed=dim)
    assert b.warp_pages() > 4
    g = torch.Generator(device="cuda").manual_seed(1)
    b.scales[:, 1] = torch.exp2(torch.randint(-apart, apart + 1, b.scales[:, 1].shape, generator=g, device="cuda").float() - 8)
    b.scales[:, 0] = torch.exp2(torch.randint(-2, 3, b.scales[:, 0].shape, generator=g, device="cuda").float() - 8)
    b.check()


@pytest.mark.parametrize("window", [100, 3000])
@BOTH
def test_many_pages_to_a_warp_behind_a_window(window, dtype):
    pages, lengths = scattered(300, 5000, seed=1, even=True)
    Batch(pages, lengths, [1] * 300, 8, 4, 64, dtype).check(window)


@BOTH
def test_more_than_32_pages_to_a_warp(dtype):
    """A warp looks up 32 pages at a time."""
    pages, lengths = scattered(256, 12600, seed=2, even=True)
    b = Batch(pages, lengths, [1] * 256, 8, 4, 64, dtype)
    assert b.warp_pages() > 64
    b.check()


def exponents(first, steps):
    """Of the groups of four pages, one for each warp of a block: what a warp meets page after page."""
    e = [first]
    for s in steps:
        e.append(min(max(e[-1] + s, ref.LOW), ref.HIGH))
    return torch.tensor(e)


STAIRS = {"falling by 29": exponents(60, [-29] * 4), "falling by 29 from the top": exponents(119, [-29] * 7), "falling by 31": exponents(119, [-31] * 7), "falling by 10": exponents(119, [-10] * 15),
          "falling by 9": exponents(119, [-9] * 15), "rising by 29": exponents(-112, [29] * 7), "rising by 31": exponents(-112, [31] * 7), "rising by 10": exponents(-112, [10] * 15),
          "up and down": exponents(0, [25, -30, 29, -20, -30, -30, 60, -11, 12, -100, 100]), "down and back": exponents(100, [-30] * 5 + [30] * 5),
          "up and back": exponents(-50, [30] * 5 + [-30] * 5)}


@pytest.mark.parametrize("stairs", list(STAIRS))
@pytest.mark.parametrize("heads,kv_heads,dim,tokens", [(4, 2, 64, 1), (14, 2, 64, 2), (8, 4, 128, 1), (12, 4, 128, 4)])
@BOTH
def test_values_of_scales_that_fall_and_rise(stairs, heads, kv_heads, dim, tokens, dtype):
    """Even weights (equal keys): the result is the mean of values whose scale changes with every page that a warp takes."""
    e = STAIRS[stairs]
    n = 512 // kv_heads
    pages = (torch.arange(4 * len(e)) + 4 * len(e) * (torch.arange(n) % 2)[:, None])
    b = Batch(pages, [4 * len(e) * PAGE - 60 * (i % 7) for i in range(n)], [tokens] * n, heads, kv_heads, dim, dtype, pool=8 * len(e))
    assert b.warp_pages() * 4 > 4 * len(e) / 2
    b.codes[:, 0] = torch.ones((), device="cuda").to(torch.float8_e4m3fn)
    b.scales[:, 1] = torch.exp2(e.repeat_interleave(4).repeat(2).float()).cuda()[:, None]
    b.check()


# A position of group g scores -`fall` g in base 2, its values stand `rise` binary places above those of the group before: what it adds is 2^((rise - fall) g).
@pytest.mark.parametrize("fall,rise", [(20, 25), (5, 11), (8, 9), (8, 8), (11, 10), (25, 20), (28, 31)])   # (31 * 4 - 8 is within the scales' 119)
@pytest.mark.parametrize("heads,kv_heads,dim,tokens", [(4, 2, 64, 1), (14, 2, 64, 2), (8, 4, 128, 1), (12, 4, 128, 4)])
@pytest.mark.parametrize("first", [True, False], ids=["largest weight first", "largest weight last"])
@BOTH
def test_large_values_of_small_weight(first, heads, kv_heads, dim, tokens, fall, rise, dtype):
    """Weights down to 2^-112 beside values that outweigh them."""
    groups = 5
    n = 512 // kv_heads
    order = torch.arange(groups) if first else torch.arange(groups).flip(0)
    per = 4 * groups
    pages = torch.arange(per) + per * (torch.arange(n) % 2)[:, None]
    b = Batch(pages, [per * PAGE - 3 * (i % 5) for i in range(n)], [tokens] * n, heads, kv_heads, dim, dtype, pool=2 * per)
    g = order.repeat_interleave(4).repeat(2).float().cuda()
    b.codes[:, 0] = (-g).view(-1, 1, 1, 1).expand(b.codes[:, 0].shape).to(torch.float8_e4m3fn)   # (whole numbers up to 16 are codes)
    b.scales[:, 0] = 1.0
    b.scales[:, 1] = torch.exp2(rise * g - 8)[:, None]
    b.q.fill_(1.0)
    # every score is -g dim scale: exact but for the factor's rounding, so a weight is as exact as its exponential
    b.check(scale=fall * math.log(2.0) / dim)


def large_batch(seqs, heads, kv_heads, dim, tokens, dtype):
    """Every query and key component 1, in pages of which one has a key scale of 2 and codes of 1/2."""
    pages, lengths = scattered(seqs, 1500, seed=4)
    b = Batch(pages, lengths, [min(x, tokens) for x in lengths], heads, kv_heads, dim, dtype)
    b.q.fill_(1.0)
    b.codes[:, 0] = torch.ones((), device="cuda").to(torch.float8_e4m3fn)
    b.codes[::3, 0] = torch.full((), 0.5, device="cuda").to(torch.float8_e4m3fn)
    b.scales[:, 0] = 1.0
    b.scales[::3, 0] = 2.0
    return b


LARGE = pytest.mark.parametrize("score", [1e4, 3e4, 3e7, 1e8, -1e8, 1e12, -1e12, 1e30])
FEW_AND_MANY = pytest.mark.parametrize("seqs,heads,kv_heads,dim,tokens", [(3, 14, 2, 64, 1), (3, 28, 4, 128, 4), (200, 8, 4, 64, 1), (200, 8, 2, 128, 3)])


@LARGE
@FEW_AND_MANY
@BOTH
def test_equal_scores_of_any_size(seqs, heads, kv_heads, dim, tokens, score, dtype):
    """Even weights."""
    large_batch(seqs, heads, kv_heads, dim, tokens, dtype).check(scale=score / dim, same_scores=True)


@LARGE
@FEW_AND_MANY
@BOTH
def test_scores_of_any_size_that_differ(seqs, heads, kv_heads, dim, tokens, score, dtype):
    """One position of a page scores half of (or, where scores are negative, twice) what the others do: these have weights of exp(-5000) and less, zero in 64 bits too."""
    b = large_batch(seqs, heads, kv_heads, dim, tokens, dtype)
    other = b.codes.clone()
    b.codes[:, 0] = (b.codes[:, 0].float() * (0.5 if score > 0 else 2.0)).to(torch.float8_e4m3fn)
    b.codes[:, 0, :, 0] = other[:, 0, :, 0]   # the first position of every page, which every token sees
    b.check(scale=score / dim, same_scores=True)


@pytest.mark.parametrize("spread", [1e3, 1e6, 1e20])
@FEW_AND_MANY
@BOTH
def test_random_scores_of_any_size(seqs, heads, kv_heads, dim, tokens, spread, dtype):
    pages, lengths = scattered(seqs, 1500, seed=5)
    b = Batch(pages, lengths, [min(x, tokens) for x in lengths], heads, kv_heads, dim, dtype)
    b.q = (b.q.float() * spread).to(dtype)
    b.check(floor=True)
    assert bool((b.run().view(-1, dim) != 0).any(-1).all())   # (so loose a tolerance would let a row of zeros pass)


def test_many_sequences_beside_a_long_prompt():
    """The largest entry's blocks of rows times all entries are more than 32 bits count; what there is to do is not."""
    n = 900
    pages, _ = scattered(n, 1024, seed=6)
    b = Batch(pages, [1024] + [40] * (n - 1), [1024] + [1] * (n - 1), 64, 2, 16, torch.float32)
    assert n * 2 * (1024 * 32 // 16) * (16 + 2 * cache_e4m3._slots_of(0, 16, 16)) > 2 ** 31
    b.check()


@pytest.mark.parametrize("score", [5e6, 1.1e7, 1.2e7, -1.1e7])
@FEW_AND_MANY
@BOTH
def test_equal_scores_as_large_as_their_factors_allow(seqs, heads, kv_heads, dim, tokens, score, dtype):
    """Key components of 448: what the largest query component and the page's scale allow is what the scores are (1.6e7 and 1.7e7 in base 2)."""
    b = large_batch(seqs, heads, kv_heads, dim, tokens, dtype)
    b.codes[:, 0] = torch.full((), 448.0, device="cuda").to(torch.float8_e4m3fn)
    b.scales[:, 0] = 2.0 ** -9
    b.check(scale=score / (dim * 448 * 2.0 ** -9), same_scores=True)
