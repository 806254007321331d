"""Writing a sequence cache in 8 bits with the rotation, and reading it back, against the plain implementation in 64 bits."""
import numpy as np
import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.ops import KernelError
from tests import e4m3_refs as ref

pytestmark = pytest.mark.gpu
PAGE = 64


class Case:
    """A batch over a cache whose pages hold random codes: starts and tokens per entry, slot -1 for padding entries."""

    def __init__(self, entries, heads, kv_heads, dim, dtype, seed=0, rot_dim=None, bias=True, extra=0, gap=0, low=-6, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        n = len(entries)
        self.heads, self.kv_heads, self.dim, self.dtype, self.n = heads, kv_heads, dim, dtype, n
        lengths = [a + t for a, t, *_ in entries]
        self.slots = [-1 if len(e) > 2 and e[2] else int(s) for s, e in zip(rng.permutation(n + 1)[:n], entries)]
        columns = max(1, max(-(-x // PAGE) for x in lengths) + 1)
        total = sum(-(-x // PAGE) for x in lengths) + 2
        ids = list(rng.permutation(total))
        self.table = np.full((n + 1, columns), -1, dtype=np.int32)
        for s in range(n):
            if self.slots[s] >= 0:
                for c in range(-(-lengths[s] // PAGE)):
                    self.table[self.slots[s], c] = ids.pop()
        self.cu_q = [0] + list(np.cumsum([t for _, t, *_ in entries]))
        self.tok_seq = np.repeat(np.arange(n), [t for _, t, *_ in entries])
        self.tok_pos = np.concatenate([np.arange(a, a + t) for a, t, *_ in entries]) if self.cu_q[-1] else np.zeros(0, dtype=int)
        self.rot_dim = dim if rot_dim is None else rot_dim
        self.inv_freq = (1.0 / 1e4 ** (torch.arange(0, self.rot_dim, 2) / max(self.rot_dim, 1))).float() if self.rot_dim else None
        width = (heads + 2 * kv_heads) * dim
        self.qkv = (spread * torch.randn((self.cu_q[-1], width + extra), generator=g)).to(dtype)
        self.bias = (0.3 * torch.randn(width, generator=g)).to(dtype) if bias else None
        self.codes = torch.randn((total, 2, kv_heads, PAGE, dim), generator=g).mul(100).clamp(-448, 448).to(torch.float8_e4m3fn)
        self.scales = torch.exp2(torch.randint(low, low + 3, (total, 2, kv_heads), generator=g).float())
        # on the device: pages (and scales of pages) perhaps apart
        page = 2 * kv_heads * PAGE * dim
        raw = torch.zeros((total, page + 16 * gap), dtype=torch.uint8, device="cuda")
        self.storage = raw.view(torch.float8_e4m3fn)[:, :page].unflatten(1, (2, kv_heads, PAGE, dim))
        raw[:, :page] = self.codes.view(torch.uint8).reshape(total, -1).cuda()
        self.raw = raw
        held = torch.zeros((total, 2 * kv_heads + gap), device="cuda")
        self.held_scales = held[:, :2 * kv_heads].unflatten(1, (2, kv_heads))
        self.held_scales.copy_(self.scales.cuda())
        i32 = lambda x: torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()   # noqa: E731
        self.dev = dict(cu_q=i32(self.cu_q), tok_seq=i32(self.tok_seq), tok_pos=i32(self.tok_pos), slots=i32(self.slots), table=i32(self.table))
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.site = ops.E4m3SiteArgs(self.storage, self.held_scales, self.dev["table"], kv_heads, dim)
        self.most = max([t for _, t, *_ in entries] + [1])

    def write(self, qkv=None, q_out=None):
        q_out = torch.full((self.cu_q[-1], self.heads * self.dim), 7.0, dtype=self.dtype, device="cuda") if q_out is None else q_out
        ops.rope_cache_write_e4m3(self.qkv.cuda() if qkv is None else qkv, self.dev["cu_q"], self.dev["tok_seq"], self.dev["tok_pos"], self.dev["slots"],
                                  None if self.inv_freq is None else self.inv_freq.cuda(), self.rot_dim, self.heads, q_out, self.site, self.most, self.err,
                                  bias=None if self.bias is None else self.bias.cuda())
        return q_out

    def plain(self):
        """queries, new rows, codes and scales that the write leaves, in 64 bits"""
        codes, scales = self.codes.double(), self.scales.double()
        q, rows = ref.write(self.qkv, self.bias, self.cu_q, torch.from_numpy(self.tok_pos), self.slots, self.inv_freq, self.rot_dim, self.heads,
                            self.kv_heads, self.dim, codes, scales, self.table)
        return q, rows, codes, scales

    def check(self, q_out):
        q, rows, codes, scales = self.plain()
        got, got_scales = self.storage.cpu().double(), self.held_scales.cpu().double()
        assert torch.equal(got_scales, scales)
        # float32 arithmetic on the way: the bias, two products with cosine and sine (2 ulp each), their sum; at most 8 roundings of 2^-24 of the
        # row's largest element each way
        slack = 8 * 2.0 ** -24 * 2 * torch.where(torch.isfinite(rows), rows.abs(), 0.0).amax(-1, keepdim=True)
        new = torch.zeros(codes.shape[:1] + codes.shape[3:4], dtype=torch.bool)
        for t, (s, p) in enumerate(zip(self.tok_seq, self.tok_pos)):
            if self.slots[s] < 0:
                continue
            page = int(self.table[self.slots[s], p // PAGE])
            new[page, p % PAGE] = True
            x, scale = rows[t], scales[page][..., None]
            value = got[page, :, :, p % PAGE] * scale
            nan = torch.isnan(x)
            assert torch.equal(torch.isnan(value), nan)
            most = ref.TOP * scale.expand_as(x)
            want = torch.where(nan, torch.zeros_like(x), torch.minimum(torch.maximum(x, -most), most))
            half = torch.exp2(torch.floor(torch.log2((want.abs() / scale).clamp(min=2.0 ** -6))) - 4) * scale
            far = (torch.where(nan, torch.zeros_like(x), value) - want).abs()
            assert bool((far <= half + slack[t]).all()), f"token {t}: {float((far - half).max())}"
        for page, row in (~new).nonzero().tolist():   # older rows, rescaled or not, and what nobody wrote: equal, bit by bit
            assert torch.equal(got[page, :, :, row], codes[page, :, :, row]), f"page {page} row {row}"
        bound = torch.finfo(self.dtype).eps / 2 * q.abs() + 2 * 8 * 2.0 ** -24 * torch.where(torch.isfinite(q), q.abs(), 0.0).view(len(q), -1, self.dim).amax(-1).repeat_interleave(self.dim, 1)
        far = (q_out.cpu().double() - q).abs()
        assert bool((far <= bound).all()), f"queries: {float((far - bound).max())}"
        assert int(self.err) == 0


ENTRIES = {
    "single tokens": [(0, 1), (63, 1), (64, 1), (500, 1), (1, 1)],
    "prompts": [(0, 130), (0, 1), (0, 64), (0, 63), (0, 65)],
    "spans": [(60, 9), (63, 2), (10, 5), (128, 64), (100, 200)],
    "padding": [(0, 3), (0, 7, True), (40, 2), (0, 1, True)],
}


@pytest.mark.parametrize("entries", list(ENTRIES), ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (28, 4, 128), (4, 2, 16), (6, 3, 96), (5, 5, 80), (3, 1, 48), (2, 1, 112), (8, 1, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_write(entries, heads, kv_heads, dim, dtype):
    c = Case(ENTRIES[entries], heads, kv_heads, dim, dtype, seed=dim + heads)
    c.check(c.write())


@pytest.mark.parametrize("rot_dim", [0, 2, 16, 34, 64])
@pytest.mark.parametrize("bias", [True, False])
def test_part_of_the_head_rotated(rot_dim, bias):
    c = Case(ENTRIES["spans"], 6, 2, 64, torch.bfloat16, seed=rot_dim, rot_dim=rot_dim, bias=bias)
    c.check(c.write())


@pytest.mark.parametrize("extra", [8, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_wider_rows_and_pages_apart(extra, dtype):
    c = Case(ENTRIES["spans"], 6, 2, 64, dtype, seed=3, extra=extra, gap=5)
    behind = c.raw[:, 2 * 2 * PAGE * 64:].clone()
    c.check(c.write())
    assert torch.equal(c.raw[:, 2 * 2 * PAGE * 64:], behind)
    odd = torch.empty(c.qkv.numel() + 1, dtype=dtype, device="cuda")[1:].view(c.qkv.shape)   # not on 16 bytes
    odd.copy_(c.qkv)
    c = Case(ENTRIES["spans"], 6, 2, 64, dtype, seed=3, extra=extra, gap=5)
    c.check(c.write(odd))


@pytest.mark.parametrize("spread,low", [(1e-3, -30), (30.0, -20), (3e4, -8), (1e-30, -112), (1e37, 100), (0.0, -6), (1.0, -112), (1.0, 60)])
def test_scales_that_grow_and_stay(spread, low):
    c = Case(ENTRIES["spans"] + ENTRIES["single tokens"], 4, 2, 64, torch.float32, seed=11, spread=spread, low=low, bias=False)
    c.check(c.write())


def test_a_far_position():
    """Angles of 32,000 radians: float32's own product would be off by 2^-24 of that, 2e-3."""
    c = Case([(32000, 3), (31999, 1)], 4, 2, 128, torch.float32, seed=5, bias=False)
    c.check(c.write())


def test_what_is_not_finite():
    c = Case([(3, 6), (64, 1), (10, 1)], 4, 2, 64, torch.float32, seed=9, rot_dim=0, bias=False)
    inf = float("inf")
    c.qkv[0, 4 * 64:4 * 64 + 4] = torch.tensor([inf, -inf, float("nan"), 2.0])
    c.qkv[1, 6 * 64:6 * 64 + 2] = torch.tensor([float("nan"), 3.0])
    c.qkv[6, 4 * 64:5 * 64] = inf          # a head of infinities alone takes the smallest scale
    c.qkv[7, 7 * 64:8 * 64] = float("nan")
    c.check(c.write())


def test_a_value_on_the_border():
    """amax = 448 * 2^e exactly takes e, the next float32 above it e + 1."""
    c = Case([(0, 1), (64, 1), (128, 1)], 1, 1, 16, torch.float32, seed=1, rot_dim=0, bias=False)
    c.qkv.zero_()
    for t, top in enumerate([448.0 * 2 ** -3, float(np.nextafter(np.float32(56.0), np.float32(100.0))), 449.0]):
        c.qkv[t, 16] = top
    c.check(c.write())
    pages = [int(c.table[c.slots[s], p // PAGE]) for s, p in enumerate(c.tok_pos)]
    assert [float(c.held_scales[p, 0, 0]) for p in pages] == [2.0 ** -3, 2.0 ** -2, 2.0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_one_at_a_time_or_all_at_once(dtype):
    """The page's scale is the same however its tokens came, and so is every value of at least 2^-6 of its unit: growth moves exponents only."""
    whole = Case([(0, 100)], 4, 2, 64, dtype, seed=21)
    whole.write()
    one = Case([(0, 100)], 4, 2, 64, dtype, seed=21)
    one.held_scales.fill_(2.0 ** 50)       # what an earlier holder left
    qkv, i32 = one.qkv.cuda(), dict(dtype=torch.int32, device="cuda")
    slots, cu = one.dev["slots"], torch.tensor([0, 1], **i32)
    q = torch.empty((1, 4 * 64), dtype=dtype, device="cuda")
    for t in range(100):
        ops.rope_cache_write_e4m3(qkv[t:t + 1], cu, torch.zeros(1, **i32), torch.tensor([t], **i32), slots, one.inv_freq.cuda(), 64, 4, q, one.site, 1, one.err,
                                  bias=one.bias.cuda())
    for p in range(2):
        page = int(one.table[one.slots[0], p])
        assert torch.equal(one.held_scales[page], whole.held_scales[page])
        rows = slice(0, 64 if p == 0 else 36)
        a, b = one.storage[page, :, :, rows].float(), whole.storage[page, :, :, rows].float()
        assert torch.equal(torch.where(b.abs() >= 2.0 ** -6, a, 0.0), torch.where(b.abs() >= 2.0 ** -6, b, 0.0))
        assert float((a - b).abs().max()) <= 2.0 ** -9   # below: twice half a step of 2^-9


def test_pages_that_are_not_held():
    c = Case([(10, 3), (70, 2)], 4, 2, 64, torch.bfloat16, seed=2)
    before = c.raw.clone()
    c.dev["table"].fill_(-1)
    q = c.write()
    assert int(c.err) == ops.ERR_NO_PAGE and torch.equal(c.raw, before) and bool((q != 7).any())
    c = Case([(10, 3)], 4, 2, 64, torch.bfloat16, seed=2)
    before = c.raw.clone()
    c.dev["tok_pos"].add_(64 * c.table.shape[1])   # behind the page table's last column
    c.write()
    assert int(c.err) == ops.ERR_NO_PAGE and torch.equal(c.raw, before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (4, 4, 128), (4, 2, 16), (6, 3, 96)])
@pytest.mark.parametrize("window", [0, 37, 64, 200])
def test_read_back(dtype, heads, kv_heads, dim, window):
    c = Case([(0, 130), (300, 7), (0, 5, True), (63, 1), (64, 1), (0, 64)], heads, kv_heads, dim, dtype, seed=4, gap=3)
    out = torch.full((len(c.codes) , 2 * kv_heads * PAGE * dim + 16), 5.0, dtype=dtype, device="cuda")
    pages = out[:, :-16].unflatten(1, (2, kv_heads, PAGE, dim))
    ops.cache_read_e4m3(pages, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, c.n, 330, c.err, window=window)
    want = torch.full(c.codes.shape, 5.0, dtype=dtype)
    for s, slot in enumerate(c.slots):
        if slot < 0:
            continue
        first, last = int(c.tok_pos[c.cu_q[s]]), int(c.tok_pos[c.cu_q[s + 1] - 1])
        for p in range(max(0, first - window + 1) if window else 0, last + 1):
            page = int(c.table[slot, p // PAGE])
            want[page, :, :, p % PAGE] = (c.codes[page, :, :, p % PAGE].double() * c.scales[page].double()[..., None]).to(dtype)
    assert torch.equal(pages.cpu(), want) and bool((out[:, -16:] == 5).all()) and int(c.err) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 10, 64, 130])
def test_read_back_of_long_spans_behind_short_windows(dtype, window):
    """More pages than a window has: a block takes several."""
    c = Case([(500, 700), (1000, 3), (65, 191), (0, 1)], 4, 2, 48, dtype, seed=5)
    out = torch.full(c.codes.shape, 5.0, dtype=dtype, device="cuda")
    ops.cache_read_e4m3(out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, c.n, 1200, c.err, window=window)
    want = torch.full(c.codes.shape, 5.0, dtype=dtype)
    for s in range(c.n):
        for p in range(max(0, int(c.tok_pos[c.cu_q[s]]) - window + 1), int(c.tok_pos[c.cu_q[s + 1] - 1]) + 1):
            page = int(c.table[c.slots[s], p // PAGE])
            want[page, :, :, p % PAGE] = (c.codes[page, :, :, p % PAGE].double() * c.scales[page].double()[..., None]).to(dtype)
    assert torch.equal(out.cpu(), want) and int(c.err) == 0


def test_read_back_is_exact_in_bfloat16():
    """Every code times scales at both ends of the range: the product has four bits, within bfloat16's exponents."""
    c = Case([(0, 64), (0, 64)], 1, 1, 16, torch.bfloat16, seed=4)
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    every = torch.where(torch.isnan(every.float()), torch.zeros(()), every.float()).to(torch.float8_e4m3fn)
    for s, e in enumerate((ref.LOW, ref.HIGH)):
        page = int(c.table[c.slots[s], 0])
        c.storage[page, 0, 0].view(torch.uint8).copy_(every.view(torch.uint8).repeat(4).view(64, 16).cuda())
        c.held_scales[page, 0, 0] = 2.0 ** e
    out = torch.zeros(c.codes.shape, dtype=torch.bfloat16, device="cuda")
    ops.cache_read_e4m3(out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, 2, 64, c.err)
    for s, e in enumerate((ref.LOW, ref.HIGH)):
        page = int(c.table[c.slots[s], 0])
        assert torch.equal(out[page, 0, 0].cpu().double(), every.double().repeat(4).view(64, 16) * 2.0 ** e)


def test_no_tokens_and_no_sequences():
    c = Case([(0, 1)], 4, 2, 64, torch.bfloat16)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.rope_cache_write_e4m3(torch.zeros((0, 8 * 64), dtype=torch.bfloat16, device="cuda"), one, empty, empty, empty, None, 0, 4,
                              torch.zeros((0, 256), dtype=torch.bfloat16, device="cuda"), c.site, 1, c.err)
    ops.cache_read_e4m3(torch.zeros(c.codes.shape, dtype=torch.bfloat16, device="cuda"), one, empty, empty, c.site, 0, 1, c.err)
    assert torch.equal(c.storage.cpu().view(torch.uint8), c.codes.view(torch.uint8))


@pytest.mark.parametrize("of", [0, 1, 7], ids=["of the first", "of the last", "of none"])
def test_a_row_behind_the_last_entry(of):
    """Whatever it says it is of."""
    c = Case([(70, 1), (5, 1)], 4, 2, 64, torch.bfloat16)
    more = lambda x, v: torch.cat((x, x.new_tensor([v])))   # noqa: E731
    qkv, q_out = torch.cat((c.qkv, c.qkv[:1] + 1)).cuda(), torch.full((3, 4 * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.rope_cache_write_e4m3(qkv, c.dev["cu_q"], more(c.dev["tok_seq"], of), more(c.dev["tok_pos"], 3), c.dev["slots"], c.inv_freq.cuda(), c.rot_dim, 4, q_out, c.site, 1,
                              c.err, bias=None if c.bias is None else c.bias.cuda())
    c.check(q_out[:2])
    assert bool((q_out[2] == 7).all()) and int(c.err) == 0


def test_rows_but_no_entry():
    c = Case([(0, 1)], 4, 2, 64, torch.bfloat16)
    none, one = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = torch.full((1, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    for most in (1, 70):
        ops.rope_cache_write_e4m3(c.qkv.cuda(), one, one, one, none, None, 0, 4, q_out, c.site, most, c.err)
    ops.attention_e4m3(q_out.clone(), q_out, one, one, none, c.site, 4, 0, 1, 0.125, 0, ops.E4m3Scratch("cuda"), c.err)
    assert bool((q_out == 7).all()) and torch.equal(c.storage.cpu().view(torch.uint8), c.codes.view(torch.uint8)) and int(c.err) == 0


def test_an_entry_longer_than_the_call_says():
    c = Case([(0, 9)], 4, 2, 64, torch.bfloat16)
    c.most = 4
    c.write()
    assert int(c.err) == ops.ERR_ROW_RANGE


def test_refusals():
    c = Case([(0, 3)], 4, 2, 64, torch.bfloat16)
    qkv, q = c.qkv.cuda(), torch.empty((3, 256), dtype=torch.bfloat16, device="cuda")
    d, freq = c.dev, c.inv_freq.cuda()

    def write(**change):
        a = dict(qkv=qkv, cu_q=d["cu_q"], tok_seq=d["tok_seq"], tok_pos=d["tok_pos"], slots=d["slots"], inv_freq=freq, rot_dim=64, n_heads=4, q_out=q, site=c.site,
                 max_q_len=3, err=c.err, bias=None)
        a.update(change)
        ops.rope_cache_write_e4m3(**a)
    for change in (dict(qkv=qkv.half()), dict(qkv=qkv.cpu()), dict(qkv=qkv[:, :-1]), dict(qkv=qkv.t().contiguous().t()), dict(q_out=q[:2]), dict(q_out=q.float()),
                   dict(tok_seq=d["tok_seq"].long()), dict(tok_seq=d["tok_seq"][:2]), dict(cu_q=d["cu_q"][:1]), dict(slots=d["slots"].long()),
                   dict(inv_freq=freq[:-1]), dict(inv_freq=freq.double()), dict(rot_dim=66), dict(n_heads=5), dict(n_heads=0), dict(max_q_len=0),
                   dict(bias=c.bias.cuda()[:-1]), dict(bias=c.bias.cuda().float()), dict(err=c.err.float()), dict(tok_pos=d["tok_pos"].cpu())):
        with pytest.raises(KernelError):
            write(**change)
    out = torch.zeros(c.codes.shape, dtype=torch.bfloat16, device="cuda")

    def read(**change):
        a = dict(out=out, cu_q=d["cu_q"], tok_pos=d["tok_pos"], slots=d["slots"], site=c.site, n_seqs=1, max_kv_len=3, err=c.err, window=0)
        a.update(change)
        ops.cache_read_e4m3(**a)
    for change in (dict(out=out.half()), dict(out=out[1:]), dict(out=out.cpu()), dict(out=out.transpose(0, 1)), dict(n_seqs=2), dict(window=-1), dict(max_kv_len=0),
                   dict(slots=d["slots"].cpu())):
        with pytest.raises(KernelError):
            read(**change)
    for args in ((c.storage.float(), c.held_scales, d["table"], 2, 64), (c.storage, c.held_scales.half(), d["table"], 2, 64), (c.storage, c.held_scales, d["table"].long(), 2, 64),
                 (c.storage, c.held_scales, d["table"], 1, 64), (c.storage, c.held_scales, d["table"], 2, 128), (c.storage, c.held_scales[1:], d["table"], 2, 64),
                 (c.storage[..., :24], c.held_scales, d["table"], 2, 24), (c.storage, c.held_scales, d["table"][0], 2, 64), (c.storage.cpu(), c.held_scales, d["table"], 2, 64)):
        with pytest.raises(KernelError):
            ops.E4m3SiteArgs(*args)
    write()
    read()
