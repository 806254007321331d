"""Python entries of the kernels for a sequence cache in 8 bits: written with the rotation, read back, attended over. The same manner as
`kernels.py`: checks on the host, raw device pointers, the current stream, error codes.

The cache holds an e4m3 code per element (`torch.float8_e4m3fn`) and a float32 power of two per page of 64 positions, plane (keys,
values) and kv head; an element stands for code * scale."""
from __future__ import annotations

from typing import Optional

import torch

from . import kernels
from .branches import PAGE_TOKENS, _F, _I, _LL, _P, _at, _function, _here, _native, _stream
from .kernels import KernelError, _check, _dev

E4M3_HEAD_DIMS = (16, 32, 48, 64, 80, 96, 112, 128)
E4M3_ROWS = 16     # most query rows of a block of the attention: tokens of a span times heads of a group
E4M3_WARPS = 4     # pages that a block has at work, and takes at the least where a sequence is cut (EA_WARPS)


class E4m3SiteArgs:
    """What the kernels need to address one schedule entry's keys and values in 8 bits. storage: float8_e4m3fn [pages, 2, kv_heads, 64,
    head_dim], scales: float32 [pages, 2, kv_heads] (a page of each dense, pages at any distance of 16 bytes' multiple), table: int32 [slots, columns]."""
    __slots__ = ("storage", "scales", "table", "kv_heads", "head_dim", "place")

    def __init__(self, storage: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, kv_heads: int, head_dim: int):
        _dev("cache", storage, torch.float8_e4m3fn, contiguous=False)
        _dev("scales", scales, torch.float32, contiguous=False)
        _dev("page table", table, torch.int32, contiguous=False)
        page = kv_heads * PAGE_TOKENS * head_dim
        if head_dim not in E4M3_HEAD_DIMS:
            raise KernelError(f"a cache in 8 bits has head sizes {', '.join(map(str, E4M3_HEAD_DIMS))}, not {head_dim}")
        if kv_heads <= 0 or storage.dim() != 5 or storage.shape[1:] != (2, kv_heads, PAGE_TOKENS, head_dim) or not storage[:1].is_contiguous():
            raise KernelError(f"a cache in 8 bits is [pages, 2, kv_heads, {PAGE_TOKENS}, head_dim], a page dense")
        if scales.shape != (storage.shape[0], 2, kv_heads) or not scales[:1].is_contiguous():
            raise KernelError("the scales of a cache in 8 bits are [pages, 2, kv_heads], a page dense")
        if storage.shape[0] > 1 and (storage.stride(0) < 2 * page or storage.stride(0) % 16 or scales.stride(0) < 2 * kv_heads):
            raise KernelError("the pages of a cache in 8 bits overlap, or do not begin on 16 bytes")
        if storage.data_ptr() % 16:
            raise KernelError("a cache in 8 bits begins on 16 bytes")
        if table.dim() != 2 or table.stride(1) != 1 or table.shape[0] < 1 or table.shape[1] < 1:
            raise KernelError("the page table is [slots, pages] with unit inner stride")
        if len({t.get_device() for t in (storage, scales, table)}) != 1:
            raise KernelError("a cache in 8 bits lies on one device")
        self.storage, self.scales, self.table, self.kv_heads, self.head_dim = storage, scales, table, kv_heads, head_dim
        one = storage.shape[0] == 1   # codes, scales, table, page_bytes, page_scales, table_stride, columns, n_slots, kv_heads, head_dim
        self.place = (storage.data_ptr(), scales.data_ptr(), table.data_ptr(), 2 * page if one else storage.stride(0), 2 * kv_heads if one else scales.stride(0),
                      table.stride(0), table.shape[1], table.shape[0], kv_heads, head_dim)


_SITE = (_P, _P, _P, _LL, _LL, _I, _I, _I, _I, _I)


def _batch(what: str, cu_q, tok_pos, slots, err) -> None:
    for name, t in (("cu_q", cu_q), ("tok_pos", tok_pos), ("slots", slots), ("err", err)):
        _dev(name, t, torch.int32)
    if cu_q.numel() != slots.numel() + 1:
        raise KernelError(f"{what}: cu_q has one element more than slots")


def rope_cache_write_e4m3(qkv: torch.Tensor, cu_q: torch.Tensor, tok_seq: torch.Tensor, tok_pos: torch.Tensor, slots: torch.Tensor,
                          inv_freq: Optional[torch.Tensor], rot_dim: int, n_heads: int, q_out: torch.Tensor, site: E4m3SiteArgs, max_q_len: int,
                          err: torch.Tensor, bias: Optional[torch.Tensor] = None, write_cache: bool = True, constants: bool = False) -> None:
    """`rope_cache_write` into a cache in 8 bits: qkv [T, (NH + 2 KVH) D] (bfloat16 or float32; perhaps the first columns of wider rows) with its bias, q and
    k heads rotated by position (split halves of the first rot_dim components; inv_freq None: not at all), q to q_out [T, NH D], k and v
    as codes. Entry s owns the tokens cu_q[s] .. cu_q[s + 1] - 1, at most max_q_len, at consecutive positions; a slot is in one entry at
    most, and no other sequence holds a page that it writes.

    A page that gets rows takes, per plane and head, the least power of two under which all their finite elements lie within +-448 (of 2^-112
    to 2^119), and no less than it has if it held rows before the new ones; those rows' codes are then rounded to the larger unit. Rounding is
    to nearest even, once, from float32. Infinities become +-448, NaN stays. Rows behind the new ones stay as they are; a padding
    entry (slot -1) writes its queries only, as does every entry with `write_cache` false. A padding entry may have more than max_q_len tokens; which of
    its queries are then written is left open.
    `constants` promises that no kernel in flight on the stream writes cu_q, tok_seq, tok_pos, slots, inv_freq or the page table (a bound model's step):
    they are then read while the kernel ahead ends."""
    if qkv.is_cuda:
        code = _native("rope_cache_write_e4m3", "cache_e4m3")(qkv, bias, cu_q, tok_seq, tok_pos, slots, inv_freq, q_out, err, site.storage, site.place, rot_dim,
                                                              n_heads, write_cache, max_q_len, constants)
        if code is not None:
            return _check(code, "rope_cache_write_e4m3")
    dtype = qkv.dtype
    is_bf16 = kernels._is_bf16(dtype)
    kernels._rows("qkv", qkv)
    _dev("q_out", q_out, dtype)
    _dev("tok_seq", tok_seq, torch.int32)
    _batch("rope_cache_write_e4m3", cu_q, tok_pos, slots, err)
    n, d, kv_heads = qkv.shape[0], site.head_dim, site.kv_heads
    width = (n_heads + 2 * kv_heads) * d
    if n_heads <= 0 or qkv.shape[1] < width or q_out.shape != (n, n_heads * d):
        raise KernelError("rope_cache_write_e4m3: qkv/q_out widths do not match the head counts")
    if tok_seq.numel() != n or tok_pos.numel() != n:
        raise KernelError("rope_cache_write_e4m3: tok_seq and tok_pos have one element per token")
    if bias is not None:
        _dev("bias", bias, dtype)
        if bias.numel() != width:
            raise KernelError("rope_cache_write_e4m3: bias must have one element per projection column")
    if inv_freq is not None:
        _dev("inv_freq", inv_freq, torch.float32)
        if not 0 <= rot_dim <= d or inv_freq.numel() * 2 != rot_dim:
            raise KernelError("rope_cache_write_e4m3: inv_freq must hold rot_dim / 2 frequencies, rot_dim at most head_dim")
    if n and max_q_len <= 0:
        raise KernelError("rope_cache_write_e4m3: max_q_len is the most tokens of an entry")
    _here("rope_cache_write_e4m3", qkv, cu_q, tok_seq, tok_pos, slots, inv_freq, q_out, site.storage, site.scales, site.table, err, bias)
    if n == 0 or slots.numel() == 0:
        return
    _check(_function("cache_e4m3", "qf_rope_cache_write_e4m3", _I, _P, _P, _LL, _P, _P, _P, _P, _P, _I, _I, _P, *_SITE, _I, _I, _I, _I, _I, _P, _P)(
        is_bf16, qkv.data_ptr(), _at(bias), qkv.stride(0), cu_q.data_ptr(), tok_seq.data_ptr(), tok_pos.data_ptr(), slots.data_ptr(), _at(inv_freq), rot_dim,
        n_heads, q_out.data_ptr(), *site.place, bool(write_cache), n, slots.numel(), max_q_len, bool(constants), err.data_ptr(), _stream()), "rope_cache_write_e4m3")


def cache_read_e4m3(out: torch.Tensor, cu_q: torch.Tensor, tok_pos: torch.Tensor, slots: torch.Tensor, site: E4m3SiteArgs, n_seqs: int, max_kv_len: int,
                    err: torch.Tensor, window: int = 0) -> None:
    """The rows that a batch's sequences hold, back as values: out [pages, 2, kv_heads, 64, head_dim] (bfloat16 or float32, exact in both), at the
    page numbers of the cache, so that its page table serves both. Of entry s the rows up to its last new token's, from the first that a
    window of `window` positions (0: all) leaves its first one; every other row of `out` stays as it is. `max_kv_len`: an upper bound of any
    sequence's length."""
    if out.is_cuda:
        code = _native("cache_read_e4m3", "cache_e4m3")(out, cu_q, tok_pos, slots, err, site.storage, site.place, n_seqs, max_kv_len, window)
        if code is not None:
            return _check(code, "cache_read_e4m3")
    is_bf16 = kernels._is_bf16(out.dtype)
    _dev("out", out, contiguous=False)
    _batch("cache_read_e4m3", cu_q, tok_pos, slots, err)
    storage, kv_heads, d = site.storage, site.kv_heads, site.head_dim
    if out.shape != storage.shape or not out[:1].is_contiguous() or (out.shape[0] > 1 and (out.stride(0) < 2 * kv_heads * PAGE_TOKENS * d or out.stride(0) % 8)):
        raise KernelError("cache_read_e4m3: out has the cache's shape, a page dense")
    if out.data_ptr() % 16:
        raise KernelError("cache_read_e4m3: out begins on 16 bytes")
    if slots.numel() != n_seqs or window < 0 or (n_seqs and max_kv_len <= 0):
        raise KernelError("cache_read_e4m3: wants n_seqs slots, a window of 0 or more and a bound on the lengths")
    _here("cache_read_e4m3", out, cu_q, tok_pos, slots, storage, site.scales, site.table, err)
    if n_seqs == 0:
        return
    pages = min(-(-int(max_kv_len) // PAGE_TOKENS), site.table.shape[1])
    _check(_function("cache_e4m3", "qf_cache_read_e4m3", _I, _P, _LL, _P, _P, _P, *_SITE, _I, _I, _I, _P, _P)(
        is_bf16, out.data_ptr(), 2 * kv_heads * PAGE_TOKENS * d if out.shape[0] == 1 else out.stride(0), cu_q.data_ptr(), tok_pos.data_ptr(), slots.data_ptr(),
        *site.place, n_seqs, pages, window, err.data_ptr(), _stream()), "cache_read_e4m3")


# Rows (tokens of a span times heads of a group) up to which `attention_e4m3` is the faster way in bfloat16: a tile of 16 rows reads the cache anew, while
# `cache_read_e4m3` with the kernels for prompts reads and writes every position once. Microseconds, codes / read back and attended over, seven heads to a
# group, spans of 4, 16, 32 and 64 tokens: 8 sequences behind 4,000 tokens, 2 kv heads of 64 15 / 42, 28 / 42, 42 / 42, 71 / 42, 4 of 128 30 / 89, 63 / 90,
# 111 / 91, 194 / 92; behind 300 12 / 11, 13 / 11, 13 / 11, 21 / 12 and 16 / 18, 17 / 18, 29 / 18, 50 / 20. Length and number of sequences move the border, and the rule has
# neither: 32 sequences behind 4,000 tokens 30 / 152, 71 / 153, 126 / 168, 237 / 181 and 74 / 361, 201 / 363, 377 / 366, 725 / 368 (spans of 32 at heads of 64 would gain a
# quarter from codes), behind 300 13 / 15, 21 / 15, 36 / 17, 59 / 21 and 15 / 48, 52 / 49, 85 / 53, 151 / 60 (spans of 16 there lose a third to them). In float32, where the
# other way is `attention_generic`, codes were faster at all sizes tried: one span of 256 behind 4,000 tokens 48 / 228 and 174 / 571, a prompt of 2,000 149 / 246 and 581 / 867;
# longer ones were not tried.
E4M3_PAYS_ROWS = 128


def attention_e4m3_pays(dtype: torch.dtype, max_q_len: int, group: int) -> bool:
    """Whether a step of up to `max_q_len` tokens per sequence, `group` query heads to a kv head, is to attend over the codes."""
    return dtype is torch.float32 or max_q_len * group <= E4M3_PAYS_ROWS


class E4m3Scratch:
    """Workspaces of `attention_e4m3`: the runs' sums with their maxima, and ticket counters (kept zero between calls by the kernel itself). Sized for
    as many blocks as the device holds at once, whatever the lengths, so that only another head size or more rows of a block ask for more (1 to 5 MB). One
    instance serves calls that run one after another on one stream; what is captured into a graph has one of its own. Should a captured call
    share one all the same, its replays take their turn like calls: what a call outgrows is kept as long as the instance, because a graph may hold its address."""
    TICKETS = 4096   # four for each of 1,024 blocks, the most that a launch has; zero from here on, where memory that a capture hands out is not

    def __init__(self, device):
        self.device = torch.device(device)
        self.part_o = self.part_ml = None
        self.tickets = torch.zeros(self.TICKETS, dtype=torch.int32, device=self.device)
        self.outgrown: list = []

    def ensure(self, blocks: int, head_dim: int, rows: int) -> None:
        rows *= 2 * blocks
        for name, size in (("part_o", rows * -(-head_dim // 32) * 32), ("part_ml", 2 * rows)):
            held = getattr(self, name)
            if held is None or held.numel() < size:
                if held is not None:
                    self.outgrown.append(held)
                setattr(self, name, torch.empty(size, dtype=torch.float32, device=self.device))


_block_slots: dict = {}


def _slots_of(is_bf16: int, head_dim: int, rows: int) -> int:
    key = (torch._C._cuda_getDevice(), is_bf16, head_dim, rows)
    n = _block_slots.get(key)
    if n is None:
        n = _function("attention_e4m3", "qf_attention_e4m3_slots", _I, _I, _I)(is_bf16, head_dim, rows)
        if n <= 0:
            raise KernelError(f"attention_e4m3: the device has no room for a block of head size {head_dim}")
        _block_slots[key] = n
    return n


def attention_e4m3(q: torch.Tensor, out: torch.Tensor, cu_q: torch.Tensor, tok_pos: torch.Tensor, slots: torch.Tensor, site: E4m3SiteArgs, n_heads: int,
                   n_seqs: int, max_q_len: int, scale: float, window: int, scratch: E4m3Scratch, err: torch.Tensor, max_kv_len: Optional[int] = None,
                   constants: bool = False) -> None:
    """Causal grouped-query attention of a step's tokens over a cache in 8 bits: single tokens, and spans (every 16 rows of tokens times the heads of
    a group read the cache anew, see `attention_e4m3_pays`). q, out [T, n_heads * head_dim], bfloat16 or
    float32; query head i reads kv head i // (n_heads / kv_heads); key j is visible to a token at p iff max(0, p - window + 1) <= j <= p
    (window 0: all up to p). Entry s owns the tokens cu_q[s] .. cu_q[s + 1] - 1, at consecutive positions, at most max_q_len; an entry may have none, and a
    padding entry (slot -1), of any number of tokens, gets zeros. `max_kv_len`: an upper bound of any sequence's length after the step (None: as long as the page
    table has room for). `constants` promises that no kernel in flight on the stream writes cu_q, tok_pos, slots, the page table or a page before an
    entry's first new token's (a bound model's step): they are then read while the kernel ahead ends."""
    if q.is_cuda:
        code = _native("attention_e4m3", "attention_e4m3")(q, out, cu_q, tok_pos, slots, err, site.storage, site.place, scratch.part_o, scratch.part_ml, scratch.tickets,
                                                           n_heads, n_seqs, max_q_len, scale, window, 1 << 40 if max_kv_len is None else max_kv_len, constants)
        if code is not None:
            return _check(code, "attention_e4m3")
    dtype, d, kv_heads = q.dtype, site.head_dim, site.kv_heads
    is_bf16 = kernels._is_bf16(dtype)
    _dev("q", q)
    _dev("out", out, dtype)
    _batch("attention_e4m3", cu_q, tok_pos, slots, err)
    if n_heads <= 0 or n_heads % kv_heads:
        raise KernelError(f"attention_e4m3: {n_heads} heads do not divide into {kv_heads} groups")
    if q.dim() != 2 or q.shape[1] != n_heads * d or out.shape != q.shape:
        raise KernelError("attention_e4m3: q/out widths do not match the head count")
    if q.data_ptr() % 16 or out.data_ptr() % 16:
        raise KernelError("attention_e4m3: q and out begin on 16 bytes")
    if slots.numel() != n_seqs or tok_pos.numel() != q.shape[0] or window < 0:
        raise KernelError("attention_e4m3: wants n_seqs slots, a position per token and a window of 0 or more")
    if n_seqs and (max_q_len <= 0 or (max_kv_len is not None and max_kv_len <= 0)):
        raise KernelError("attention_e4m3: max_q_len and max_kv_len bound an entry's tokens and its sequence's length")
    _here("attention_e4m3", q, out, cu_q, tok_pos, slots, site.storage, site.scales, site.table, err)
    if q.shape[0] == 0 or n_seqs == 0:
        return
    columns = site.table.shape[1]
    most = columns if max_kv_len is None else min(columns, -(-int(max_kv_len) // PAGE_TOKENS))
    if window > 0:
        most = min(most, -(-(window + max_q_len - 1) // PAGE_TOKENS) + 1)
    rows = min(max_q_len, q.shape[0]) * (n_heads // kv_heads)
    block_rows = 8 if rows <= 8 else E4M3_ROWS
    chunks = -(-rows // block_rows)
    block_slots = _slots_of(is_bf16, d, block_rows)
    blocks = min(block_slots, n_seqs * kv_heads * chunks * -(-most // E4M3_WARPS))
    scratch.ensure(block_slots, d, block_rows)
    _here("attention_e4m3: scratch", scratch.part_o, scratch.tickets)
    _check(_function("attention_e4m3", "qf_attention_e4m3", _I, _P, _P, _P, _P, _P, *_SITE, _I, _I, _I, _I, _I, _I, _I, _I, _I, _F, _I, _I, _P, _P, _P, _P, _P)(
        is_bf16, q.data_ptr(), out.data_ptr(), cu_q.data_ptr(), tok_pos.data_ptr(), slots.data_ptr(), *site.place, n_heads, n_seqs, q.shape[0],
        max_q_len == 1 and q.shape[0] == n_seqs, block_rows, chunks, most, blocks, block_slots, scale, window, bool(constants), scratch.part_o.data_ptr(), scratch.part_ml.data_ptr(), scratch.tickets.data_ptr(), err.data_ptr(), _stream()), "attention_e4m3")
