"""Python entries of the kernels for several continuations of one prompt: copies of cache pages, attention of sequences whose
caches begin with the same pages, verification of drafted tokens. The same manner as `kernels.py`: checks on the host, raw device
pointers, the current stream, error codes."""
from __future__ import annotations

import ctypes
import threading
from array import array
from itertools import chain
from typing import Optional, Sequence

import numpy as np
import torch

from ..csrc import library
from . import host, kernels
from .kernels import KernelError, _check, _dev

PAGE_TOKENS = 64   # positions of a cache page (QF_PAGE of the kernels, and what the cache hands out)
_P, _I, _LL, _ULL, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_ulonglong, ctypes.c_float
_functions: dict = {}   # exported functions with their argument types (numbers are then converted by the call itself)


def _function(lib: str, name: str, *types):
    fn = _functions.get(name)
    if fn is None:
        fn = getattr(library(lib), name)
        fn.argtypes, fn.restype = types, _I
        _functions[name] = fn
    return fn


def _native(name: str, lib: str):
    """The native function of an entry below. It checks and launches where everything is in order; what it answers None for, the entry checks and launches
    itself, in Python."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = host.entry(name, lib)
    return fn


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _here(what: str, *tensors) -> None:
    """The tensors lie on the current device, whose current stream the kernels run on."""
    current = -1
    for t in tensors:
        if t is not None and (t.get_device() != current or current < 0):
            if not t.is_cuda:
                raise KernelError(f"{what}: a tensor is on {t.device}: the kernels of this library run on CUDA devices only")
            if current < 0:
                current = torch._C._cuda_getDevice()
            if t.get_device() == current:
                continue
            raise KernelError(f"{what}: a tensor is on {t.device}, the current device is cuda:{current}")


# ---------------------------------------------------------------------------------------------------------------- pages
_MOVES_WRONG = {-1: "a move names a page outside 0 .. {pages}", -2: "a move names rows outside 0 .. {rows}", -3: "a page is the target of two moves",
                -4: "a page is the source of one move and the target of another", -5: "no memory for checking the moves"}


def _flat_moves(moves, n_rows: int) -> array:
    try:
        if isinstance(moves, np.ndarray):
            moves = moves.tolist()
        widths = set(map(len, moves))
        if not widths <= {3}:
            if widths != {2}:
                raise KernelError("copy_pages: moves are (from, to) or (from, to, rows)")
            moves = [(source, target, n_rows) for source, target in moves]
        return array("i", chain.from_iterable(moves))
    except (TypeError, OverflowError) as exc:
        raise KernelError(f"copy_pages: moves are (from, to) or (from, to, rows), small whole numbers ({exc})") from None


def _moves_error(code: int, n_pages: int, n_rows: int) -> KernelError:
    return KernelError("copy_pages: " + _MOVES_WRONG[code].format(pages=n_pages - 1, rows=n_rows))


def page_moves(moves, n_pages: int, n_rows: int) -> np.ndarray:
    """`moves` as int32 [n, 3] (from, to, rows), checked: pages 0 .. n_pages - 1, rows 0 .. n_rows (whole pages where the moves name
    none), no page a target twice, none both a source and a target."""
    flat = _flat_moves(moves, n_rows)
    code = _function("page_copy", "qf_page_moves_check", _P, _I, _I, _I)(flat.buffer_info()[0], len(flat) // 3, n_pages, n_rows)
    if code:
        raise _moves_error(code, n_pages, n_rows)
    return np.array(flat, dtype=np.int32).reshape(-1, 3)


def copy_pages(storage: torch.Tensor, moves) -> None:
    """Copies rows of pages inside `storage`, for every schedule entry at once. storage: [entries, pages, ..., rows, width] of any dtype
    (a page dense, entries and pages at any distance; a storage of two or three dimensions has pages of one row). moves: (from, to, rows)
    or (from, to) on the host: the first `rows` rows of page `from`, in each of its planes and heads, become those of page `to`; the
    others stay as they are. No page may be the target of two moves, or both a source and a target."""
    if storage.is_cuda:
        code = _native("copy_pages", "page_copy")(storage, moves)
        if code is not None:
            if code < 0:
                raise _moves_error(code, storage.shape[1], storage.shape[-2] if storage.dim() >= 4 else 1)
            kernels.launches += -(-len(moves) // 1024) - 1
            return _check(code, "copy_pages")
    shape, strides = storage.shape, storage.stride()
    if len(shape) < 2:
        raise KernelError("copy_pages: storage has entries and pages")
    entries, pages = shape[0], shape[1]
    n_rows, width = (shape[-2], shape[-1]) if len(shape) >= 4 else (1, shape[2] if len(shape) == 3 else 1)
    segments, want = 1, 1
    for size, stride in zip(shape[:1:-1], strides[:1:-1]):
        if size != 1 and stride != want:
            raise KernelError("copy_pages: a page of the storage is not contiguous")
        want *= size
    for size in shape[2:-2]:
        segments *= size
    page = want
    e_stride, p_stride = strides[0] if entries > 1 else 0, strides[1] if pages > 1 else 0
    if (pages > 1 and p_stride < page) or (entries > 1 and e_stride < page) or (
            entries > 1 and pages > 1 and e_stride < (pages - 1) * p_stride + page and p_stride < (entries - 1) * e_stride + page):
        if page > 0:
            raise KernelError("copy_pages: pages of the storage overlap")
    if entries > 65535:
        raise KernelError(f"copy_pages: {entries} entries are more than a launch takes (65,535)")
    _here("copy_pages", storage)
    flat, item = _flat_moves(moves, n_rows), storage.element_size()
    n, base, row = len(flat) // 3, storage.data_ptr(), width * item
    e_bytes, p_bytes = e_stride * item, p_stride * item
    low = base | row | e_bytes | p_bytes
    unit = 16 if not low & 15 else 4 if not low & 3 else 2 if not low & 1 else 1
    code = _function("page_copy", "qf_copy_pages", _P, _I, _I, _I, _LL, _LL, _I, _LL, _LL, _I, _P, _I, _P)(
        base, entries, pages, n_rows, e_bytes, p_bytes, segments if page else 0, n_rows * row, row, unit, flat.buffer_info()[0], n, _stream())
    if code < 0:
        raise _moves_error(code, pages, n_rows)
    kernels.launches += -(-n // 1024) - 1 if page and entries else -1
    _check(code, "copy_pages")


# ---------------------------------------------------------------------------------------------------------------- attention
SHARED_MAX_HEAD_DIM = 256
SHARED_MAX_SEQS = 2048
SHARED_TEAM = 4   # warps of a block of the parts' kernel (SH_TEAM)


class SharedPrefix:
    """Which sequences of a batch begin with the same cache pages. groups: (batch entries, pages) each; the entries of a group hold the
    same page ids in the first `pages` places of their page tables, whole pages that none of them writes any more (`SequenceCache.fork`
    makes such sequences, `SequenceCache.shared_groups` finds them). An entry is in one group at most; groups without pages are left
    out. Stays valid while these pages are shared, however long the sequences get, also where some of them have ended (slot -1).
    `bound_pages`: the most pages that any group may share when what is shared is replaced later (`load`) under a captured graph."""

    def __init__(self, groups: Sequence[tuple], n_seqs: int, device, bound_pages: int = 0):
        self.n_seqs = int(n_seqs)
        if self.n_seqs <= 0:
            raise KernelError("SharedPrefix: a batch has at least one sequence")
        kept = [([int(e) for e in entries], int(pages)) for entries, pages in groups]
        named = [e for entries, _ in kept for e in entries]
        if any(not entries or pages < 0 for entries, pages in kept):
            raise KernelError("SharedPrefix: a group has entries, and no fewer than 0 pages")
        if len(set(named)) != len(named) or any(not 0 <= e < self.n_seqs for e in named):
            raise KernelError(f"SharedPrefix: an entry is in two groups or outside 0 .. {self.n_seqs - 1}")
        self.groups = [g for g in kept if g[1] > 0]
        entry_pages, entry_group, members, begin = [0] * self.n_seqs, [-1] * self.n_seqs, [], [0]
        for g, (entries, pages) in enumerate(self.groups):
            members += entries
            begin.append(len(members))
            for e in entries:
                entry_pages[e], entry_group[e] = pages, g
        pages = [p for _, p in self.groups]
        self.most_pages = max(pages, default=0)
        if 0 < bound_pages < self.most_pages:
            raise KernelError(f"SharedPrefix: a group shares {self.most_pages} pages, more than the bound of {bound_pages}")
        self.bound_pages = max(self.most_pages, int(bound_pages))
        self.columns = 1 << 30   # the fewest that a page table of its calls has had
        self.saved_pages = self._saved()
        self.least_pages = 0 if bound_pages else min(entry_pages)
        sizes = (self.n_seqs, self.n_seqs, len(members), len(begin), len(pages))
        packed = torch.tensor(entry_pages + entry_group + members + begin + pages, dtype=torch.int32).to(device)
        self.entry_pages, self.entry_group, self.members, self.begin, self.pages = packed.split(sizes)
        self.sizes: dict = {}   # shape of an attention -> what its plans and workspaces are sized by

    def __len__(self) -> int:
        return len(self.groups)

    def _saved(self) -> int:
        """Pages that the batch's sequences read for themselves where nothing is shared, and need not."""
        return sum((len(entries) - 1) * pages for entries, pages in self.groups)

    def addresses(self) -> tuple:
        return tuple(t.data_ptr() for t in (self.entry_pages, self.entry_group, self.members, self.begin, self.pages))

    def shape(self) -> tuple:
        """What the launches go by: the batch, the groups' members, the bound on their pages."""
        return (self.n_seqs, tuple(len(entries) for entries, _ in self.groups), self.bound_pages)

    def load(self, other: "SharedPrefix") -> None:
        """Take over what `other`, of the same members per group and within the bound, says is shared; the addresses stay."""
        if other.shape()[:2] != self.shape()[:2] or other.most_pages > min(self.bound_pages, self.columns):
            raise KernelError("SharedPrefix: what is loaded has other groups, or more pages than the bound or the page table has room for")
        for name in ("entry_pages", "entry_group", "members", "begin", "pages"):
            getattr(self, name).copy_(getattr(other, name))
        self.groups, self.most_pages, self.saved_pages = other.groups, other.most_pages, other.saved_pages


# A call costs more than `attention_decode` with its plan made before (two launches and a plan of its own: 9 to 13 microseconds against 4 to 7), which what it
# does not read has to make up for. Microseconds, one group with 70 tokens each of their own, decode / shared (saved bytes): 14 heads over 2 of 64, 64
# sequences x 64 pages 21.0 / 15.0 (132 MB), 24 x 64 11.4 / 14.1 (48 MB), 256 x 8 24.6 / 14.1 (67 MB); 28 over 4 of 128, 8 x 64 17.0 / 15.4 (57 MB), 16 x 16
# 12.2 / 13.7 (31 MB), 64 x 8 20.4 / 15.4 (64 MB), 256 x 64 305 / 41. The kernels for other sizes and float32 take as long as the longest sequence:
# `attention_generic` / shared, float32, 14 over 2 of 64, 8 x 1 page 9.6 / 10.5, 8 x 4 17.4 / 10.7, 2 x 64 171 / 14; 32 x 4, 16 over 2 of 128, 27.8 / 24.5.
SHARED_PAYS_BYTES = 56_000_000
SHARED_PAYS_PAGES = 4


def attention_shared_pays(share: SharedPrefix, dtype, kv_heads: int, head_dim: int) -> bool:
    """Whether `attention_shared` takes this shape, and is faster than the attention that reads every sequence's pages for itself."""
    if share.n_seqs > SHARED_MAX_SEQS or head_dim > SHARED_MAX_HEAD_DIM:
        return False
    if dtype is torch.bfloat16 and head_dim in kernels.FAST_ATTENTION_HEAD_DIMS:
        return share.saved_pages * kv_heads * head_dim * 4 * PAGE_TOKENS >= SHARED_PAYS_BYTES
    return share.most_pages >= SHARED_PAYS_PAGES


class SharedScratch:
    """Workspaces of `attention_shared`: the parts' sums with their maxima, and how many parts a row has. One instance serves calls that run
    one after another on one stream; what is captured into a graph has one of its own."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.part_o = self.part_ml = self.part_n = None

    def ensure(self, n_seqs: int, parts: int, head_dim: int) -> None:
        if self.part_o is None or self.part_o.numel() < parts * head_dim:
            self.part_o = torch.empty(parts * head_dim, dtype=torch.float32, device=self.device)
        if self.part_ml is None or self.part_ml.numel() < parts * 2:
            self.part_ml = torch.empty(parts * 2, dtype=torch.float32, device=self.device)
        if self.part_n is None or self.part_n.numel() < n_seqs:
            self.part_n = torch.empty(n_seqs, dtype=torch.int32, device=self.device)


def _shared_sizes(dtype, head_dim: int, kv_heads: int, n_heads: int, share: SharedPrefix, own_pages: int) -> tuple:
    """(units, tile records, most shared parts, most own parts of a row): bounds of what the device's plan can come to, whatever the
    lengths. It gives a warp at least `pages x tiles x kv heads / warps` pages, so units of a block's run cover, up to twice, no more
    than the warps there are, and so do single warps' records but for one more per item. Tile records: the pairs of tiles, uncut."""
    held = share.sizes.get((dtype, head_dim, kv_heads, n_heads, own_pages))
    if held is not None:
        return held
    sizes = (_I * 8)()
    code = _function("attention_shared", "qf_attention_shared_shape", _I, _I, _P)(int(dtype == torch.bfloat16), head_dim, sizes)
    if code:
        raise KernelError(f"attention_shared: CUDA error {code} when asked for its sizes")
    row_tile, warps, team, most, tile_rows, tile_work, sms, tile_ints = sizes
    group_heads = n_heads // kv_heads

    def parts(pages: int, tiles: int) -> int:
        return max(team, min(most, -(-pages // team), warps // (team * kv_heads * tiles) + 1))
    own_tiles = -(-group_heads // row_tile)
    tiles = [-(-len(entries) * group_heads // row_tile) for entries, _ in share.groups]
    most_shared = max((parts(share.bound_pages, t) for t in tiles), default=0)
    rows = [len(entries) * group_heads for entries, _ in share.groups]
    pairs = [-(-r // 256) for r in rows if r >= tile_rows and r * share.bound_pages >= tile_work]
    if not tile_rows or 2 * share.n_seqs + 6 * len(share) > tile_ints:
        pairs = []
    if pairs:   # (everything else is cut for single warps then)
        most_shared = max(most_shared, min(most // 4, share.bound_pages))
    for n in pairs:
        most_shared = max(most_shared, min(most, -(-share.bound_pages // 4), sms // (kv_heads * n) + 1))
    singles = warps // kv_heads + 1 + sum(tiles) + share.n_seqs * own_tiles
    units = 2 * warps // (team * kv_heads) + 2 + -(-singles // SHARED_TEAM)
    if len(share.sizes) >= 64:
        share.sizes.clear()
    held = share.sizes[dtype, head_dim, kv_heads, n_heads, own_pages] = (
        units, sum(pairs), most_shared, min(most // 2, own_pages) if pairs else parts(own_pages, own_tiles))
    return held


def _own_pages(max_kv_len: Optional[int], table: torch.Tensor, share: SharedPrefix) -> int:
    """The most pages that a sequence has to itself."""
    return max(1, (table.shape[1] if max_kv_len is None else -(-int(max_kv_len) // PAGE_TOKENS)) - share.least_pages)


def _batch_refused(cu_q, tok_pos, slots, n_seqs: int, kv_heads: int, n_heads: int, head_dim: int, dtype, share: SharedPrefix) -> None:
    """Raises what is wrong with a batch, its shape or what it shares; returns if nothing is."""
    i32 = torch.int32
    if not (cu_q.dtype is i32 and tok_pos.dtype is i32 and slots.dtype is i32 and cu_q.is_contiguous() and tok_pos.is_contiguous() and slots.is_contiguous()):
        for name, t in (("cu_q", cu_q), ("tok_pos", tok_pos), ("slots", slots)):
            _dev(name, t, i32)
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise KernelError(f"attention_shared: dtype {dtype} is not supported (bfloat16 or float32)")
    if not 0 < head_dim <= SHARED_MAX_HEAD_DIM:
        raise KernelError(f"attention_shared: head_dim {head_dim} > {SHARED_MAX_HEAD_DIM} is not supported")
    if kv_heads <= 0 or n_heads <= 0 or n_heads % kv_heads:
        raise KernelError(f"attention_shared: {n_heads} heads do not divide into {kv_heads} groups")
    if not 0 < n_seqs <= SHARED_MAX_SEQS:
        raise KernelError(f"attention_shared: a batch of {n_seqs} sequences is not supported (1 to {SHARED_MAX_SEQS})")
    if share.n_seqs != n_seqs or slots.numel() != n_seqs or cu_q.numel() != n_seqs + 1 or tok_pos.numel() != n_seqs:
        raise KernelError("attention_shared: wants exactly one token per sequence, and a SharedPrefix of this batch")


def attention_shared(q: torch.Tensor, out: torch.Tensor, cu_q: torch.Tensor, tok_pos: torch.Tensor, slots: torch.Tensor, site, n_heads: int,
                     n_seqs: int, scale: float, share: SharedPrefix, scratch: SharedScratch, err: torch.Tensor,
                     max_kv_len: Optional[int] = None, sinks: Optional[torch.Tensor] = None) -> None:
    """Attention of ONE new token per sequence over its cache, where sequences share their first pages (`share`): what they share is read
    once for all of them. The result is that of `attention_decode`: query head i reads kv head i // (n_heads / kv_heads), key j is visible
    iff j <= the token's position (a token that stands inside the pages that it shares has them read for itself alone). bfloat16 or float32, head sizes up to 256 (bfloat16 of 32, 64, 96 and 128 on tensor cores). A padding
    entry (slot -1) gets zeros. `max_kv_len`: an upper bound of any sequence's length after the step (None: as long as the page table
    has room for); it sizes the workspaces and the launch. `sinks` (float32 [n_heads]): a logit per head that joins the softmax's denominator
    once, with no key and no value."""
    storage, table, d, kv_heads, dtype = site.storage, site.table, site.head_dim, site.kv_heads, q.dtype
    if table.dim() == 2 and table.shape[1] < share.columns:
        share.columns = table.shape[1]   # (a graph of this call reads no further, whatever is loaded later)
    if q.is_cuda and table.dim() == 2:
        sizes = share.sizes.get((dtype, d, kv_heads, n_heads, _own_pages(max_kv_len, table, share)))   # (there from the second call on)
        if sizes is not None:
            code = _native("attention_shared", "attention_shared")(
                q, out, cu_q, tok_pos, slots, storage, table, share.entry_pages, share.entry_group, share.members, share.begin, share.pages, scratch.part_o,
                scratch.part_ml, scratch.part_n, sinks, err, site.page_elems, kv_heads, d, n_heads, n_seqs, scale, len(share.groups), share.most_pages, *sizes)
            if code is not None:
                kernels.launches += 1
                return _check(code, "attention_shared")
    _batch_refused(cu_q, tok_pos, slots, n_seqs, kv_heads, n_heads, d, dtype, share)
    if not (out.dtype is dtype and storage.dtype is dtype and q.is_contiguous() and out.is_contiguous() and table.dtype is torch.int32
            and err.dtype is torch.int32):
        for name, t, of, dense in (("q", q, dtype, True), ("out", out, dtype, True), ("cache", storage, dtype, False), ("page table", table, torch.int32, False),
                                   ("err", err, torch.int32, True)):
            _dev(name, t, of, dense)
    if q.shape != (n_seqs, n_heads * d) or out.shape != q.shape:
        raise KernelError("attention_shared: wants exactly one token per sequence, q and out [n_seqs, n_heads * head_dim]")
    page, strides = kv_heads * PAGE_TOKENS * d, storage.stride()
    if len(strides) != 5 or storage.shape[1:] != (2, kv_heads, PAGE_TOKENS, d) or (strides[1:] != (page, PAGE_TOKENS * d, d, 1) and not storage[:1].is_contiguous()) or site.page_elems < 2 * page:
        raise KernelError(f"attention_shared: the cache is [pages, 2, kv_heads, {PAGE_TOKENS}, head_dim], a page dense")
    if table.dim() != 2 or table.stride(1) != 1:
        raise KernelError("attention_shared: the page table is [slots, pages] with unit inner stride")
    if share.most_pages > table.shape[1]:
        raise KernelError(f"attention_shared: a group shares {share.most_pages} pages, the page table has room for {table.shape[1]}")
    q_at, storage_at = q.data_ptr(), storage.data_ptr()
    if dtype is torch.bfloat16 and d in kernels.FAST_ATTENTION_HEAD_DIMS and (q_at % 16 or storage_at % 16 or site.page_elems % d):
        raise KernelError("attention_shared: q and the cache begin on 16 bytes, and a page holds whole rows")
    if sinks is not None:
        _dev("sinks", sinks, torch.float32)
        if sinks.numel() != n_heads:
            raise KernelError("attention_shared: sinks must hold one float32 per query head")
    _here("attention_shared", q, out, cu_q, tok_pos, slots, storage, table, share.entry_pages, err, sinks)
    units, tiles, most_shared, most_own = _shared_sizes(dtype, d, kv_heads, n_heads, share, _own_pages(max_kv_len, table, share))
    scratch.ensure(n_seqs, n_seqs * n_heads * (most_shared + most_own), d)
    code = _function("attention_shared", "qf_attention_shared", _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _P, _LL, _I, _I, _I, _I, _I, _F, _P,
                     _P, _P, _P, _P, _P)(
        dtype is torch.bfloat16, q_at, out.data_ptr(), tok_pos.data_ptr(), slots.data_ptr(), *share.addresses(), len(share.groups), units, tiles, most_shared,
        most_own, storage_at, table.data_ptr(), site.page_elems, site.table_stride, kv_heads, d, n_heads, n_seqs, scale, scratch.part_o.data_ptr(),
        scratch.part_ml.data_ptr(), scratch.part_n.data_ptr(), _at(sinks), err.data_ptr(), _stream())
    kernels.launches += 1   # (the parts, and their joining)
    _check(code, "attention_shared")


# ---------------------------------------------------------------------------------------------------------------- drafts
VERIFY_CHUNK = 8192        # logits of a block, and tokens of one that draws at the least (VF_CHUNK, VR_CHUNK of the kernels)
VERIFY_RACE_CHUNK = 2048


class VerifyScratch:
    """Workspaces of `verify_drafts`: what its kernels leave for one another, and ticket counters (kept zero between calls by the kernel
    itself). One instance serves calls that run one after another on one stream; what is captured into a graph has one of its own."""

    def __init__(self):
        self.held = self.counters = None   # one buffer of 8-byte words for all but the counters

    def ensure(self, row_chunks: int, entry_chunks: int, entries: int, device) -> tuple:
        """The addresses of sums, tops and best."""
        starts = (0, row_chunks, 2 * row_chunks)   # (sums of 8 bytes, tops of 8; what blocks leave, of 16, begins on 16)
        need = starts[2] + 2 * entry_chunks
        if self.held is None or self.held.numel() < need or self.held.device != device:
            self.held = torch.empty(need, dtype=torch.float64, device=device)
        if self.counters is None or self.counters.numel() < entries or self.counters.device != device:
            self.counters = torch.zeros(entries, dtype=torch.int32, device=device)
        base = self.held.data_ptr()
        return base, base + 8 * starts[1], base + 8 * starts[2]


class _StreamScratches(threading.local):
    """Of callers that bring none: one per thread and stream, since calls on two streams run at once, and two threads may launch in between each other."""

    MOST = 64   # (what goes was allocated on its own stream, behind whose work its memory is used again)

    def __init__(self):
        self.held: dict = {}

    def get(self, device: int, stream: int) -> VerifyScratch:
        scratch = self.held.get((device, stream))
        if scratch is None:
            while len(self.held) >= self.MOST:
                self.held.pop(next(iter(self.held)))
            scratch = self.held[device, stream] = VerifyScratch()
        return scratch


_verify_scratches = _StreamScratches()


def _callers_scratch() -> VerifyScratch:
    if torch._C._cuda_isCurrentStreamCapturing():
        raise KernelError("verify_drafts: a call that is captured into a graph wants a scratch of its own, which lives as long as the graph")
    return _verify_scratches.get(torch._C._cuda_getDevice(), _stream())


def verify_drafts(target: torch.Tensor, draft: Optional[torch.Tensor], drafted: torch.Tensor, first: torch.Tensor, uniforms: torch.Tensor,
                  temperature: float, seed: int, seq_ids: torch.Tensor, steps: torch.Tensor, accepted: torch.Tensor, tokens: torch.Tensor,
                  scratch: Optional[VerifyScratch] = None, redraw_seed: Optional[int] = None) -> None:
    """Which drafted tokens a model keeps, and the token that follows them. Entry s has the rows first[s] .. first[s + 1] - 1 of
    `target` (float32 logits of the model that decides): one behind each of its drafted tokens' contexts and one behind all of them, so
    one row more than it has drafts (none at all for a padding entry). Its drafts, the rows of `draft` (float32 logits of the model that
    drafted, or None: drafts that were not drawn at random, such as those looked up in the prompt) and `uniforms` (float32 in [0, 1))
    lie one after another, without the further rows.

    With p and q the softmax of both at `temperature`, draft d is kept while  u q(d) < p(d)  (q(d) = 1 without draft logits). The token
    behind the last kept one is drawn from max(0, p - q), or p without d, if a draft was refused, and from p behind the last:
    the token with the largest r / E, E = -ln of the sampler's own random number for (seed, seq_ids[s], steps[s] + kept, token), where
    steps[s] counts the tokens that the sequence has generated. So kept and drawn tokens together are distributed as the model's own
    draws, if the uniforms, each draft and the numbers of the draw are independent. Drafts that `sample` drew for the same sequences and steps
    are independent of them under another seed only: `redraw_seed` is the seed of draws behind a refused draft with draft logits (None:
    `seed`, for drafts that were drawn with other numbers; `Sampler.verify` sets it). temperature <= 0: a draft is kept while it is the row's argmax (the lowest
    id of equals), and the next token is the argmax.

    accepted int32 [n]: drafts kept; tokens int32 [n, most + 1]: kept drafts, the next token, then -1. An entry of no rows gets 0 and
    -1; one whose rows lie outside `target`, or with more drafts than `tokens` has room for, -1 and -1. A drafted id outside the
    vocabulary is refused. Logits are finite or -infinity. `scratch`: whoever captures the call into a CUDA graph passes one of
    its own, which then lives as long as the graph; None is one that the thread's calls on the current stream share."""
    if target.is_cuda:
        scratch = scratch or _callers_scratch()
        code = _native("verify_drafts", "verify_drafts")(target, draft, drafted, first, uniforms, seq_ids, steps, accepted, tokens, scratch.held, scratch.counters,
                                                         temperature, int(seed), int(seed) if redraw_seed is None else int(redraw_seed), VERIFY_CHUNK, VERIFY_RACE_CHUNK)
        if code is not None:
            kernels.launches += 1
            return _check(code, "verify_drafts")
    f32, i32 = torch.float32, torch.int32
    for name, t, dtype in (("target logits", target, f32), ("drafted", drafted, i32), ("first", first, i32), ("uniforms", uniforms, f32), ("accepted", accepted, i32),
                           ("tokens", tokens, i32)):
        if t.dtype is not dtype or not (t is target or t.is_contiguous()):
            _dev(name, t, dtype, contiguous=t is not target)
    if target.dim() != 2 or target.stride(1) != 1 or target.shape[1] <= 0:
        raise KernelError("verify_drafts: logits must be 2-d with unit inner stride")
    rows, vocab = target.shape
    n, total = accepted.numel(), drafted.numel()
    if first.numel() != n + 1 or tokens.dim() != 2 or tokens.shape[0] != n or tokens.shape[1] < 1:
        raise KernelError("verify_drafts: wants first [n + 1], accepted [n] and tokens [n, most drafts + 1]")
    if n == 0:
        return
    if total < rows - n:
        raise KernelError(f"verify_drafts: {rows} rows of {n} entries go with {rows - n} drafted tokens or more, not {total}")
    if max(n, rows + total) > 65535:
        raise KernelError(f"verify_drafts: {n} entries with {rows} rows and {total} drafts are more than a launch takes (65,535)")
    used, sampling = None, temperature > 0
    if sampling:
        if uniforms.numel() != total:
            raise KernelError("verify_drafts: uniforms must have one element per drafted token")
        if seq_ids is None or steps is None:
            raise KernelError("verify_drafts: sampling needs seq_ids and steps")
        if seq_ids.dtype is not torch.int64 or steps.dtype is not i32 or not seq_ids.is_contiguous() or not steps.is_contiguous():
            _dev("seq_ids", seq_ids, torch.int64)
            _dev("steps", steps, i32)
        if seq_ids.numel() != n or steps.numel() != n:
            raise KernelError("verify_drafts: seq_ids and steps must have one element per entry")
        _here("verify_drafts", target, seq_ids, steps)
        if draft is not None:
            _dev("draft logits", draft, f32, contiguous=False)
            if draft.dim() != 2 or draft.shape != (total, vocab) or (total > 0 and draft.stride(1) != 1):
                raise KernelError("verify_drafts: draft logits must have a row of the same vocabulary per drafted token")
            used = draft if total > 0 else None
    _here("verify_drafts", target, used, drafted, first, uniforms, accepted, tokens)
    all_rows = rows + (total if used is not None else 0)
    places = scratch.ensure(all_rows * -(-vocab // VERIFY_CHUNK), n * -(-vocab // VERIFY_RACE_CHUNK), n, target.device)
    code = _function("verify_drafts", "qf_verify_drafts", _P, _I, _I, _LL, _P, _LL, _P, _I, _P, _I, _P, _F, _ULL, _ULL, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P)(
        target.data_ptr(), rows, vocab, target.stride(0), _at(used), used.stride(0) if used is not None else 0, drafted.data_ptr(), total,
        first.data_ptr(), n, uniforms.data_ptr(), max(float(temperature), 0.0), int(seed) & 0xFFFFFFFFFFFFFFFF,
        int(seed if redraw_seed is None else redraw_seed) & 0xFFFFFFFFFFFFFFFF, seq_ids.data_ptr() if sampling else None,
        steps.data_ptr() if sampling else None, accepted.data_ptr(), tokens.data_ptr(), tokens.shape[1] - 1, *places, scratch.counters.data_ptr(), _stream())
    kernels.launches += all_rows > 0   # (the rows' statistics, and the decision with the draw)
    _check(code, "verify_drafts")
