"""Python entries of the kernels for several continuations of one prompt: copies of cache pages, attention of sequences whose
caches begin with the same pages, verification of drafted tokens. The same manner as `kernels.py`: checks on the host, raw device
pointers, the current stream, error codes."""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import numpy as np
import torch

from ..csrc import library
from . import kernels
from .kernels import _F, _I, _LL, _P, _ULL, KernelError, _check, _dev, _ptr, _stream


PAGE_TOKENS = 64   # positions of a cache page (QF_PAGE of the kernels, and what the cache hands out)


def _here(what: str, *tensors) -> None:
    """The tensors lie on the current device, whose current stream the kernels run on."""
    current = torch._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.device.index != current:
            raise KernelError(f"{what}: a tensor is on {t.device}, the current device is cuda:{current}")


def page_moves(moves, n_pages: int, n_rows: int) -> np.ndarray:
    """`moves` as int32 [n, 3] (from, to, rows), checked: pages 0 .. n_pages - 1, rows 0 .. n_rows (whole pages where a move names
    none), no page a target twice, none both a source and a target."""
    array = np.asarray(moves, dtype=np.int64)
    if array.size == 0:
        return np.zeros((0, 3), dtype=np.int32)
    if array.ndim != 2 or array.shape[1] not in (2, 3):
        raise KernelError("copy_pages: moves are (from, to) or (from, to, rows)")
    if array.shape[1] == 2:
        array = np.concatenate((array, np.full((len(array), 1), n_rows, dtype=np.int64)), axis=1)
    if array[:, :2].min() < 0 or array[:, :2].max() >= n_pages:
        raise KernelError(f"copy_pages: a move names a page outside 0 .. {n_pages - 1}")
    if array[:, 2].min() < 0 or array[:, 2].max() > n_rows:
        raise KernelError(f"copy_pages: a move names rows outside 0 .. {n_rows}")
    seen = np.zeros(n_pages, dtype=np.uint8)
    seen[array[:, 1]] = 1
    if int(seen.sum()) != len(array):
        raise KernelError("copy_pages: a page is the target of two moves")
    if seen[array[:, 0]].any():
        raise KernelError("copy_pages: a page is the source of one move and the target of another")
    return np.ascontiguousarray(array, dtype=np.int32)


def copy_pages(storage: torch.Tensor, moves) -> None:
    """Copies rows of pages inside `storage`, for every schedule entry at once. storage: [entries, pages, ..., rows, width] of any dtype
    (a page dense, entries and pages at any distance; a storage of two or three dimensions has pages of one row). moves: (from, to, rows)
    or (from, to) on the host: the first `rows` rows of page `from`, in each of its planes and heads, become those of page `to`; the
    others stay as they are. No page may be the target of two moves, or both a source and a target."""
    _dev("storage", storage, contiguous=False)
    if storage.dim() < 2:
        raise KernelError("copy_pages: storage has entries and pages")
    entries, pages = storage.shape[:2]
    inner = tuple(storage.shape[2:])
    n_rows, width = (inner[-2], inner[-1]) if len(inner) >= 2 else (1, inner[0] if inner else 1)
    segments = 1
    for d in inner[:-2]:
        segments *= d
    checked = page_moves(moves, pages, n_rows)
    page = segments * n_rows * width
    if page == 0 or entries == 0 or len(checked) == 0:
        return
    want = 1
    for size, stride in zip(reversed(inner), reversed(storage.stride()[2:])):
        if size != 1 and stride != want:
            raise KernelError("copy_pages: a page of the storage is not contiguous")
        want *= size
    e_stride, p_stride = storage.stride(0), storage.stride(1)
    if (pages > 1 and p_stride < page) or (entries > 1 and e_stride < page) or (
            entries > 1 and pages > 1 and e_stride < (pages - 1) * p_stride + page and p_stride < (entries - 1) * e_stride + page):
        raise KernelError("copy_pages: pages of the storage overlap")
    _here("copy_pages", storage)
    item = storage.element_size()
    sizes = (storage.data_ptr(), width * item, e_stride * item if entries > 1 else 0, p_stride * item if pages > 1 else 0)
    unit = next(u for u in (16, 4, 2, 1) if all(s % u == 0 for s in sizes))
    launched = _I(0)
    code = library("page_copy").qf_copy_pages(
        _ptr(storage), _I(entries), _LL(sizes[2]), _LL(sizes[3]), _I(segments), _LL(n_rows * width * item), _LL(width * item), _I(unit),
        _P(checked.ctypes.data), _I(len(checked)), ctypes.byref(launched), _stream())
    kernels.launches += launched.value - 1
    _check(code, "copy_pages")


SHARED_MAX_HEAD_DIM = 256
SHARED_MAX_SEQS = 2048


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
        self.least_pages = 0 if bound_pages else min(entry_pages)
        sizes = (self.n_seqs, self.n_seqs, len(members), len(begin), len(pages))
        packed = torch.tensor(entry_pages + entry_group + members + begin + pages, dtype=torch.int32).to(device)
        self.entry_pages, self.entry_group, self.members, self.begin, self.pages = packed.split(sizes)

    def __len__(self) -> int:
        return len(self.groups)

    def shape(self) -> tuple:
        """What the launches go by: the batch, the groups' members, the bound on their pages."""
        return (self.n_seqs, tuple(len(entries) for entries, _ in self.groups), self.bound_pages)

    def load(self, other: "SharedPrefix") -> None:
        """Take over what `other`, of the same members per group and within the bound, says is shared; the addresses stay."""
        if other.shape()[:2] != self.shape()[:2] or other.most_pages > self.bound_pages:
            raise KernelError("SharedPrefix: what is loaded has other groups, or more pages than the bound")
        for name in ("entry_pages", "entry_group", "members", "begin", "pages"):
            getattr(self, name).copy_(getattr(other, name))
        self.groups, self.most_pages = other.groups, other.most_pages


class SharedScratch:
    """Workspaces of `attention_shared`: the parts' sums with their maxima, and the plans. One instance serves calls that run one after
    another on one stream; what is captured into a graph has one of its own."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.part_o = self.part_ml = None
        self.plans: dict = {}

    def ensure(self, parts: int, head_dim: int) -> None:
        if self.part_o is None or self.part_o.numel() < parts * head_dim:
            self.part_o = torch.empty(parts * head_dim, dtype=torch.float32, device=self.device)
        if self.part_ml is None or self.part_ml.numel() < parts * 2:
            self.part_ml = torch.empty(parts * 2, dtype=torch.float32, device=self.device)


class SharedPlan:
    """What `attention_shared_plan` made: the tensor (which block and warp takes which run) and the sizes that the attention's launch goes by."""
    __slots__ = ("tensor", "key", "records", "most_parts")

    def __init__(self, tensor, key, records, most_parts):
        self.tensor, self.key, self.records, self.most_parts = tensor, key, records, most_parts


def _shared_sizes(dtype, head_dim: int, kv_heads: int, n_heads: int, share: SharedPrefix, own_pages: int) -> tuple:
    """((block records, warp records, tile records) of the plan, most shared parts, most own parts of a row): bounds of what the plan kernel
    can come to, whatever the lengths. It gives a warp at least `pages x tiles x kv heads / warps` pages, so block records cover, up to
    twice, no more than the warps there are; tile records fill the SMs once, or are the pairs of tiles uncut."""
    sizes = (_I * 7)()
    code = library("attention_shared").qf_attention_shared_shape(_I(int(dtype == torch.bfloat16)), _I(head_dim), sizes)
    if code:
        raise KernelError(f"attention_shared: CUDA error {code} when asked for its sizes")
    row_tile, warps, team, most, tile_rows, tile_pages, sms = sizes
    group_heads = n_heads // kv_heads

    def parts(pages: int, tiles: int) -> int:
        return max(team, min(most, -(-pages // team), warps // (team * kv_heads * tiles) + 1))
    own_tiles = -(-group_heads // row_tile)
    tiles = [-(-len(entries) * group_heads // row_tile) for entries, _ in share.groups]
    most_shared = max((parts(share.bound_pages, t) for t in tiles), default=0)
    pairs = [-(-len(entries) * group_heads // 256) for entries, _ in share.groups if len(entries) * group_heads >= tile_rows]
    if not tile_rows or share.bound_pages < tile_pages:
        pairs = []
    for n in pairs:
        most_shared = max(most_shared, min(most, -(-share.bound_pages // 4), sms // (kv_heads * n) + 1))
    records = (2 * warps // (team * kv_heads) + 2, warps // kv_heads + 1 + sum(tiles) + share.n_seqs * own_tiles,
               max(sms // kv_heads, sum(pairs)) if pairs else 0)
    return records, most_shared, parts(own_pages, own_tiles)


def attention_shared_plan(cu_q: torch.Tensor, tok_pos: torch.Tensor, slots: torch.Tensor, kv_heads: int, head_dim: int, n_heads: int,
                          n_seqs: int, share: SharedPrefix, scratch: SharedScratch, dtype: torch.dtype, max_kv_len: int) -> SharedPlan:
    """The plan of one step for `attention_shared` of this shape, worked out on the device from the batch's lengths; it serves every
    layer of the step with this shape. `max_kv_len`: an upper bound of any sequence's length after the step. The tensor belongs to
    `scratch` and is overwritten by the next plan of the same shape."""
    for name, t in (("cu_q", cu_q), ("tok_pos", tok_pos), ("slots", slots)):
        _dev(name, t, torch.int32)
    if dtype not in (torch.bfloat16, torch.float32):
        raise KernelError(f"attention_shared: dtype {dtype} is not supported (bfloat16 or float32)")
    if not 0 < head_dim <= SHARED_MAX_HEAD_DIM:
        raise KernelError(f"attention_shared: head_dim {head_dim} > {SHARED_MAX_HEAD_DIM} is not supported")
    if kv_heads <= 0 or n_heads <= 0 or n_heads % kv_heads:
        raise KernelError(f"attention_shared: {n_heads} heads do not divide into {kv_heads} groups")
    if not 0 < n_seqs <= SHARED_MAX_SEQS:
        raise KernelError(f"attention_shared: a batch of {n_seqs} sequences is not supported (1 to {SHARED_MAX_SEQS})")
    if share.n_seqs != n_seqs or slots.numel() != n_seqs or cu_q.numel() != n_seqs + 1 or tok_pos.numel() != n_seqs:
        raise KernelError("attention_shared: wants exactly one token per sequence, and a SharedPrefix of this batch")
    _here("attention_shared", cu_q, tok_pos, slots, share.entry_pages)
    own_pages = max(1, -(-int(max_kv_len) // PAGE_TOKENS) - share.least_pages)
    records, most_shared, most_own = _shared_sizes(dtype, head_dim, kv_heads, n_heads, share, own_pages)
    key = (n_seqs, kv_heads, n_heads, head_dim, dtype)
    ints = 4 + -(-n_seqs // 4) * 4 + sum(records) * 8
    held = scratch.plans.get(key)
    if held is None or held.numel() < ints:
        held = scratch.plans[key] = torch.empty(ints, dtype=torch.int32, device=cu_q.device)
    _check(library("attention_shared").qf_attention_shared_plan(
        _ptr(tok_pos), _ptr(slots), _I(n_seqs), _ptr(share.entry_pages), _ptr(share.entry_group), _ptr(share.begin), _ptr(share.pages), _I(len(share)),
        _I(kv_heads), _I(n_heads), _I(int(dtype == torch.bfloat16)), _I(head_dim), _I(most_shared), _I(most_own),
        _ptr(held), *map(_I, records), _stream()), "attention_shared_plan")
    return SharedPlan(held, key, records, most_shared + most_own)


def attention_shared(q: torch.Tensor, out: torch.Tensor, cu_q: torch.Tensor, tok_pos: torch.Tensor, slots: torch.Tensor, site, n_heads: int,
                     n_seqs: int, scale: float, share: SharedPrefix, scratch: SharedScratch, err: torch.Tensor,
                     max_kv_len: Optional[int] = None, plan: Optional[SharedPlan] = None, sinks: Optional[torch.Tensor] = None) -> None:
    """Attention of ONE new token per sequence over its cache, where sequences share their first pages (`share`): what they share is read
    once for all of them. The result is that of `attention_decode`: query head i reads kv head i // (n_heads / kv_heads), key j is visible
    iff j <= the token's position. bfloat16 or float32, head sizes up to 256 (bfloat16 of 32, 64, 96 and 128 on tensor cores). A padding
    entry (slot -1) gets zeros. `max_kv_len`: an upper bound of any sequence's length after the step (None: as long as the page table
    has room for). `plan` (`attention_shared_plan` with the same shape, made in this step) is made here when absent. `sinks` (float32
    [n_heads]): a logit per head that joins the softmax's denominator once, with no key and no value."""
    _dev("q", q)
    _dev("out", out, q.dtype)
    _dev("cache", site.storage, q.dtype, contiguous=False)
    _dev("page table", site.table, torch.int32, contiguous=False)
    _dev("err", err, torch.int32)
    d, page = site.head_dim, PAGE_TOKENS
    if q.shape != (n_seqs, n_heads * d) or out.shape != q.shape:
        raise KernelError("attention_shared: wants exactly one token per sequence, q and out [n_seqs, n_heads * head_dim]")
    if site.storage.dim() != 5 or tuple(site.storage.shape[1:]) != (2, site.kv_heads, page, d) or not site.storage[:1].is_contiguous() \
            or site.page_elems < 2 * site.kv_heads * page * d:
        raise KernelError(f"attention_shared: the cache is [pages, 2, kv_heads, {page}, head_dim], a page dense")
    if site.table.dim() != 2 or site.table.stride(1) != 1:
        raise KernelError("attention_shared: the page table is [slots, pages] with unit inner stride")
    if share.most_pages > site.table.shape[1]:
        raise KernelError(f"attention_shared: a group shares {share.most_pages} pages, the page table has room for {site.table.shape[1]}")
    fast = q.dtype == torch.bfloat16 and d in kernels.FAST_ATTENTION_HEAD_DIMS
    if fast and (q.data_ptr() % 16 or site.storage.data_ptr() % 16 or site.page_elems % d):
        raise KernelError("attention_shared: q and the cache begin on 16 bytes, and a page holds whole rows")
    if sinks is not None:
        _dev("sinks", sinks, torch.float32)
        if sinks.numel() != n_heads:
            raise KernelError("attention_shared: sinks must hold one float32 per query head")
    _here("attention_shared", q, out, cu_q, tok_pos, slots, site.storage, site.table, share.entry_pages, err, sinks)
    if plan is None:
        longest = site.table.shape[1] * page if max_kv_len is None else int(max_kv_len)
        plan = attention_shared_plan(cu_q, tok_pos, slots, site.kv_heads, d, n_heads, n_seqs, share, scratch, q.dtype, longest)
    elif plan.key != (n_seqs, site.kv_heads, n_heads, d, q.dtype):
        raise KernelError("attention_shared: the plan was made for another shape")
    scratch.ensure(n_seqs * n_heads * plan.most_parts, d)
    code = library("attention_shared").qf_attention_shared(
        _I(int(q.dtype == torch.bfloat16)), _ptr(q), _ptr(out), _ptr(tok_pos), _ptr(slots), _ptr(share.members), _ptr(share.begin),
        _ptr(plan.tensor), *map(_I, plan.records), _ptr(site.storage), _ptr(site.table), _LL(site.page_elems),
        _I(site.table_stride), _I(site.kv_heads), _I(d), _I(n_heads), _I(n_seqs), _F(scale), _I(plan.most_parts), _ptr(scratch.part_o),
        _ptr(scratch.part_ml), _ptr(sinks), _ptr(err), _stream())
    kernels.launches += 2 if plan.records[2] else 1   # (the tiles, the parts, and their joining)
    _check(code, "attention_shared")


class VerifyScratch:
    """Workspaces of `verify_drafts`: what the blocks of a row and of an entry leave for one another, and ticket counters (kept zero
    between calls by the kernel itself). One instance serves calls that run one after another on one stream; what is captured into a
    graph has one of its own."""

    def __init__(self):
        self.sums = self.tops = self.best = self.counters = None

    def ensure(self, row_chunks: int, entry_chunks: int, entries: int, device) -> None:
        def room(held, count, width, dtype):
            if held is None or held.numel() < count * width or held.device != device:
                return torch.zeros(count * width, dtype=dtype, device=device)
            return held
        self.sums = room(self.sums, row_chunks, 1, torch.float64)
        self.tops = room(self.tops, row_chunks, 2, torch.int32)     # (float32 maximum, id)
        self.best = room(self.best, entry_chunks, 2, torch.float64)  # (score, id)
        self.counters = room(self.counters, entries, 1, torch.int32)


_verify_scratch = VerifyScratch()


def verify_drafts(target: torch.Tensor, draft: Optional[torch.Tensor], drafted: torch.Tensor, first: torch.Tensor, uniforms: torch.Tensor,
                  temperature: float, seed: int, seq_ids: torch.Tensor, steps: torch.Tensor, accepted: torch.Tensor, tokens: torch.Tensor,
                  scratch: Optional[VerifyScratch] = None) -> None:
    """Which drafted tokens a model keeps, and the token that follows them. Entry s has the rows first[s] .. first[s + 1] - 1 of
    `target` (float32 logits of the model that decides): one behind each of its drafted tokens' contexts and one behind all of them, so
    one row more than it has drafts (none at all for a padding entry). Its drafts, the rows of `draft` (float32 logits of the model that
    drafted, or None: drafts that were not drawn at random, such as those looked up in the prompt) and `uniforms` (float32 in [0, 1))
    lie one after another, without the further rows.

    With p and q the softmax of both at `temperature`, draft d is kept while  u q(d) < p(d)  (q(d) = 1 without draft logits). The token
    behind the last kept one is drawn from max(0, p - q), or p without d, if a draft was refused, and from p behind the last:
    the token with the largest r / E, E = -ln of the sampler's own random number for (seed, seq_ids[s], steps[s] + kept, token), where
    steps[s] counts the tokens that the sequence has generated. So kept and drawn tokens together are distributed as the model's own
    draws. temperature <= 0: a draft is kept while it is the row's argmax (the lowest id of equals), and the next token is the argmax.

    accepted int32 [n]: drafts kept; tokens int32 [n, most + 1]: kept drafts, the next token, then -1. An entry of no rows gets 0 and
    -1; one whose rows lie outside `target`, or with more drafts than `tokens` has room for, -1 and -1. A drafted id outside the
    vocabulary is refused. Logits are finite or -infinity. `scratch`: as in `sample`."""
    _dev("target logits", target, torch.float32, contiguous=False)
    if target.dim() != 2 or target.stride(1) != 1 or target.shape[1] <= 0:
        raise KernelError("verify_drafts: logits must be 2-d with unit inner stride")
    rows, vocab = target.shape
    n = accepted.numel()
    for name, t, dtype in (("drafted", drafted, torch.int32), ("first", first, torch.int32), ("uniforms", uniforms, torch.float32),
                           ("accepted", accepted, torch.int32), ("tokens", tokens, torch.int32)):
        _dev(name, t, dtype)
    if first.numel() != n + 1 or tokens.dim() != 2 or tokens.shape[0] != n or tokens.shape[1] < 1:
        raise KernelError("verify_drafts: wants first [n + 1], accepted [n] and tokens [n, most drafts + 1]")
    if n == 0:
        return
    total = drafted.numel()
    if total < rows - n:
        raise KernelError(f"verify_drafts: {rows} rows of {n} entries go with {rows - n} drafted tokens or more, not {total}")
    if max(n, rows + total) > 65535:
        raise KernelError(f"verify_drafts: {n} entries with {rows} rows and {total} drafts are more than a launch takes (65,535)")
    sampling = temperature > 0
    if sampling:
        if uniforms.numel() != total:
            raise KernelError("verify_drafts: uniforms must have one element per drafted token")
        _dev("seq_ids", seq_ids, torch.int64)
        _dev("steps", steps, torch.int32)
        if seq_ids.numel() != n or steps.numel() != n:
            raise KernelError("verify_drafts: seq_ids and steps must have one element per entry")
        if draft is not None:
            _dev("draft logits", draft, torch.float32, contiguous=False)
            if draft.dim() != 2 or draft.shape != (total, vocab) or (total > 0 and draft.stride(1) != 1):
                raise KernelError("verify_drafts: draft logits must have a row of the same vocabulary per drafted token")
    used = draft if sampling and total > 0 else None
    _here("verify_drafts", target, used, drafted, first, uniforms, accepted, tokens, *((seq_ids, steps) if sampling else ()))
    lib = library("verify_drafts")
    sizes = (_I * 2)()
    lib.qf_verify_chunks(_I(vocab), sizes)
    all_rows = rows + (total if used is not None else 0)
    scratch = scratch or _verify_scratch
    scratch.ensure(max(all_rows, 1) * sizes[0], n * sizes[1], n, target.device)
    code = lib.qf_verify_drafts(
        _ptr(target), _I(rows), _I(vocab), _LL(target.stride(0)), _ptr(used), _LL(used.stride(0) if used is not None else 0), _ptr(drafted), _I(total),
        _ptr(first), _I(n), _ptr(uniforms), _F(max(float(temperature), 0.0)), _ULL(int(seed) & 0xFFFFFFFFFFFFFFFF), _ptr(seq_ids if sampling else None),
        _ptr(steps if sampling else None), _ptr(accepted), _ptr(tokens), _I(tokens.shape[1] - 1), _ptr(scratch.sums), _ptr(scratch.tops),
        _ptr(scratch.best), _ptr(scratch.counters), _stream())
    kernels.launches += 1   # (the rows' statistics, and the choice)
    _check(code, "verify_drafts")
