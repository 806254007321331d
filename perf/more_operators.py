"""Operators of a sequence cache in 8 bits, in plain form and as this library's calls.

  write   a step's new keys and values, rotated and with their biases, appended to the cache as e4m3 codes
  read    the rows that a batch's sequences hold, back as bfloat16 or float32 pages
  attend  attention of single tokens and of short spans (drafted tokens) over that cache

The cache holds a code per element and a power of two per page of 64 positions, plane (keys, values) and kv head; an element stands
for code * 2^e. A step that adds rows to a page takes e = the least exponent with amax <= 448 * 2^e over its rows (finite elements; between
-112 and 119), and no less than the page's own if the page had rows before: their codes are then rounded again to the larger step.
What is finite and too large, or infinite, becomes +-448; NaN stays NaN.

`run` computes the plain form (elementary torch operations) where `own` is false and makes the library's calls where it is true.
Sizes are those of the Qwen2.5 presets (heads, head size, longest sequence) and of the test configurations.
"""
import math
import zlib

import numpy as np
import torch

own = False

PAGE = 64                       # positions of a cache page
LOW, HIGH = -112, 119           # exponents of a page's scale
TOP = 448.0                     # largest e4m3 value
# (query heads, kv heads, head size, rope theta): the 0.5B, 3B and 7B presets, and shapes of the tests
HEADS = {"0.5b": (14, 2, 64, 1e6), "3b": (16, 2, 128, 1e6), "7b": (28, 4, 128, 1e6), "small": (7, 1, 64, 1e6), "wide": (6, 3, 96, 1e4),
         "tiny": (4, 2, 16, 1e4), "pairs": (4, 2, 128, 1e6), "single": (5, 5, 80, 1e4)}


# ------------------------------------------------------------------------------------------------ cases
def _case(name, kind, model, seqs, longest, tokens, dtype="bfloat16", window=0, even=False):
    """seqs sequences whose lengths after the step are up to `longest` (ragged, or `even`: all of them nearly that), with up to `tokens` new
    ones each (as many as fit)."""
    return {"name": name, "kind": kind, "model": model, "seqs": seqs, "longest": longest, "tokens": tokens, "dtype": dtype, "window": window, "even": even}


def listed():
    return [
        # a chat's next token: the smallest write, all latency
        _case("append-1", "write", "0.5b", 1, 1000, 1),
        # a serving batch's next tokens
        _case("append-96", "write", "7b", 96, 700, 1),
        # ragged prompts that start together, in the float32 path
        _case("prompts-12-float32", "write", "3b", 12, 900, 900, "float32"),
        # one long prompt
        _case("prompt-8192", "write", "7b", 1, 8192, 8192, even=True),
        # what a prompt's continuation reads back of an earlier turn
        _case("read-700", "read", "0.5b", 1, 700, 50),
        # four long documents continued by a question each
        _case("read-documents", "read", "7b", 4, 30000, 90),
        # a chat's next token
        _case("chat-1", "attend", "0.5b", 1, 900, 1),
        # a small batch of 4,000 tokens each
        _case("batch-8", "attend", "0.5b", 8, 4096, 1, even=True),
        # a full serving batch, ragged
        _case("serving-64", "attend", "7b", 64, 8000, 1),
        # one document that fills the context
        _case("document-1", "attend", "3b", 1, 32000, 1, even=True),
        # drafted tokens verified: spans of up to five
        _case("drafts-12", "attend", "7b", 12, 3000, 5),
        # the float32 path, ragged
        _case("float32-20", "attend", "3b", 20, 3500, 1, "float32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "write", "read", "attend", "attend", "attend"])
    model = rng.choice(list(HEADS))
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    width = HEADS[model][1] * HEADS[model][2]
    seqs = _log_int(rng, 1, 96)
    if kind == "write":
        tokens = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4000)
        seqs = max(1, min(seqs, 6000 // tokens))
        longest = max(tokens, min(_log_int(rng, 1, 8000), 60000 * 512 // (seqs * width)))
        return _case(None, kind, model, seqs, longest, tokens, dtype, even=rng.random() < 0.3)
    most = (100_000 if kind == "read" else 250_000) * 512 // width // (2 if dtype == "float32" else 1)
    longest = max(1, min(_log_int(rng, 1, 32000), most // seqs))
    if kind == "read":
        return _case(None, kind, model, seqs, longest, _log_int(rng, 1, 100), dtype, rng.choice([0, 0, 0, 37, 500]))
    tokens = rng.choice([1, 1, 1, 2, 4, 5, 8])   # (no more products than the largest listed case has)
    return _case(None, kind, model, seqs, max(1, longest // tokens), tokens, dtype, rng.choice([0, 0, 0, 0, 37, 1000]), rng.random() < 0.3)


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) + 1)


def _layout(case):
    """(new tokens, length after the step) of every sequence: the case's own, so that every seed has the same work."""
    rng = np.random.default_rng(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    low = case["longest"] - case["longest"] // 50 if case["even"] else 1
    lengths = rng.integers(low, case["longest"] + 1, case["seqs"])
    if case["seqs"] == 1:
        lengths[:] = case["longest"]
    new = np.minimum(lengths, case["tokens"] if case["tokens"] == 1 or case["even"] else rng.integers(1, case["tokens"] + 1, case["seqs"]))
    return new.tolist(), lengths.tolist()


def _codes(x, e):
    """x / 2^e as e4m3 values, exponents broadcast."""
    return (x * torch.exp2(-e)).clamp(-TOP, TOP).to(torch.float8_e4m3fn)


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, within the range; amax = m * 2^k with m in [1/2, 1), and 448 = 7/8 * 2^9."""
    m, k = torch.frexp(amax)
    e = torch.where(m <= 0.875, k - 9, k - 8)
    return torch.where(amax > 0, e, LOW).clamp(LOW, HIGH)


def prepare(case, seed):
    heads, kv_heads, dim, theta = HEADS[case["model"]]
    dtype = getattr(torch, case["dtype"])
    new, lengths = _layout(case)
    n, total, window = len(new), sum(new), case["window"]
    counts = [-(-x // PAGE) for x in lengths]
    kept = [max(0, x - t - window + 1) // PAGE if window > 0 else 0 for x, t in zip(lengths, new)]   # pages before it were given back
    ids = np.random.default_rng(int(seed) + 29).permutation(sum(counts) - sum(kept)).astype(np.int32)   # pages lie anywhere in the storage
    slots = np.random.default_rng(int(seed) + 31).permutation(n + 2)[:n].astype(np.int32)
    table = np.full((n + 2, max(counts)), -1, dtype=np.int32)
    at = 0
    for s in range(n):
        held = counts[s] - kept[s]
        table[slots[s], kept[s]:counts[s]] = ids[at:at + held]
        at += held
    cu_q = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tok_seq = np.repeat(np.arange(n, dtype=np.int32), new)
    tok_pos = np.concatenate([np.arange(x - t, x, dtype=np.int32) for x, t in zip(lengths, new)])
    g = _generator(seed)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=g)   # noqa: E731
    # some channels of a key head are several times as large as the others
    channel = torch.exp(0.7 * torch.randn((2, kv_heads, dim), device="cuda", generator=g))
    storage = torch.empty((len(ids), 2, kv_heads, PAGE, dim), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((len(ids), 2, kv_heads), device="cuda")
    for lo in range(0, len(ids), 1024):   # (in pieces: the values are four times the codes)
        x = rand(min(1024, len(ids) - lo), 2, kv_heads, PAGE, dim) * channel[:, :, None]
        e = _exponent(x.abs().amax((-1, -2))).float()
        storage[lo:lo + 1024] = _codes(x, e[..., None, None])
        scales[lo:lo + 1024] = torch.exp2(e)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()   # noqa: E731
    state = {"case": case, "storage": storage, "scales": scales, "table": to(table), "cu_q": to(cu_q), "tok_seq": to(tok_seq), "tok_pos": to(tok_pos),
             "slots": to(slots), "err": torch.zeros(1, dtype=torch.int32, device="cuda"), "n": n, "max_q": max(new), "max_kv": max(lengths),
             "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window, "lengths": lengths, "new": new}
    width = (heads + 2 * kv_heads) * dim
    if case["kind"] == "write":
        spread = torch.cat([torch.ones(heads * dim, device="cuda"), channel.reshape(-1)])
        state["qkv"] = (rand(total, width) * spread).to(dtype)
        state["bias"] = (0.3 * rand(width)).to(dtype)
        state["inv_freq"] = (1.0 / theta ** (torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)).float()
        state["q_out"] = torch.empty((total, heads * dim), dtype=dtype, device="cuda")
        state["touched"] = to(np.unique(table[slots[tok_seq], tok_pos // PAGE]).astype(np.int64))
    elif case["kind"] == "read":
        state["out"] = torch.zeros(storage.shape, dtype=dtype, device="cuda")
        owner, page = zip(*[(s, p) for s in range(n) for p in range(kept[s], counts[s])])
        owner, page = np.array(owner), np.array(page)
        state["pages"] = to(table[slots[owner], page].astype(np.int64))
        state["first"] = to((np.maximum(0, np.array(lengths) - np.array(new) - window + 1 if window > 0 else 0 * np.array(lengths))[owner] - page * PAGE))
        state["behind"] = to(np.array(lengths)[owner] - page * PAGE)
    else:
        state["q"] = (1.3 * rand(total, heads * dim)).to(dtype)
        state["out"] = torch.empty((total, heads * dim), dtype=dtype, device="cuda")
        state["scale"] = dim ** -0.5
        # entry, place in its span: where each token's row stands in a padded batch
        state["place"] = to(np.concatenate([np.arange(t) for t in new]))
    if own:
        from qwenforge_b200 import ops
        state["site"] = ops.E4m3SiteArgs(storage, scales, state["table"], kv_heads, dim)
        if case["kind"] == "attend":
            state["scratch"] = ops.E4m3Scratch(storage.device)
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_write(s):
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    storage, scales = s["storage"], s["scales"]
    x = (s["qkv"].float() + s["bias"].float()).view(-1, heads + 2 * kv_heads, dim)
    angle = s["tok_pos"].double()[:, None] * s["inv_freq"].double()
    c, sn = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[:, :heads + kv_heads, :dim // 2], x[:, :heads + kv_heads, dim // 2:]
    turned = torch.cat((a * c - b * sn, b * c + a * sn), -1)
    s["q_out"].copy_(turned[:, :heads].reshape(s["q_out"].shape))
    rows = torch.stack((turned[:, heads:], x[:, heads + kv_heads:]), 1)            # [T, 2, kv heads, dim]
    pos = s["tok_pos"].long()
    page, at = s["table"][s["slots"].long()[s["tok_seq"].long()], pos // PAGE].long(), pos % PAGE
    finite = torch.where(rows.isfinite(), rows.abs(), 0.0).amax(-1)
    amax = torch.zeros_like(scales).index_reduce_(0, page, finite, "amax")
    first = torch.full((len(scales),), PAGE, device=page.device).index_reduce_(0, page, at, "amin")
    t = s["touched"]
    first = first[t][:, None, None]
    before = torch.where(first > 0, torch.frexp(scales[t])[1] - 1, LOW)
    e = torch.maximum(_exponent(amax[t]), before).float()
    old = storage[t]
    again = _codes(old.float() * torch.exp2(before.float())[..., None, None], e[..., None, None])
    kept = torch.arange(PAGE, device=page.device)[:, None] < first[..., None, None]
    storage[t] = torch.where(kept, again.view(torch.uint8), old.view(torch.uint8)).view(torch.float8_e4m3fn)
    scales[t] = torch.exp2(e)
    storage.view(torch.uint8)[page, :, :, at] = _codes(rows, scales[page].log2()[..., None]).view(torch.uint8)
    return {"q": s["q_out"], "codes": storage, "scales": scales}


def _plain_read(s):
    row = torch.arange(PAGE, device="cuda")
    held = (row >= s["first"][:, None]) & (row < s["behind"][:, None])
    values = s["storage"][s["pages"]].float() * s["scales"][s["pages"]][..., None, None]
    s["out"][s["pages"]] = torch.where(held[:, None, None, :, None], values.to(s["out"].dtype), s["out"][s["pages"]])
    return s["out"]


def _plain_attend(s):
    heads, kv_heads, dim, n, most = s["heads"], s["kv_heads"], s["dim"], s["n"], s["max_q"]
    tables = s["table"][s["slots"].long()]                                          # [n, pages]
    pages = tables.clamp(min=0).long()
    values = lambda plane: (s["storage"][pages, plane].float() * s["scales"][pages, plane][..., None, None]).transpose(1, 2).flatten(2, 3)  # noqa: E731
    entry, place = s["tok_seq"].long(), s["place"]
    q = torch.zeros((n, most, heads, dim), device="cuda")
    q[entry, place] = s["q"].float().view(-1, heads, dim)
    at = torch.full((n, most), -1, device="cuda")
    at[entry, place] = s["tok_pos"].long()
    key = torch.arange(tables.shape[1] * PAGE, device="cuda")
    seen = key <= at[..., None]
    if s["window"] > 0:
        seen &= key > at[..., None] - s["window"]
    group = heads // kv_heads
    rows = q.view(n, most, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kv_heads, most * group, dim)
    scores = torch.matmul(rows, values(0).transpose(-1, -2)) * s["scale"]           # [n, kv heads, rows, keys]
    mask = seen[:, None, :, None].expand(-1, -1, -1, group, -1).flatten(2, 3)
    scores.masked_fill_(~mask, -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp(min=-3e38)                        # (a row of padding sees nothing)
    weights = scores.exp_()
    some = seen.any(1)[:, None, :, None]
    out = torch.matmul(weights, torch.where(some, values(1), 0.0)) / weights.sum(-1, keepdim=True)
    out = out.view(n, kv_heads, most, group, dim).permute(0, 2, 1, 3, 4).reshape(n, most, heads * dim)
    s["out"].copy_(out[entry, place])
    return s["out"]


# ------------------------------------------------------------------------------------------------ run
def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        from qwenforge_b200 import ops
        if kind == "write":
            ops.rope_cache_write_e4m3(s["qkv"], s["cu_q"], s["tok_seq"], s["tok_pos"], s["slots"], s["inv_freq"], s["dim"], s["heads"], s["q_out"],
                                      s["site"], s["max_q"], s["err"], bias=s["bias"])
            return {"q": s["q_out"], "codes": s["storage"], "scales": s["scales"]}
        if kind == "read":
            ops.cache_read_e4m3(s["out"], s["cu_q"], s["tok_pos"], s["slots"], s["site"], s["n"], s["max_kv"], s["err"], window=s["window"])
            return s["out"]
        ops.attention_e4m3(s["q"], s["out"], s["cu_q"], s["tok_pos"], s["slots"], s["site"], s["heads"], s["n"], s["max_q"], s["scale"], s["window"],
                           s["scratch"], s["err"], max_kv_len=s["max_kv"])
        return s["out"]
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[kind](s)


def work(case):
    heads, kv_heads, dim, _ = HEADS[case["model"]]
    new, lengths = _layout(case)
    item, total, row = 2 if case["dtype"] == "bfloat16" else 4, sum(new), 2 * kv_heads * dim
    seen = [min(x, t + case["window"] - 1) if case["window"] > 0 else x for x, t in zip(lengths, new)]
    if case["kind"] == "write":
        return {"bytes": total * ((2 * heads * dim + row) * item + row), "flops": total * (3 * (heads + kv_heads) * dim + 3 * row)}
    if case["kind"] == "read":
        return {"bytes": sum(seen) * row * (1 + item), "flops": sum(seen) * row}
    pairs = sum(min(p + 1, case["window"]) if case["window"] > 0 else p + 1 for x, t in zip(lengths, new) for p in range(x - t, x))
    return {"bytes": sum(seen) * row + 2 * total * heads * dim * item, "flops": 4 * pairs * heads * dim}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_rows(values):
    """values in float64 -> the page's exponent and its codes, one page's rows of one plane: [..., rows, dim]."""
    size = torch.where(values.isfinite(), values.abs(), 0.0).amax((-1, -2))
    e = torch.ceil(torch.log2(size.clamp(min=1e-300) / TOP)).clamp(LOW, HIGH)
    return torch.where(size > 0, e, float(LOW))


def _e4m3(x):
    """x in float64 rounded to e4m3: a step of 2^-3 within a binade, and of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def exact(case, seed):
    s = prepare(case, seed)
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    table, slots, new, lengths = s["table"].tolist(), s["slots"].tolist(), s["new"], s["lengths"]
    if case["kind"] == "read":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        for i, (t, x) in enumerate(zip(new, lengths)):
            lo = max(0, x - t - case["window"] + 1) if case["window"] > 0 else 0
            for p in range(lo // PAGE, -(-x // PAGE)):
                a, b, page = max(lo - p * PAGE, 0), min(x - p * PAGE, PAGE), table[slots[i]][p]
                out[page, :, :, a:b] = s["storage"][page, :, :, a:b].double() * s["scales"][page, :, :, None, None].double()
        return out
    if case["kind"] == "write":
        x = (s["qkv"].double() + s["bias"].double()).view(-1, heads + 2 * kv_heads, dim)
        half = dim // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["tok_pos"].double()[:, None] * s["inv_freq"].double())[:, None]
        z = torch.complex(x[:, :heads + kv_heads, :half], x[:, :heads + kv_heads, half:]) * turn
        turned = torch.cat((z.real, z.imag), -1)
        rows = torch.stack((turned[:, heads:], x[:, heads + kv_heads:]), 1)
        codes, scales, base = s["storage"].double(), s["scales"].double(), 0
        for i, (t, length) in enumerate(zip(new, lengths)):
            pos = length - t
            while pos < length:
                end = min(length, (pos // PAGE + 1) * PAGE)
                page, at = table[slots[i]][pos // PAGE], pos % PAGE
                fresh = rows[base:base + end - pos].permute(1, 2, 0, 3)             # [2, kv heads, rows, dim]
                e = _exact_rows(fresh)
                if at > 0:
                    e = torch.maximum(e, torch.log2(scales[page]))
                    codes[page, :, :, :at] = _e4m3(codes[page, :, :, :at] * (scales[page] / torch.exp2(e))[..., None, None])
                codes[page, :, :, at:at + end - pos] = _e4m3(fresh / torch.exp2(e)[..., None, None])
                scales[page] = torch.exp2(e)
                base, pos = base + end - pos, end
        return {"q": turned[:, :heads].reshape(s["q_out"].shape), "codes": codes, "scales": scales}
    out, base, group = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda"), 0, heads // kv_heads
    for i, (t, x) in enumerate(zip(new, lengths)):
        lo = max(0, x - t - case["window"] + 1) if case["window"] > 0 else 0
        ids = torch.tensor(table[slots[i]][lo // PAGE:-(-x // PAGE)], device="cuda")
        kv = (s["storage"][ids].double() * s["scales"][ids].double()[..., None, None]).permute(1, 2, 0, 3, 4).reshape(2, kv_heads, -1, dim)
        skip = lo // PAGE * PAGE
        for j in range(t):
            p = x - t + j
            first = max(0, p - case["window"] + 1) if case["window"] > 0 else 0
            k, v = kv[0, :, first - skip:p + 1 - skip], kv[1, :, first - skip:p + 1 - skip]
            q = s["q"][base + j].double().view(kv_heads, group, dim)
            w = torch.softmax(torch.einsum("hgd,hkd->hgk", q, k) * s["scale"], -1)
            out[base + j] = torch.einsum("hgk,hkd->hgd", w, v).reshape(-1)
        base += t
    return out
