"""Operators for several continuations of one prompt, in plain form and as this library's calls.

  attention_shared  single tokens of sequences whose caches begin with the same pages: the common part is attended to once for all
  copy_pages        rows of cache pages copied inside a group's storage, every schedule entry at once (a fork's last page, a compaction)
  verify_drafts     drafted tokens accepted or refused against the target model's logits, and the token that follows them

`run` computes the plain form (elementary torch operations) where `own` is false and makes the library's calls where it is true.
Sizes are those of the Qwen2.5 presets (heads, head size, layers, vocabulary) and of the test configurations.
"""
import math
import zlib

import numpy as np
import torch

own = False

PAGE = 64                       # positions of a cache page
MASK = 0xFFFFFFFF
# (query heads, kv heads, head size): the 0.5B, 3B and 7B presets, and two shapes of the tests
HEADS = {"0.5b": (14, 2, 64), "3b": (16, 2, 128), "7b": (28, 4, 128), "small": (7, 1, 64), "wide": (6, 3, 96)}
LAYERS = {"0.5b": 24, "3b": 36, "7b": 28, "small": 2, "wide": 3}


# ------------------------------------------------------------------------------------------------ cases
def _attention(name, model, groups, alone, own_most, dtype="bfloat16"):
    """groups: "members x pages" per prompt; alone: sequences that share nothing; own_most: most tokens behind the shared pages."""
    return {"name": name, "kind": "attention", "model": model, "groups": groups, "alone": alone, "own_most": own_most, "dtype": dtype}


def _copy(name, model, pages, kind, moves, dtype="bfloat16"):
    return {"name": name, "kind": "copy", "model": model, "pages": pages, "what": kind, "moves": moves, "dtype": dtype}


def _verify(name, vocab, seqs, drafts, temperature, draft_logits):
    return {"name": name, "kind": "verify", "vocab": vocab, "seqs": seqs, "drafts": drafts, "temperature": temperature,
            "draft_logits": draft_logits}


def listed():
    return [
        # two answers to one question, a few tokens in: the smallest call, all latency
        _attention("answers-2", "0.5b", "2x16", 0, 9),
        # eight samples of one prompt of 4,096 tokens
        _attention("samples-8", "0.5b", "8x64", 0, 300),
        # a batch of two prompts with system texts of their own, and requests that share nothing
        _attention("two-prompts", "3b", "20x31,23x95", 5, 700),
        # a search over 64 branches behind 8,192 tokens
        _attention("branches-64", "7b", "64x128", 0, 500),
        # 250 short answers to questions about one document of 16,000 tokens
        _attention("document-250", "0.5b", "250x250", 0, 130),
        # a group of branches in the float32 path
        _attention("float32-12", "0.5b", "12x24", 1, 200, "float32"),
        # a prompt forked seven times: one partly filled page, copied to each fork, all layers at once
        _copy("fork-7", "0.5b", 96, "fork", 7),
        # many sequences forked once each in a step of a search, ragged last pages
        _copy("fork-each-64", "3b", 160, "forks", 64),
        # live pages moved to the front of the storage
        _copy("compact-120", "3b", 300, "compact", 120),
        # one sequence with four drafted tokens
        _verify("draft-4", 151936, 1, 4, 0.8, True),
        # a batch with up to seven drafts each, ragged
        _verify("draft-batch", 151936, 48, 7, 1.0, True),
        # greedy decoding with drafts looked up in the prompt (no draft model)
        _verify("lookup-greedy", 152064, 16, 5, 0.0, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "copy", "verify", "verify"])
    if kind == "attention":
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        model = rng.choice(list(HEADS))
        heads, kv_heads, dim = HEADS[model]
        groups, left = [], 250
        for _ in range(rng.choice([1, 1, 1, 2, 3])):
            members = min(left, _log_int(rng, 1, 250))
            if members < 1:
                break
            left -= members
            # (no more score products than the largest listed case has, a twentieth of them in float32)
            most = 250 * 250 * 14 * 64 / (members * heads * dim) / 3
            if dtype == "float32":
                most /= 20
            groups.append(f"{members}x{min(250, max(1, min(int(most), _log_int(rng, 1, 250))))}")
        alone = rng.choice([0, 0, 1, rng.randint(1, 12)])
        return _attention(None, model, ",".join(groups), min(alone, left), _log_int(rng, 1, 400), dtype)
    if kind == "copy":
        model = rng.choice(list(LAYERS))
        what = rng.choice(["fork", "forks", "compact"])
        pages = _log_int(rng, 8, 260)
        return _copy(None, model, pages, what, max(1, min(pages // 2 - 1, _log_int(rng, 1, 100))), rng.choice(["bfloat16", "bfloat16", "float32"]))
    vocab = rng.choice([151936, 152064, rng.randint(200, 60000), rng.randint(200, 60000)])
    seqs = _log_int(rng, 1, 48)
    return _verify(None, vocab, seqs, rng.randint(1, 7), rng.choice([0.0, 0.3 + rng.random(), 1.0]), rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed, where="cuda"):
    return torch.Generator(device=where).manual_seed(int(seed) + 1)


def _sizes(case):
    """The generator of a case's ragged sizes: the case's own, so that every seed has the same work."""
    return np.random.default_rng(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))


def _layout(case):
    """Members and pages of every group in a shuffled batch, and every sequence's own tokens (the new one among them)."""
    rng = _sizes(case)
    sizes = [tuple(int(x) for x in g.split("x")) for g in case["groups"].split(",")]
    n = sum(m for m, _ in sizes) + case["alone"]
    order = rng.permutation(n).tolist()
    groups, at = [], 0
    for members, pages in sizes:
        groups.append((sorted(order[at:at + members]), pages))
        at += members
    prefix = [0] * n
    for members, pages in groups:
        for s in members:
            prefix[s] = pages
    own_tokens = rng.integers(1, case["own_most"] + 1, n).tolist()
    return groups, prefix, own_tokens


def _prepare_attention(case, seed):
    heads, kv_heads, dim = HEADS[case["model"]]
    dtype = getattr(torch, case["dtype"])
    groups, prefix, own_tokens = _layout(case)
    n = len(prefix)
    lengths = [p * PAGE + t for p, t in zip(prefix, own_tokens)]
    columns = max(-(-x // PAGE) for x in lengths)
    n_pages = sum(p for _, p in groups) + sum(-(-t // PAGE) for t in own_tokens)
    ids = np.random.default_rng(int(seed) + 29).permutation(n_pages).tolist()   # pages lie anywhere in the storage
    table = np.full((n + 2, columns), -1, dtype=np.int32)
    slots = np.random.default_rng(int(seed) + 31).permutation(n + 2)[:n].astype(np.int32)
    for members, pages in groups:
        common = [ids.pop() for _ in range(pages)]
        for s in members:
            table[slots[s], :pages] = common
    for s in range(n):
        for p in range(prefix[s], -(-lengths[s] // PAGE)):
            table[slots[s], p] = ids.pop()
    g = _generator(seed)
    storage = torch.randn((n_pages, 2, kv_heads, PAGE, dim), device="cuda", generator=g).to(dtype)
    q = (1.5 * torch.randn((n, heads * dim), device="cuda", generator=g)).to(dtype)
    to = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    state = dict(case=case, groups=groups, prefix=to(prefix), storage=storage, table=to(table), q=q, out=torch.zeros_like(q),
                 cu_q=torch.arange(n + 1, dtype=torch.int32, device="cuda"), tok_pos=to([x - 1 for x in lengths]), slots=to(slots),
                 own_most=max(own_tokens), longest=max(lengths), n=n, scale=dim ** -0.5)
    if own:
        from qwenforge_b200 import ops
        state["share"] = ops.SharedPrefix(groups, n, "cuda")
        state["scratch"] = ops.SharedScratch("cuda")
        state["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return state


def _copied_rows(case):
    n, rng = case["moves"], _sizes(case)
    if case["what"] == "compact":
        return [PAGE] * n
    rows = rng.integers(1, PAGE + 1, n).tolist()
    return rows[:1] * n if case["what"] == "fork" else rows


def _prepare_copy(case, seed):
    heads, kv_heads, dim = HEADS[case["model"]]
    rng = np.random.default_rng(int(seed) + 41)
    ids = rng.permutation(case["pages"]).tolist()
    n, rows = case["moves"], _copied_rows(case)
    if case["what"] == "fork":        # one page to n others, its first rows
        source = ids.pop()
        moves = [(source, ids.pop(), r) for r in rows]
    elif case["what"] == "forks":     # n pages to one other each
        moves = [(ids.pop(), ids.pop(), r) for r in rows]
    else:                             # whole pages from the back to free ones at the front
        free = sorted(rng.permutation(case["pages"] // 2)[:n].tolist())
        back = sorted((case["pages"] // 2 + rng.permutation(case["pages"] - case["pages"] // 2)[:n]).tolist())
        moves = [(b, f, r) for b, f, r in zip(reversed(back), free, rows)]
    storage = torch.randn((LAYERS[case["model"]], case["pages"], 2, kv_heads, PAGE, dim), device="cuda", generator=_generator(seed))
    return dict(case=case, storage=storage.to(getattr(torch, case["dtype"])), moves=moves)


def _draft_counts(case):
    if case["seqs"] == 1:
        return [case["drafts"]]
    return _sizes(case).integers(0, case["drafts"] + 1, case["seqs"]).tolist()


def _prepare_verify(case, seed):
    counts = _draft_counts(case)
    n, total, vocab = len(counts), sum(counts), case["vocab"]
    first = np.concatenate([[0], np.cumsum([c + 1 for c in counts])]).astype(np.int32)
    g = _generator(seed)
    # a language model's logits: a broad bulk and a few tokens far above it
    target = 2.0 * torch.randn((n + total, vocab), device="cuda", generator=g)
    ahead = torch.randint(0, vocab, (n + total, 12), device="cuda", generator=g)
    target.scatter_add_(1, ahead, 4.0 + 9.0 * torch.rand((n + total, 12), device="cuda", generator=g))
    rows = torch.tensor([first[s] + j for s in range(n) for j in range(counts[s])], dtype=torch.long, device="cuda")
    draft = target[rows] + 0.7 * torch.randn((total, vocab), device="cuda", generator=g)
    noise = -torch.log(-torch.log(torch.rand((total, vocab), device="cuda", generator=g).clamp_(1e-7, 1 - 1e-6)))
    sharp = max(case["temperature"], 0.05)
    drafted = (draft / sharp + noise).argmax(1).to(torch.int32) if total else torch.zeros(0, dtype=torch.int32, device="cuda")
    to = lambda a, t=torch.int32: torch.tensor(a, dtype=t, device="cuda")
    state = dict(case=case, n=n, most=case["drafts"], target=target, draft=draft if case["draft_logits"] else None, drafted=drafted,
                 first=to(first), uniforms=torch.rand(total, device="cuda", generator=g), temperature=float(case["temperature"]),
                 seed=int(seed) * 2654435761 + 12345, seq_ids=to([7 * s + 3 for s in range(n)], torch.int64),
                 steps=to([11 * s % 50 for s in range(n)]), accepted=torch.zeros(n, dtype=torch.int32, device="cuda"),
                 tokens=torch.zeros((n, case["drafts"] + 1), dtype=torch.int32, device="cuda"))
    if own:
        from qwenforge_b200 import ops
        state["scratch"] = ops.VerifyScratch()
    return state


def prepare(case, seed):
    return {"attention": _prepare_attention, "copy": _prepare_copy, "verify": _prepare_verify}[case["kind"]](case, seed)


# ------------------------------------------------------------------------------------------------ one pass
def _run_attention(s):
    heads, kv_heads, dim = HEADS[s["case"]["model"]]
    if own:
        from qwenforge_b200 import ops
        site = ops.KvSiteArgs(s["storage"], s["table"], kv_heads, dim)
        ops.attention_shared(s["q"], s["out"], s["cu_q"], s["tok_pos"], s["slots"], site, heads, s["n"], s["scale"], s["share"],
                             s["scratch"], s["err"], max_kv_len=s["longest"])
        return s["out"]
    n, group = s["n"], heads // kv_heads
    q = s["q"].float().view(n, kv_heads, group, dim) * s["scale"]
    rows = s["table"][s["slots"].long()].long()
    # every sequence's own positions, behind what it shares
    start = s["prefix"].long() * PAGE
    pos = start[:, None] + torch.arange(s["own_most"], device="cuda")
    seen = pos <= s["tok_pos"].long()[:, None]
    page = torch.gather(rows, 1, (pos // PAGE).clamp_(max=rows.shape[1] - 1)).clamp_(min=0)
    k = s["storage"][page, 0, :, pos % PAGE].float()      # [n, own, kv_heads, dim]
    v = s["storage"][page, 1, :, pos % PAGE].float()
    score = torch.einsum("nhgd,nphd->nhgp", q, k).masked_fill_(~seen[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    acc = torch.einsum("nhgp,nphd->nhgd", weight, v)
    out = torch.empty_like(q)
    grouped = torch.zeros(n, dtype=torch.bool)
    for members, pages in s["groups"]:
        index = torch.tensor(members, device="cuda")
        grouped[members] = True
        common = rows[members[0], :pages]
        k = s["storage"][common, 0].float().transpose(0, 1).reshape(kv_heads, pages * PAGE, dim)
        v = s["storage"][common, 1].float().transpose(0, 1).reshape(kv_heads, pages * PAGE, dim)
        score = torch.einsum("nhgd,hpd->nhgp", q[index], k)
        high = torch.maximum(score.amax(-1, keepdim=True), top[index])
        weight = torch.exp(score.sub_(high))
        keep = torch.exp(top[index] - high)
        den = weight.sum(-1, keepdim=True) + keep * total[index]
        out[index] = (torch.einsum("nhgp,hpd->nhgd", weight, v) + keep * acc[index]) / den
    rest = (~grouped).nonzero().flatten().cuda()
    out[rest] = acc[rest] / total[rest]
    return out.view(n, heads * dim).to(s["q"].dtype)


def _run_copy(s):
    if own:
        from qwenforge_b200 import ops
        ops.copy_pages(s["storage"], s["moves"])
        return s["storage"]
    moves = torch.tensor(s["moves"], dtype=torch.long).cuda()
    kept = torch.arange(PAGE, device="cuda")[None, :] < moves[:, 2:]
    storage = s["storage"]
    storage[:, moves[:, 1]] = torch.where(kept[None, :, None, None, :, None], storage[:, moves[:, 0]], storage[:, moves[:, 1]])
    return storage


def _mix32(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & MASK
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & MASK
    return x ^ (x >> 16)


def _waits(seed, seq_ids, steps, vocab):
    """-ln u of every (sequence, token): the sampler's own random numbers, keyed by (seed, sequence, step)."""
    seed &= (1 << 64) - 1
    key = _mix32(torch.full_like(seq_ids, (seed & MASK) ^ 0x9E3779B9))
    key = _mix32(key ^ (seed >> 32))
    key = _mix32(key ^ (seq_ids & MASK))
    key = _mix32(key ^ ((seq_ids >> 32) & MASK) ^ 0x85EBCA6B)
    key = _mix32(key ^ (steps.long() & MASK))
    i = torch.arange(vocab, device=seq_ids.device)
    bits = _mix32(key[:, None] ^ _mix32(i ^ 0x27D4EB2F)[None, :])
    return -torch.log(((bits >> 9).double() + 0.5) / 8388608.0)


def _run_verify(s):
    if own:
        from qwenforge_b200 import ops
        ops.verify_drafts(s["target"], s["draft"], s["drafted"], s["first"], s["uniforms"], s["temperature"], s["seed"], s["seq_ids"],
                          s["steps"], s["accepted"], s["tokens"], s["scratch"])
        return {"accepted": s["accepted"], "tokens": s["tokens"]}
    n, most, temperature = s["n"], s["most"], s["temperature"]
    first = s["first"].long()
    counts = first[1:] - first[:-1] - 1
    place = torch.arange(most, device="cuda")
    live = place[None, :] < counts[:, None]                                       # [n, most]
    at = (first[:-1] - torch.arange(n, device="cuda"))[:, None] + place           # the drafted token's index
    at = torch.where(live, at, torch.zeros_like(at))
    row = torch.where(live, first[:-1, None] + place, torch.zeros_like(at))
    drafted = s["drafted"].long()[at] if s["drafted"].numel() else torch.zeros_like(at)
    # in 64 bits: a decision must not turn on the last bits of a sum over the vocabulary
    if temperature <= 0:
        best = s["target"].argmax(1)
        ok = live & (best[row] == drafted)
    else:
        p = torch.softmax(s["target"].double() / temperature, 1)
        here = p[row, drafted]
        if s["draft"] is not None:
            q = torch.softmax(s["draft"].double() / temperature, 1)
            there = q[at, drafted] if q.shape[0] else torch.ones_like(here)
        else:
            there = torch.ones_like(here)
        u = s["uniforms"].double()[at] if s["uniforms"].numel() else torch.zeros_like(here)
        ok = live & (u * there < here)
    accepted = ok.long().cumprod(1).sum(1)
    chosen_row = first[:-1] + accepted
    if temperature <= 0:
        chosen = best[chosen_row]
    else:
        mass = p[chosen_row]
        refused = accepted < counts
        last = accepted.clamp(max=most - 1)[:, None]
        index, refused_token = at.gather(1, last)[:, 0], drafted.gather(1, last)
        if s["draft"] is None:
            mass.scatter_(1, refused_token, torch.where(refused[:, None], 0.0, mass.gather(1, refused_token)))
        elif q.shape[0]:
            mass = (mass - torch.where(refused[:, None], q[index], 0.0)).clamp_(min=0)
        chosen = (mass / _waits(s["seed"], s["seq_ids"], s["steps"].long() + accepted, mass.shape[1])).argmax(1)
    place = torch.arange(most + 1, device="cuda")[None, :]
    tokens = torch.cat((drafted, drafted[:, :1]), 1)
    tokens = torch.where(place < accepted[:, None], tokens, torch.where(place == accepted[:, None], chosen[:, None], -1))
    return {"accepted": accepted.to(torch.int32), "tokens": tokens.to(torch.int32)}


def run(state):
    return {"attention": _run_attention, "copy": _run_copy, "verify": _run_verify}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case.get("dtype") == "float32" else 2
    if case["kind"] == "attention":
        heads, kv_heads, dim = HEADS[case["model"]]
        groups, prefix, own_tokens = _layout(case)
        n = len(prefix)
        keys = sum(p for _, p in groups) * PAGE + sum(own_tokens)
        scores = sum((p * PAGE + t) for p, t in zip(prefix, own_tokens)) * heads
        return {"bytes": keys * kv_heads * dim * 2 * size + 2 * n * heads * dim * size, "flops": scores * dim * 4}
    if case["kind"] == "copy":
        _, kv_heads, dim = HEADS[case["model"]]
        row = LAYERS[case["model"]] * 2 * kv_heads * dim * size
        rows = _copied_rows(case)
        return {"bytes": row * (sum(rows) + (rows[0] if case["what"] == "fork" else sum(rows))), "flops": 0}
    counts = _draft_counts(case)
    rows = sum(counts) + len(counts) + (sum(counts) if case["draft_logits"] and case["temperature"] > 0 else 0)
    # (an exponential, a sum and a comparison for each logit)
    return {"bytes": rows * case["vocab"] * 4, "flops": rows * case["vocab"] * (3 if case["temperature"] > 0 else 1)}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def _exact_attention(case, seed):
    heads, kv_heads, dim = HEADS[case["model"]]
    s = _prepare_attention(case, seed)
    out = torch.empty((s["n"], heads, dim), dtype=torch.float64, device="cuda")
    table, lengths, slots = s["table"].cpu(), (s["tok_pos"] + 1).tolist(), s["slots"].tolist()
    for i in range(s["n"]):
        pages = table[slots[i], :-(-lengths[i] // PAGE)].long().cuda()
        # [pages, 2, kv_heads, 64, dim] -> [2, kv_heads, positions, dim]
        kv = s["storage"][pages].double().permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :lengths[i]]
        for h in range(heads):
            keys, values = kv[0, h * kv_heads // heads], kv[1, h * kv_heads // heads]
            z = keys @ s["q"][i, h * dim:(h + 1) * dim].double() / math.sqrt(dim)
            w = (z - z.max()).exp()
            out[i, h] = (w @ values) / w.sum()
    return out.view(s["n"], heads * dim)


def exact(case, seed):
    if case["kind"] == "attention":
        groups, prefix, own_tokens = _layout(case)
        heads, kv_heads, dim = HEADS[case["model"]]
        read = sum(p * PAGE + t for p, t in zip(prefix, own_tokens)) * kv_heads * dim
        return _exact_attention(case, seed) if read < 2.0e9 and len(prefix) * heads < 8000 else None
    return None   # copies and tokens are not computed numbers
