"""`ops.verify_drafts` against its definition in float64, token for token; against the sampler; the distribution it draws from; refusals.

What is compared is whole numbers. The kernel's decisions are made on sums and exponentials that are good to 2^-20, so inputs on which a
decision is closer than that (u q(d) against p(d), the two largest scores of a draw) are not told apart; `Case.margin` says how close the
closest decision of a case is, and the cases, which are fixed by their seeds, are required to be further apart than 2^-19."""
import math

import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.sampling import Sampler, SamplingParams

pytestmark = pytest.mark.gpu
MASK = 0xFFFFFFFF


def mix32(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & MASK
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & MASK
    return x ^ (x >> 16)


def waits(seed, seq_id, step, vocab):
    """-ln of the sampler's number for every token of one draw, float64."""
    seed &= 2 ** 64 - 1
    key = mix32((seed & MASK) ^ 0x9E3779B9)
    key = mix32(key ^ (seed >> 32))
    key = mix32(key ^ (seq_id & MASK))
    key = mix32(key ^ ((seq_id >> 32) & MASK) ^ 0x85EBCA6B)
    key = mix32(key ^ (step & MASK))
    i = torch.arange(vocab, dtype=torch.int64)
    bits = mix32(torch.tensor(key) ^ mix32(i ^ 0x27D4EB2F))
    return -torch.log(((bits >> 9).double() + 0.5) / 2 ** 23)


class Case:
    def __init__(self, counts, vocab, temperature, with_draft=True, seed=0, stride=0, sharp=2.0, most=None):
        g = torch.Generator().manual_seed(seed)
        self.counts, self.vocab, self.temperature, self.seed = counts, vocab, temperature, 1234567 + (seed << 33)
        n, total = len(counts), sum(c for c in counts if c >= 0)
        rows = sum(c + 1 for c in counts)
        self.n, self.most = n, max([0] + counts) if most is None else most
        self.target = sharp * torch.randn((rows, vocab), generator=g)
        self.first = torch.tensor([0] + torch.tensor([c + 1 for c in counts]).cumsum(0).tolist(), dtype=torch.int32)
        at = [int(self.first[s]) + j for s in range(n) for j in range(counts[s])]
        self.draft = self.target[at] + 0.5 * torch.randn((total, vocab), generator=g) if with_draft else None
        base = self.draft if with_draft else self.target[at]
        self.drafted = (base + 1.5 * torch.randn(base.shape, generator=g)).argmax(-1).to(torch.int32) if total else torch.zeros(0, dtype=torch.int32)
        self.uniforms = torch.rand(total, generator=g)
        self.seq_ids = torch.tensor([s * 7 + (s % 2 << 40) for s in range(n)], dtype=torch.int64)
        self.steps = torch.tensor([5 * s for s in range(n)], dtype=torch.int32)
        self.stride = stride

    def run(self, scratch=None):
        pad = lambda t: None if t is None else torch.cat((t, torch.full((t.shape[0], self.stride), 99.0)), 1).cuda()[:, :self.vocab]
        self.accepted = torch.full((self.n,), -9, dtype=torch.int32, device="cuda")
        self.tokens = torch.full((self.n, self.most + 1), -9, dtype=torch.int32, device="cuda")
        ops.verify_drafts(pad(self.target), pad(self.draft), self.drafted.cuda(), self.first.cuda(), self.uniforms.cuda(), self.temperature, self.seed,
                          self.seq_ids.cuda(), self.steps.cuda(), self.accepted, self.tokens, scratch)
        return self.accepted.tolist(), self.tokens.tolist()

    def want(self):
        accepted, tokens, at, self.margin = [], [], 0, math.inf
        for s, count in enumerate(self.counts):
            row = int(self.first[s])
            if count < 0:
                accepted.append(0)
                tokens.append([-1] * (self.most + 1))
                continue
            kept, refused = 0, False
            p_of = lambda r: torch.softmax(self.target[r].double() / self.temperature, 0)
            q_of = lambda r: torch.softmax(self.draft[r].double() / self.temperature, 0)
            for j in range(count):
                d = int(self.drafted[at + j])
                if self.temperature <= 0:
                    ok = int(self.target[row + j].argmax()) == d
                else:
                    p = float(p_of(row + j)[d]) if 0 <= d < self.vocab else 0.0
                    q = 1.0 if self.draft is None else float(q_of(at + j)[d]) if 0 <= d < self.vocab else 1.0
                    ok = 0 <= d < self.vocab and float(self.uniforms[at + j]) * q < p
                    if 0 <= d < self.vocab and max(p, q) > 0:
                        self.margin = min(self.margin, abs(float(self.uniforms[at + j]) * q - p) / max(p, q))
                if not ok:
                    refused = True
                    break
                kept += 1
            if self.temperature <= 0:
                token = int(self.target[row + kept].argmax())
            else:
                mass = p_of(row + kept)
                slack = mass.clone()
                if refused and self.draft is not None:
                    q = q_of(at + kept)
                    slack = mass + q
                    mass = (mass - q).clamp(min=0)
                elif refused and 0 <= int(self.drafted[at + kept]) < self.vocab:
                    mass[int(self.drafted[at + kept])] = 0
                score = mass / waits(self.seed, int(self.seq_ids[s]), int(self.steps[s]) + kept, self.vocab)
                token = int(score.argmax())
                two = score.topk(min(2, self.vocab)).values
                if len(two) > 1 and float(two[0]) > 0:
                    self.margin = min(self.margin, float((two[0] - two[1]) / two[0]))
            accepted.append(kept)
            tokens.append(self.drafted[at:at + kept].tolist() + [token] + [-1] * (self.most - kept))
            at += count
        return accepted, tokens

    def check(self, **kw):
        want = self.want()
        assert self.margin > 2.0 ** -19, self.margin
        assert self.run(**kw) == want


COUNTS = [[0], [4], [0, 3, 1], [7, 0, 5, 2, 1, 0, 6], [1] * 20, [13, 2]]


@pytest.mark.parametrize("vocab", [1, 7, 256, 2048, 2051, 8192, 20001])
@pytest.mark.parametrize("temperature", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("with_draft", [True, False])
def test_tokens(vocab, temperature, with_draft):
    for i, counts in enumerate(COUNTS):
        Case(counts, vocab, temperature, with_draft, seed=i).check()


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_a_whole_vocabulary(temperature):
    Case([4, 0, 2], 151936, temperature, seed=3, sharp=3.0).check()
    Case([3], 152064, temperature, with_draft=False, seed=4, sharp=3.0).check()


@pytest.mark.parametrize("stride", [1, 3, 4])
def test_rows_at_any_distance(stride):
    Case([3, 2], 5000, 0.9, seed=5, stride=stride).check()


def test_entries_without_rows_and_wrong_ones():
    c = Case([2, -1, 3, -1, -1, 1, -1], 500, 0.9, seed=6)
    c.check()
    good = c.want()
    c.most = 2   # no room for the third draft of entry 2
    accepted, tokens = c.run()
    assert accepted == [good[0][0], 0, -1, 0, 0, good[0][5], 0] and tokens[2] == [-1] * 3
    c = Case([2, 3], 500, 0.9, seed=7)
    c.first = torch.tensor([0, 3, 9], dtype=torch.int32)   # rows that are not there
    assert c.run()[0][1] == -1
    c.first = torch.tensor([0, -3, 4], dtype=torch.int32)
    assert c.run()[0] == [-1, -1]


def test_ids_outside_the_vocabulary_are_refused():
    for with_draft in (True, False):
        for bad in (-1, 300, 2 ** 31 - 1):
            for temperature in (0.0, 1.0):
                c = Case([3, 2], 300, temperature, with_draft, seed=8)
                c.drafted[0] = bad
                c.check()


def test_masked_and_certain_logits():
    """-infinity in both models' logits; a row with one token left; drafts that either model rules out."""
    for with_draft in (True, False):
        c = Case([3, 3, 1], 3000, 0.7, with_draft, seed=9)
        c.target[:, ::2] = -math.inf
        c.target[1] = -math.inf
        c.target[1, 1234] = 5.0
        c.drafted[1] = 1234
        c.target[4] = -math.inf
        c.target[4, 7] = -3.0
        if with_draft:
            c.draft[:, ::3] = -math.inf
            c.draft[1, 1234] = 2.0
        c.drafted[5] = 2
        c.check()


def test_extreme_logits():
    for scale in (1e4, 1e30):
        c = Case([3, 0, 2], 4000, 1.0, seed=10)
        c.target *= scale
        c.draft *= scale
        accepted, tokens = c.run()
        assert (accepted, tokens) == c.want()


def test_equal_logits_take_the_lowest_id():
    c = Case([2, 0], 9000, 0.0, with_draft=False, seed=11)
    c.target[:] = 1.0
    c.drafted[:] = torch.tensor([0, 1], dtype=torch.int32)
    assert c.run() == ([1, 0], [[0, 0, -1], [0, -1, -1]])


def test_nothing_drafted_is_the_sampler():
    """Without drafts the next token is the one that `sample` draws under the same key."""
    for temperature in (0.0, 0.6, 1.3):
        c = Case([0] * 40, 30000, temperature, seed=12)
        c.check()
        out = Sampler(SamplingParams(temperature, c.seed))(c.target.cuda(), c.seq_ids.cuda(), c.steps.cuda())
        assert out.tolist() == c.tokens[:, 0].tolist()


def test_equal_models_keep_every_draft():
    c = Case([5, 5], 2000, 0.9, seed=13)
    c.draft = torch.cat((c.target[0:5], c.target[6:11]))
    assert c.run()[0] == [5, 5]


def test_the_first_token_is_distributed_as_the_model_says():
    """Whatever the draft model proposes, the first token of an entry is a draw from p: the counts of n entries are within 5 standard
    deviations, sqrt(n p (1 - p)), of n p (for 9 tokens a chance of 5e-6 under the hypothesis, and the inputs are fixed)."""
    n, vocab, t = 20000, 9, 0.8
    g = torch.Generator().manual_seed(14)
    p_logits, q_logits = 1.5 * torch.randn(vocab, generator=g), 1.5 * torch.randn(vocab, generator=g)
    for with_draft in (True, False):
        q = torch.softmax(q_logits.double() / t, 0) if with_draft else torch.nn.functional.one_hot(torch.tensor(4), vocab).double()
        drafted = torch.multinomial(q, n, replacement=True, generator=g).to(torch.int32).cuda()
        accepted, tokens = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros((n, 2), dtype=torch.int32, device="cuda")
        ops.verify_drafts(p_logits.repeat(2 * n, 1).cuda(), q_logits.repeat(n, 1).cuda() if with_draft else None, drafted,
                          2 * torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.rand(n, generator=g).cuda(), t, 99,
                          torch.arange(n, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), accepted, tokens)
        p = torch.softmax(p_logits.double() / t, 0)
        counts = torch.bincount(tokens[:, 0].cpu().long(), minlength=vocab).double()
        assert ((counts - n * p).abs() <= 5 * torch.sqrt(n * p * (1 - p))).all()
        kept = float((accepted > 0).double().mean())
        share = float(torch.minimum(p, q).sum())
        assert abs(kept - share) <= 5 * math.sqrt(share * (1 - share) / n)


def test_captured_twice_with_scratches_of_their_own():
    cases = [Case([3, 0, 2], 20000, 0.9, seed=20), Case([1, 4], 20000, 0.9, seed=21)]
    graphs = []
    for c in cases:
        c.want()
        args = [t.cuda() for t in (c.target, c.draft, c.drafted, c.first, c.uniforms)]
        c.accepted, c.tokens = torch.zeros(c.n, dtype=torch.int32, device="cuda"), torch.zeros((c.n, c.most + 1), dtype=torch.int32, device="cuda")
        scratch, ids, steps = ops.VerifyScratch(), c.seq_ids.cuda(), c.steps.cuda()
        call = lambda: ops.verify_drafts(*args, 0.9, c.seed, ids, steps, c.accepted, c.tokens, scratch)
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, args, scratch, ids, steps))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for c in cases:
            c.accepted.zero_()
            c.tokens.zero_()
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for c in cases:
            assert (c.accepted.tolist(), c.tokens.tolist()) == c.want()


def test_refusals():
    c = Case([2, 1], 300, 0.9, seed=15)
    good = dict(target=c.target.cuda(), draft=c.draft.cuda(), drafted=c.drafted.cuda(), first=c.first.cuda(), uniforms=c.uniforms.cuda(), temperature=0.9, seed=1,
                seq_ids=c.seq_ids.cuda(), steps=c.steps.cuda(), accepted=torch.zeros(2, dtype=torch.int32, device="cuda"),
                tokens=torch.zeros((2, 3), dtype=torch.int32, device="cuda"))
    ops.verify_drafts(**good)
    for name, bad in (("target", good["target"].double()), ("target", good["target"].t()), ("target", good["target"].view(-1)), ("draft", good["draft"][:2]),
                      ("draft", good["draft"][:, :200]), ("draft", good["draft"].half()), ("drafted", good["drafted"][:2]), ("drafted", good["drafted"].long()),
                      ("first", good["first"][:2]), ("uniforms", good["uniforms"][:2]), ("uniforms", good["uniforms"].double()), ("seq_ids", good["seq_ids"].int()),
                      ("seq_ids", good["seq_ids"][:1]), ("steps", good["steps"][:1]), ("tokens", good["tokens"][:1]), ("tokens", good["tokens"][:, ::2]),
                      ("accepted", good["accepted"].long()), ("target", good["target"].cpu())):
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(**{**good, name: bad})
