"""What `Sampler.verify` draws where the drafts come from the sampler itself: the deciding model's distribution all the same."""
import pytest
import torch

from qwenforge_b200.sampling import Sampler, SamplingParams

pytestmark = pytest.mark.gpu


def counts_fit(counts, p):
    """Counts of n independent draws are within 5 standard deviations, sqrt(n p (1 - p)), of n p: a chance of 6e-7 per count under the
    hypothesis, and the inputs are fixed by their seeds."""
    n = counts.sum()
    assert ((counts - n * p).abs() <= 5 * torch.sqrt(n * p * (1 - p))).all(), ((counts - n * p) / torch.sqrt(n * p * (1 - p))).tolist()


@pytest.mark.parametrize("draws", [14, 15, 16])
def test_drafts_of_the_sampler_itself(draws):
    """Drafts that the same sampler drew for the same sequences and steps: the first token is a draw of the deciding model all the same."""
    n, vocab, t = 20000, 9, 0.8
    g = torch.Generator().manual_seed(draws)
    p_logits, q_logits = 1.5 * torch.randn(vocab, generator=g), 1.5 * torch.randn(vocab, generator=g)
    sampler = Sampler(SamplingParams(t, 99))
    ids, steps = torch.arange(n, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    draft_logits = q_logits.repeat(n, 1).cuda()
    drafted = sampler(draft_logits, ids, steps)
    first = 2 * torch.arange(n + 1, dtype=torch.int32, device="cuda")
    accepted, tokens = sampler.verify(p_logits.repeat(2 * n, 1).cuda(), drafted, first, 1, torch.rand(n, generator=g).cuda(), draft_logits, ids, steps)
    p, q = (torch.softmax(x.double() / t, 0) for x in (p_logits, q_logits))
    counts_fit(torch.bincount(tokens[:, 0].cpu().long(), minlength=vocab).double(), p)
    kept = torch.bincount(accepted.cpu().long(), minlength=2).double()
    share = torch.minimum(p, q).sum()
    counts_fit(kept, torch.stack((1 - share, share)))


def test_two_tokens_over_rounds_of_drafts():
    """A chain of two tokens, each step's logits given by the token before: two drafts, and for the sequences whose first was refused a second
    round that drafts one token with the numbers of the step that the refused round has drafted for already. Pairs are distributed as the model's."""
    n, vocab, t = 16000, 4, 1.1
    g = torch.Generator().manual_seed(3)
    p_logits, q_logits = 1.3 * torch.randn((vocab + 1, vocab), generator=g).cuda(), 1.3 * torch.randn((vocab + 1, vocab), generator=g).cuda()   # (row: the token before)
    sampler = Sampler(SamplingParams(t, 7))
    ids, i32 = torch.arange(n, device="cuda"), dict(dtype=torch.int32, device="cuda")
    start = torch.full((n,), vocab, device="cuda")
    zero, one = torch.zeros(n, **i32), torch.ones(n, **i32)
    d1 = sampler(q_logits[start], ids, zero)
    d2 = sampler(q_logits[d1.long()], ids, one)
    rows = torch.stack((start, d1.long(), d2.long()), 1).flatten()
    drafted, before = torch.stack((d1, d2), 1).flatten(), torch.stack((start, d1.long()), 1).flatten()
    accepted, tokens = [], []
    for half in (slice(0, n // 2), slice(n // 2, n)):   # (a call takes 65,535 rows)
        a, b = half.start, half.stop
        m = b - a
        out = sampler.verify(p_logits[rows[3 * a:3 * b]], drafted[2 * a:2 * b], 3 * torch.arange(m + 1, **i32), 2, torch.rand(2 * m, generator=g).cuda(),
                             q_logits[before[2 * a:2 * b]], ids[half], zero[half])
        accepted.append(out[0])
        tokens.append(out[1])
    accepted, tokens = torch.cat(accepted), torch.cat(tokens)
    again = (accepted == 0).nonzero().flatten()
    m, last = again.numel(), tokens[again, 0].long()
    draft_logits = q_logits[last]
    d = sampler(draft_logits, ids[again], one[again])
    out = sampler.verify(p_logits[torch.stack((last, d.long()), 1).flatten()], d, 2 * torch.arange(m + 1, **i32), 1, torch.rand(m, generator=g).cuda(), draft_logits,
                         ids[again], one[again])[1]
    tokens[again, 1] = out[:, 0]
    p = torch.softmax(p_logits.cpu().double() / t, 1)
    pair = (tokens[:, 0] * vocab + tokens[:, 1]).cpu().long()
    counts_fit(torch.bincount(pair, minlength=vocab * vocab).double(), (p[vocab][:, None] * p[:vocab]).flatten())
