"""The token behind a refused draft where draft and target logits are nearly, or exactly, the same: what is left of p when q is taken off is then small
beside both, and so beside what a sum or an exponential in float32 is off by."""
import math

import pytest
import torch

from tests.test_verify_drafts_gpu import Case

pytestmark = pytest.mark.gpu


class Close(Case):
    """Entries of one draft each: logits of the draft model are the target's but for `noise`, the draft is the token with the largest q / p, and the uniform
    the largest below 1, so that every draft is refused."""

    def __init__(self, n, vocab, noise, seed, temperature=0.9, sharp=2.0):
        super().__init__([1] * n, vocab, temperature, seed=seed, sharp=sharp)
        g = torch.Generator().manual_seed(seed + 1000)
        base = self.target[0::2]
        self.draft = (base.double() + noise * torch.randn(base.shape, generator=g, dtype=torch.float64)).float()
        p, q = (torch.softmax(x.double() / temperature, 1) for x in (base, self.draft))
        self.drafted = (q / p).argmax(1).to(torch.int32)
        self.uniforms = torch.full((n,), 1 - 2.0 ** -24)
        # (u q and p are as far apart as some 4 standard deviations of the logits' noise over the temperature: at 1e-5 20 times the decisions' 2^-19)


@pytest.mark.parametrize("noise", [1e-5, 3e-5, 1e-4, 1e-3])
@pytest.mark.parametrize("n,vocab", [(450, 30001), (40, 50000), (3, 151936)])   # (one block an entry; several; many)
def test_nearly_equal_models(n, vocab, noise):
    c = Close(n, vocab, noise, seed=n)
    accepted, tokens = c.want()
    assert accepted == [0] * n and c.margin > 2.0 ** -19
    assert c.run() == (accepted, tokens)


def test_a_flat_row_of_nearly_equal_models():
    """Every token's share is small, and no token's is far from another's."""
    c = Close(450, 4000, 2e-5, seed=9, temperature=1.0, sharp=1e-3)
    want = c.want()
    assert want[0] == [0] * 450 and c.margin > 2.0 ** -19
    assert c.run() == want


def test_nothing_is_left_of_equal_models():
    """A draft that is refused (an id outside the vocabulary) though p = q: every token's score is 0, and the lowest id is taken."""
    for with_draft, n, vocab in ((True, 450, 5000), (True, 2, 20000), (False, 3, 1)):
        c = Case([1] * n, vocab, 0.9, with_draft, seed=4)
        if with_draft:
            c.draft = c.target[0::2].clone()
            c.drafted[:] = -1
        else:   # (the only token there is, which is refused)
            c.drafted[:] = 0
            c.uniforms[:] = 1 - 2.0 ** -24
            c.target[0::2] = -math.inf
        accepted, tokens = c.run()
        assert accepted == [0] * n and tokens == [[0, -1]] * n
