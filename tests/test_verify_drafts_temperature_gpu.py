"""Temperatures close to zero: what is drawn is the argmax, whatever 1 / T overflows to."""
import pytest

from tests.test_verify_drafts_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [1e-6, 1e-30, 1e-38, 1e-40, 1.5e-45, 1e-50])
@pytest.mark.parametrize("with_draft", [True, False])
def test_tiny_temperatures(temperature, with_draft):
    c = Case([3, 0, 2, 4], 9001, temperature, with_draft, seed=2)
    best = c.target.argmax(1)
    at = [0, 1, 2, 5, 6, 8, 9, 10, 11]   # the rows that decide on drafts
    c.drafted[:] = best[at].to(c.drafted.dtype)
    c.drafted[4] = (c.drafted[4] + 1) % 9001   # entry 2 keeps its first draft only
    if with_draft:
        c.draft.fill_(-1.0)
        for j, d in enumerate(c.drafted.tolist()):
            c.draft[j, d] = 3.0
    accepted, tokens = c.run()
    assert accepted == [3, 0, 1, 4]
    rows = [3, 4, 6, 12]
    for s, (kept, row) in enumerate(zip(accepted, tokens)):
        assert row[kept] == int(best[rows[s]])
