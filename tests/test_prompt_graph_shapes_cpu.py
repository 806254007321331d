"""Which prompt steps share a captured graph."""
from types import SimpleNamespace

import pytest
import torch

from qwenforge_b200.engine.graphs import PrefillGraphs
from qwenforge_b200.engine.step import pack_step


class Graph:
    def replay(self):
        pass


def captured(monkeypatch, cache_dtype, steps):
    """The steps that are captured when each of `steps`, lists of (start, tokens), comes twice."""
    seen = []

    def capture(self, cache, step):
        seen.append(step)
        return Graph(), torch.zeros(step.packed.size, dtype=torch.int32), None, 0

    monkeypatch.setattr(PrefillGraphs, "_capture", capture)
    graphs = PrefillGraphs(SimpleNamespace())
    for entries in steps:
        triples = [(slot, start, [1] * n) for slot, (start, n) in enumerate(entries)]
        for _ in range(2):
            graphs.run(SimpleNamespace(serial=1, kv_dtype=cache_dtype), pack_step(triples, None), triples, None)
    return seen


BEHIND = [[(start, 30)] for start in (0, 100, 226, 227, 400, 482, 483, 2000)]   # 30 .. 256, 257 .. 512, 513, 2030 after the step


def test_lengths_are_no_part_of_a_shape(monkeypatch):
    step, = captured(monkeypatch, None, BEHIND)
    assert step.max_span is None and step.max_q_len == 64


def test_a_cache_in_8_bits_has_a_bound_on_the_lengths(monkeypatch):
    steps = captured(monkeypatch, torch.float8_e4m3fn, BEHIND)
    assert [s.max_kv_len for s in steps] == [256, 512, 1024, 2048] and {s.max_q_len for s in steps} == {64}


@pytest.mark.parametrize("spans,bounds", [([2, 5, 6, 31, 32], [2, 6, 32]), ([33, 64, 65, 100], [64, 128])])
def test_and_one_on_the_spans(monkeypatch, spans, bounds):
    """Of the entries that have a slot: the padding entry that fills the shape up has as many tokens as it takes."""
    steps = captured(monkeypatch, torch.float8_e4m3fn, [[(10, n), (10, n)] for n in spans])
    assert sorted({s.max_span for s in steps}) == bounds
    for s in steps:
        assert all(n <= s.max_span for n, slot in zip(s.host_q_lens, s.host_slots) if slot >= 0) and max(s.host_q_lens) <= s.max_q_len
