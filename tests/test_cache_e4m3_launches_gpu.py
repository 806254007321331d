"""The entries of a cache in 8 bits check and launch in native code where everything is in order, and in Python otherwise: both do the same."""
import pytest
import torch

from qwenforge_b200 import ops
from tests.test_attention_e4m3_gpu import SPANS, TOKENS, query
from tests.test_branches_launches_gpu import watch, without
from tests.test_cache_e4m3_gpu import Case

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(14, 2, 64, torch.bfloat16), (4, 2, 96, torch.bfloat16), (28, 4, 128, torch.float32)])


@KINDS
@pytest.mark.parametrize("bias", [True, False])
def test_write(monkeypatch, heads, kv_heads, dim, dtype, bias):
    make = lambda: Case(SPANS + TOKENS, heads, kv_heads, dim, dtype, seed=2, bias=bias)   # noqa: E731
    a, b = make(), make()
    answers = watch(monkeypatch, "rope_cache_write_e4m3", "cache_e4m3")
    before = ops.kernels.launches
    q = a.write()
    assert answers == [0] and ops.kernels.launches == before + 1
    with monkeypatch.context() as m:
        without(m, "rope_cache_write_e4m3")
        assert torch.equal(b.write(), q)
    assert torch.equal(a.raw, b.raw) and torch.equal(a.held_scales, b.held_scales)


@KINDS
@pytest.mark.parametrize("window", [0, 37])
def test_read(monkeypatch, heads, kv_heads, dim, dtype, window):
    c = Case(SPANS, heads, kv_heads, dim, dtype, seed=2)
    answers = watch(monkeypatch, "cache_read_e4m3", "cache_e4m3")
    outs = []
    for native in (True, False):
        out = torch.zeros(c.codes.shape, dtype=dtype, device="cuda")
        with monkeypatch.context() as m:
            if not native:
                without(m, "cache_read_e4m3")
            ops.cache_read_e4m3(out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, c.n, 800, c.err, window=window)
        outs.append(out)
    assert answers == [0] and torch.equal(*outs) and bool(outs[0].any())


@KINDS
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("max_kv_len", [None, 1400])
def test_attention(monkeypatch, heads, kv_heads, dim, dtype, window, max_kv_len):
    for entries in (TOKENS, SPANS):
        c = Case(entries, heads, kv_heads, dim, dtype, seed=2)
        q, scratch, outs = query(c).cuda(), ops.E4m3Scratch("cuda"), []
        answers = watch(monkeypatch, "attention_e4m3", "attention_e4m3")
        for native in (None, True, False):   # (Python's first, which sizes the workspaces)
            out = torch.empty_like(q)
            with monkeypatch.context() as m:
                if native is False:
                    without(m, "attention_e4m3")
                ops.attention_e4m3(q, out, c.dev["cu_q"], c.dev["tok_pos"], c.dev["slots"], c.site, heads, c.n, c.most, 0.1, window, scratch, c.err, max_kv_len)
            outs.append(out)
        assert answers == [None, 0] and torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
