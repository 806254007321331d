"""The entries for several continuations of one prompt check and launch in native code where everything is in order, and in Python otherwise: both do
the same."""
import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.ops import branches
from tests.test_attention_shared_gpu import Batch
from tests.test_copy_pages_gpu import draw_moves, expected, random_storage
from tests.test_verify_drafts_gpu import Case

pytestmark = pytest.mark.gpu


def watch(monkeypatch, name, library):
    """The answers of a native function from now on."""
    native, answers = branches._native(name, library), []

    def watched(*args):
        answers.append(native(*args))
        return answers[-1]
    monkeypatch.setitem(branches._functions, name, watched)
    return answers


def without(monkeypatch, name):
    monkeypatch.setitem(branches._functions, name, lambda *args: None)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(14, 2, 64, torch.bfloat16), (4, 2, 96, torch.bfloat16), (6, 3, 20, torch.float32)])
def test_attention(monkeypatch, heads, kv_heads, dim, dtype):
    b = Batch([([0, 2], 4)], [5, 6, 70], heads, kv_heads, dim, dtype)
    answers = watch(monkeypatch, "attention_shared", "attention_shared")
    sinks = torch.linspace(-3, 3, heads, device="cuda")
    for kw in ({}, {"sinks": sinks}, {"max_kv_len": None}):
        b.run(**kw)   # (Python's first, which sizes the workspaces)
        before = ops.kernels.launches
        native = b.run(**kw).clone()
        assert ops.kernels.launches - before == 2 and answers[-1] == 0
        with monkeypatch.context() as m:
            without(m, "attention_shared")
            assert torch.equal(b.run(**kw), native)


def test_attention_that_native_code_does_not_take(monkeypatch):
    b = Batch([([0, 2], 4)], [5, 6, 70], 14, 2, 64, torch.bfloat16)
    answers = watch(monkeypatch, "attention_shared", "attention_shared")
    b.run()
    b.run()
    assert answers == [0]
    small = ops.SharedScratch("cuda")
    ops.attention_shared(b.q, b.out, b.cu_q, b.tok_pos, b.slots, b.site, b.heads, b.n, b.scale, b.share, small, b.err, max_kv_len=max(b.lengths))
    assert answers[-1] is None
    b.check()
    for bad in (dict(sinks=torch.zeros(13, device="cuda")), dict(sinks=torch.zeros(14)), dict(max_kv_len="long")):
        with pytest.raises((ops.KernelError, ValueError)):
            b.run(**bad)


@pytest.mark.parametrize("temperature,with_draft", [(0.0, True), (0.8, True), (0.8, False)])
def test_drafts(monkeypatch, temperature, with_draft):
    case, scratch = Case([3, -1, 0, 5], 9001, temperature, with_draft), ops.VerifyScratch()
    answers = watch(monkeypatch, "verify_drafts", "verify_drafts")
    first = case.run(scratch)
    assert answers == [None]   # (no workspaces yet)
    assert case.run(scratch) == first and answers[-1] == 0
    without(monkeypatch, "verify_drafts")
    assert case.run(scratch) == first == tuple(case.want())


@pytest.mark.parametrize("shape", [(3, 9, 2, 2, 64, 64), (2, 7, 1, 1, 64, 23), (2, 6, 5, 3), (2, 12, 7), (5, 8)])
def test_pages(monkeypatch, shape):
    answers = watch(monkeypatch, "copy_pages", "page_copy")
    storage = random_storage(shape, torch.bfloat16)
    moves = draw_moves(shape[1], 3, shape[-2] if len(shape) >= 4 else 1, 1, 1000)
    for given in (moves, [m[:2] for m in moves], [list(m) for m in moves], tuple(moves)):
        here, want = storage.clone(), expected(storage, given)
        ops.copy_pages(here, given)
        assert torch.equal(here, want)
    assert answers == [0, 0, None, None]
    for bad in ([(0, shape[1], 1)], [(0, 1, 99)], [(0, 1, -1)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(0, 2 ** 31, 1)], [(0, 2 ** 80, 1)], [(0, 1), (2, 3, 1)],
                [(0, 1, 1, 1)], [(0, 1.0, 1)]):
        here = storage.clone()
        with pytest.raises(ops.KernelError):
            ops.copy_pages(here, bad)
        assert torch.equal(here, storage)
