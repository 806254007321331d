"""`ops.verify_drafts` by callers that bring no workspaces: on several streams and threads at once, with sizes that change, and under a capture."""
import threading

import pytest
import torch

from qwenforge_b200 import ops
from tests.test_verify_drafts_gpu import Case

pytestmark = pytest.mark.gpu


def prepare(case):
    """The call as a function that leaves its outputs in case.accepted and case.tokens."""
    case.want()
    args = [None if t is None else t.cuda() for t in (case.target, case.draft, case.drafted, case.first, case.uniforms)]
    ids, steps = case.seq_ids.cuda(), case.steps.cuda()
    case.accepted, case.tokens = torch.zeros(case.n, dtype=torch.int32, device="cuda"), torch.zeros((case.n, case.most + 1), dtype=torch.int32, device="cuda")
    return lambda scratch=None: ops.verify_drafts(*args, case.temperature, case.seed, ids, steps, case.accepted, case.tokens, scratch)


def check(cases):
    torch.cuda.synchronize()
    for case in cases:
        assert (case.accepted.tolist(), case.tokens.tolist()) == case.want()


def batches():
    return [Case([5, 0, 3, 7] * 6, 60000, 0.9, seed=30), Case([2] * 9, 90001, 0.7, with_draft=False, seed=31), Case([4, 1], 30000, 1.0, seed=32)]


def test_streams_at_once():
    cases = batches()
    calls, streams = [prepare(c) for c in cases], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for turn in range(8):
        for k in range(len(cases)):
            call, stream = calls[(k + turn) % 3], streams[(k + turn) % 3]
            with torch.cuda.stream(stream):
                for _ in range(4):
                    call()
        check(cases)


def test_threads_on_one_stream():
    cases = batches()
    calls = [prepare(c) for c in cases]
    torch.cuda.synchronize()
    threads = [threading.Thread(target=lambda call=call: [call() for _ in range(40)]) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    check(cases)


def test_a_capture_wants_a_scratch_of_its_own():
    case = Case([3, 1], 20000, 0.9, seed=33)
    call, scratch = prepare(case), ops.VerifyScratch()
    call(scratch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ops.KernelError, match="scratch"):
            call()
        call(scratch)
    case.accepted.zero_()
    graph.replay()
    check([case])
