"""The workspaces of `ops.verify_drafts` that callers who bring none share: never those of another stream, device or thread."""
import threading

from qwenforge_b200.ops import branches


def test_one_per_thread_device_and_stream():
    held = branches._StreamScratches()
    a, b, c = held.get(0, 0), held.get(0, 12345), held.get(1, 0)
    assert a is not b and a is not c and b is not c
    assert held.get(0, 0) is a and held.get(0, 12345) is b and held.get(1, 0) is c
    theirs = []
    thread = threading.Thread(target=lambda: theirs.append(held.get(0, 0)))
    thread.start()
    thread.join()
    assert theirs[0] is not a and held.get(0, 0) is a


def test_no_more_than_there_is_room_for():
    held = branches._StreamScratches()
    for stream in range(3 * held.MOST):
        held.get(0, stream)
        assert len(held.held) <= held.MOST
    last = held.get(0, 3 * held.MOST - 1)
    assert last is held.get(0, 3 * held.MOST - 1)
