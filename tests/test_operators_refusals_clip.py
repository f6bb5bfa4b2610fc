"""Buffers that a call of the gradient clipping may not share, on the C entry point itself: refused
on a queue that has nothing but an error callback, before anything is launched."""
import pytest

from test_operators_refusals import F16, F32, P, Q, FakeQueue, clip

SHARED = [
    ("tensor 1: two outputs are one buffer", [(Q[0], P, 4, F32), (Q[1], P, 4, F32)]),
    ("tensor 2: two outputs are one buffer", [(P, P, 4, F32), (Q[1], Q[2], 4, F16), (P, P, 4, F32)]),  # twice in place
    ("tensor 1: an output is another tensor's input", [(Q[0], Q[1], 4, F32), (Q[1], Q[2], 4, F32)]),
    ("tensor 0: an output is another tensor's input", [(Q[2], Q[0], 4, F32), (Q[1], Q[2], 4, F32)]),
    ("tensor 1: the norm is a tensor's buffer", [(Q[0], Q[1], 4, F32), (Q[2], P + 4096, 1, F32)]),
    ("tensor 0: the norm is a tensor's buffer", [(P + 4096, Q[1], 1, F32)]),
]


@pytest.mark.parametrize("k", range(len(SHARED)))
def test_shared_buffers_are_refused(k):
    match, table = SHARED[k]
    q = FakeQueue()
    assert clip(q.ptr, table=table, n=len(table), norm_=P + 4096, work=P + (1 << 16)) == 1
    assert len(q.messages) == 1 and match in q.messages[0], q.messages


def test_the_last_of_many_tensors():
    q = FakeQueue()
    table = [(P + (k << 12), P + (k << 12), 4, F32) for k in range(1000)]
    table.append((P + (1 << 30), P + (7 << 12), 4, F32))
    assert clip(q.ptr, table=table, n=len(table), norm_=P - 4096, work=P - (1 << 16)) == 1
    assert len(q.messages) == 1 and "tensor 1000: two outputs" in q.messages[0], q.messages
