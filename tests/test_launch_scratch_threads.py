"""Scratch on the per-thread default stream: one handle (2) for a stream of each thread.

Threads' calls there run side by side, so each thread has memory of its own.  On the host (fake_hip.py): whether a
call allocates is seen by letting allocations fail.
"""
from __future__ import annotations

import pytest

from tests.fake_hip import fake_hip  # noqa: F401  (fixture)

CALLS = {
    "one-token attention": "attention(1, 4000, stream=STREAM)",
    "integer linear": "lib.lh_linear(C.byref(weight(8, 256, 2048, 128)), buffer.ptr, 64, 8, buffer.ptr, None, STREAM)",
    "8-bit cache attention": "lib.lh_attention_kv8(C.byref(batch), C.byref(cache), buffer.ptr, 4, 0, buffer.ptr, None, 0, STREAM)",
}
SETUP = """
import time
batch = rt.KvBatch(requests=3, tokens=8, max_rows=4, block=16, blocks=10, width=64, **{k: buffer.ptr for k in
                   ("table", "lengths", "starts", "rows")})
cache = rt.Kv8(buffer.ptr, buffer.ptr, buffer.ptr, buffer.ptr, 2, 64, 0)
STREAM = 2
def allowed(): fake.fake_set_malloc_limit(1 << 40)
def refused(): fake.fake_set_malloc_limit(0)
class Worker:                                       # a thread that calls when it is told to
    def __init__(self, call):
        self.call, self.go, self.done, self.out = call, threading.Semaphore(0), threading.Semaphore(0), []
        self.thread = threading.Thread(target=self.run)
        self.thread.start()
    def run(self):
        while True:
            self.go.acquire()
            if self.call is None: return
            self.out.append(self.call())
            self.done.release()
    def __call__(self):
        self.go.release()
        self.done.acquire()
        return self.out[-1]
    def end(self):
        self.call = None
        self.go.release()
        self.thread.join()
"""


@pytest.mark.parametrize("call", CALLS)
def test_threads_have_scratch_of_their_own(fake_hip, call):  # noqa: F811
    first, other, again, shared = fake_hip(SETUP + f"""
call = lambda: {CALLS[call]}
a, b = Worker(call), Worker(call)
allowed()
first = a()
refused()
other, again = b(), a()                             # b needs memory, a has it
allowed()
first = [first, b()]
refused()
again = [again, a(), b()]
# any other stream's scratch belongs to the stream, whichever thread calls
stream = rt.Stream()
STREAM = stream.handle
allowed()
shared = [a()]
refused()
shared += [b(), a()]
a.end(); b.end()
result = first, other, again, shared
""")
    assert first == [0, 0] and again == [0, 0, 0] and shared == [0, 0, 0]
    assert other != 0


@pytest.mark.parametrize("call", CALLS)
def test_ended_threads_leave_their_scratch_to_new_ones(fake_hip, call):  # noqa: F811
    # a program that makes a thread per request does not grow
    one, later = fake_hip(SETUP + f"""
call = lambda: {CALLS[call]}
allowed()
a = Worker(call)
one = a()
a.end()
refused()
later = []
for _ in range(5):
    for attempt in range(100):                      # (the thread's end is a little later than its join)
        b = Worker(call)
        status = b()
        b.end()
        if status == 0: break
        time.sleep(0.02)
    later.append(status)
result = one, later
""")
    assert one == 0 and later == [0] * 5


def test_captured_scratch_is_not_handed_on(fake_hip):  # noqa: F811
    # a graph may hold it after its thread's end
    statuses = fake_hip(SETUP + f"""
call = lambda: {CALLS["8-bit cache attention"]}
allowed()
a = Worker(call)
statuses = [a()]
fake.fake_set_capturing(1)
statuses.append(a())
fake.fake_set_capturing(0)
a.end()
time.sleep(0.2)
refused()
b = Worker(call)
statuses.append(b())
b.end()
allowed()
result = statuses
""")
    assert statuses[:2] == [0, 0] and statuses[2] != 0


def test_first_call_of_a_thread_in_a_capture_is_refused(fake_hip):  # noqa: F811
    statuses = fake_hip(SETUP + f"""
call = lambda: {CALLS["8-bit cache attention"]}
allowed()
a, b = Worker(call), Worker(call)
statuses = [a()]
fake.fake_set_capturing(1)
statuses += [b(), a()]
fake.fake_set_capturing(0)
statuses.append(b())
a.end(); b.end()
result = statuses
""")
    assert [s == 0 for s in statuses] == [True, False, True, True]


def test_per_thread_stream_is_not_destroyed(fake_hip):  # noqa: F811
    # its handle stands for other threads' streams too, whose scratch may be in use
    assert fake_hip("result = [lib.lh_stream_destroy(2), lib.lh_last_error().decode()]") == \
        [1, "Leaf decoder: only a created stream can be destroyed"]
