"""Calls of several threads on the per-thread default stream (hipStreamPerThread), whose launches overlap on the GPU.

Calls of more than one launch keep something between them in scratch, which is each thread's own there: every result
has the bits that a call alone gives.
"""
from __future__ import annotations

import threading

import numpy as np
import pytest

from leaf_amd.artifact import quantize
from tests import kv8_reference as ref
from tests import test_gpu_kv8 as kv8

pytestmark = pytest.mark.gpu
PER_THREAD = 2                                      # hipStreamPerThread


@pytest.fixture(scope="module")
def rt():
    from leaf_amd import runtime
    runtime.library()
    return runtime


def cache_call(rt, rng, batch):
    c = kv8.attention_case(rng, batch, 8, 2, 64, 32, ref.INT8)
    d = {k: kv8.ints(rt, c[k]) for k in ("table", "lengths", "starts", "rows")}
    data = [rt.DeviceArray.of(c[k]) for k in ("keys", "values", "key_scales", "value_scales")]
    desc = rt.KvBatch(requests=len(c["rows"]), tokens=c["q"].shape[1], max_rows=int(c["rows"].max()), block=32,
                      blocks=len(c["keys"]), width=c["table"].shape[1], **{k: v.ptr for k, v in d.items()})
    q, out = rt.DeviceArray.of(c["q"]), rt.DeviceArray((c["q"].shape[1], 8, 64), np.float32)
    cache = rt.Kv8(*(a.ptr for a in data), 2, 64, ref.INT8)
    return lambda stream: rt.attention_kv8(desc, cache, q, 8, out, stream=stream), out, (d, data)


def token_call(rt, rng, keys):
    kv = [rt.DeviceArray.of(rng.standard_normal((2, keys, 64)).astype(np.float32)) for _ in range(2)]
    q, out = rt.DeviceArray.of(rng.standard_normal((8, 1, 64)).astype(np.float32)), rt.DeviceArray((1, 8, 64), np.float32)
    lib = rt.library()
    return (lambda stream: rt.check(lib.lh_attention(q.ptr, kv[0].ptr, kv[1].ptr, keys, 8, 2, 64, 1, keys - 1, 0, out.ptr, stream)),
            out, (q, kv))


def linear_call(rt, rng, tokens):
    data, scales = quantize((0.02 * rng.standard_normal((512, 2048))).astype(np.float32), 8, 128)
    w, x = rt.DeviceWeight(data, 8, 2048, scales, 128), rt.DeviceArray.of(rng.standard_normal((tokens, 2048), dtype=np.float32))
    y = rt.DeviceArray((tokens, 512), np.float32)
    return lambda stream: rt.linear(w, x, tokens, 8, y, stream=stream), y, (w, x)


def test_threads_on_their_own_default_streams(rt):
    rng = np.random.default_rng(0)
    work = [[cache_call(rt, rng, [(3000, 1)] * 6), cache_call(rt, rng, [(2500, 1), (800, 1), (4000, 1)]), token_call(rt, rng, 4000),
             linear_call(rt, rng, 64)],
            [cache_call(rt, rng, [(1000, 1)] * 20), cache_call(rt, rng, [(3000, 70)]), token_call(rt, rng, 2500), linear_call(rt, rng, 200)],
            [linear_call(rt, rng, 30), token_call(rt, rng, 3999), cache_call(rt, rng, [(5000, 1)] * 3)]]
    want = []
    for calls in work:
        for call, _, _ in calls:
            call(None)
        rt.synchronize()
        want.append([out.numpy() for _, out, _ in calls])
    for _ in range(2):                              # the second time by new threads, with the first ones' scratch
        wrong, gate = [], threading.Barrier(len(work))

        def run(i):
            try:
                gate.wait()
                for turn in range(20):
                    for call, _, _ in work[i]:
                        call(PER_THREAD)
                    if turn % 7 == 6:
                        rt.synchronize()
                        for k, (_, out, _) in enumerate(work[i]):
                            if not np.array_equal(out.numpy().view(np.uint32), want[i][k].view(np.uint32)):
                                wrong.append((i, k, turn))
            except BaseException as e:              # (an assertion in a thread ends no test)
                wrong.append(repr(e))
        threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong
