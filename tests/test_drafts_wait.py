"""LEAF_VERIFY_WAIT, after how many cycles verification computes what another workgroup owes: read once, and bounded.

On the host the value is taken from the arguments of a launch (native/launch_arguments.cpp); on the GPU a process that
starts with the switch at 0 has to find what the plain form finds.
"""
from __future__ import annotations

import json
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from tests import fake_hip

ROOT = Path(__file__).resolve().parents[1]
DEFAULT = 200000

# a call that is one launch of (call, how), how = (segments, size, ahead, wait); the switch is changed between two calls
WAITS = '''
import ctypes as C, os, struct, sys
spy = C.CDLL(sys.argv[2], mode=C.RTLD_GLOBAL)
''' + fake_hip.PRELUDE + '''
C.c_void_p.in_dll(spy, "next").value = C.cast(fake.hipLaunchKernel, C.c_void_p).value
C.c_size_t.in_dll(spy, "second_argument_bytes").value = 24
names = ("logits", "ids", "parents", "temperatures", "accept", "sample", "path", "kept", "next")
batch = rt.KvBatch(requests=300, tokens=600, max_rows=512, block=16, blocks=1, width=1, starts=buffer.ptr, rows=buffer.ptr)

def wait():
    rt.verify_drafts(batch, rt.Drafts(vocab=2000, **{n: buffer.ptr for n in names}))
    assert ["verify_kernel" in k for k in kernels()] == [True]
    segments, size, ahead, cycles = struct.unpack("ii?7xq", bytes((C.c_char * 24).in_dll(spy, "second_argument")))
    assert (segments, size, ahead) == (1, 2000, False)
    return cycles
first = wait()
os.environ["LEAF_VERIFY_WAIT"] = "77"
print("RESULT " + json.dumps([first, wait()]))
'''


@pytest.fixture(scope="module")
def libraries(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ is not installed")
    from leaf_amd import runtime
    if not runtime.LIBRARY.exists():
        pytest.skip("libleafhip.so is not built")
    made = [tmp_path_factory.mktemp("waits") / f"lib{name}.so" for name in ("fake_hip", "launch_arguments")]
    for library in made:
        subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", str(ROOT / "tests" / "native" / (library.stem[3:] + ".cpp")),
                        "-o", str(library), "-lpthread"], check=True)
    return list(map(str, made))


# the default is also the longest: a wait without end would leave workgroups waiting for one that cannot start
@pytest.mark.parametrize("given,expected", [(None, DEFAULT), ("0", 0), ("1500", 1500), ("-3", 0), (str(10 ** 18), DEFAULT), ("9" * 30, DEFAULT),
                                            ("soon", DEFAULT), ("", DEFAULT)])
def test_the_switch_is_read_once_and_bounded(libraries, given, expected):
    environment = {k: v for k, v in os.environ.items() if k != "LEAF_VERIFY_WAIT"}
    if given is not None:
        environment["LEAF_VERIFY_WAIT"] = given
    done = subprocess.run([sys.executable, "-c", WAITS, *libraries], cwd=ROOT, env=environment, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr
    assert json.loads(done.stdout.rsplit("RESULT ", 1)[1]) == [expected, expected]


NO_WAIT = '''
import numpy as np
from leaf_amd import runtime as rt
from tests.test_gpu_drafts import check_verify, draft_case
for vocab in (5000, 32000, 50257):
    for with_draft in (False, True):
        rng = np.random.default_rng(vocab)
        for counts in ([6], [8] * 40):
            check_verify(rt, draft_case(rng, counts, vocab, 3, with_draft, np.where(np.arange(len(counts)) % 5 == 4, 0.0, 0.9), padding=1))
            print("checked", vocab, with_draft, len(counts), flush=True)
'''


@pytest.mark.gpu
def test_a_process_that_never_waits():
    # a workgroup that waits for no other computes all that they owe it, to the same results
    done = subprocess.run([sys.executable, "-c", NO_WAIT], cwd=ROOT, env={**os.environ, "LEAF_VERIFY_WAIT": "0"}, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout + done.stderr
    assert done.stdout.count("checked") == 12
