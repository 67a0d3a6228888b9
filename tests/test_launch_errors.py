"""What a failed call leaves behind: on the host with a HIP runtime whose allocations can fail (fake_hip.py)."""
from __future__ import annotations

import pytest

from tests.fake_hip import fake_hip  # noqa: F401  (fixture)

FAIL = {
    "allocation": "lib.lh_device_alloc(1 << 20, C.byref(C.c_void_p()))",
    "scratch of one-token attention": "attention(1, 4000)",
    "scratch of an integer linear": "lib.lh_linear(C.byref(weight(8, 256, 2048, 128)), buffer.ptr, 64, 8, buffer.ptr, None, None)",
}


@pytest.mark.parametrize("failed", FAIL)
def test_an_error_is_reported_once(fake_hip, failed):  # noqa: F811
    # HIP keeps the last error until it is asked for: the next call's launch is not to find it
    statuses = fake_hip(f"""
        fake.fake_set_malloc_limit(0)
        statuses = [{FAIL[failed]}]
        statuses.append(lib.lh_silu_gate(buffer.ptr, 4, 64, buffer.ptr, None))
        fake.fake_set_malloc_limit(1 << 40)
        statuses.append({FAIL[failed]})
        result = statuses
    """)
    assert statuses == [4, 0, 0]
