"""The 8-bit KV cache's entry points on the host: what they refuse, and the plain forms that their tests compare with.

No kernel runs (fake_hip.py).
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import kv8_reference as ref
from tests.fake_hip import fake_hip  # noqa: F401  (fixture)

CALLS = '''
def batch(**changed):
    given = dict(requests=3, tokens=8, max_rows=4, block=16, blocks=10, width=4)
    names = ("cached", "fresh", "free_blocks", "free_count", "free_left", "table", "lengths", "starts", "rows", "positions", "slots")
    return rt.KvBatch(**{**given, **{k: buffer.ptr for k in names}, **changed})
def cache(**changed):
    given = dict(keys=buffer.ptr, values=buffer.ptr, key_scales=buffer.ptr, value_scales=buffer.ptr, kv_heads=2, dim=64, format=0)
    return rt.Kv8(**{**given, **changed})
def status(code): return [code, lib.lh_last_error().decode(), len(kernels())]
def assign(b): return status(lib.lh_kv_assign(C.byref(b) if b else None, None))
def rope(b=None, c=None, qkv=0, heads=4, rotary=64, cos=0, sin=0, positions=100, q=0):
    b, c = b or batch(), c or cache()
    return status(lib.lh_rope_kv8(C.byref(b), C.byref(c), buffer.ptr + qkv, heads, rotary, cos and (buffer.ptr + cos - 1),
                                  sin and (buffer.ptr + sin - 1), positions, buffer.ptr + q, None))
def attend(b=None, c=None, q=0, heads=4, window=0, out=0, workspace=None, bytes=0, stream=None):
    b, c = b or batch(), c or cache()
    return status(lib.lh_attention_kv8(C.byref(b), C.byref(c), buffer.ptr + q, heads, window, buffer.ptr + out, workspace, bytes, stream))
'''


def refused(fake_hip, calls):
    results = fake_hip(CALLS + "result = [" + ", ".join(calls) + "]")
    for (code, message, launched), call in zip(results, calls):
        assert code == 1 and message.startswith("Leaf decoder: ") and launched == 0, (call, code, message)


BATCHES = ["width=2**20, block=128, blocks=4, requests=1, tokens=2**31", "width=2**24, block=128, blocks=4, requests=1", "requests=0", "requests=4001", "tokens=0", "tokens=2**31", "max_rows=0", "block=0", "block=8", "block=48",
           "block=256", "blocks=0", "blocks=2**28", "width=0", "width=2**31"]
CACHES = ["kv_heads=0", "kv_heads=257", "kv_heads=65536", "dim=0", "dim=8", "dim=72", "dim=272", "format=2", "keys=None", "values=None",
          "key_scales=None", "value_scales=None", "keys=buffer.ptr + 8", "values=buffer.ptr + 4"]


def test_refused_batches_and_caches(fake_hip):  # noqa: F811
    refused(fake_hip, ["assign(None)"] + [f"assign(batch({b}))" for b in BATCHES] +
            [f"attend(batch({b}))" for b in BATCHES] + [f"rope(batch({b}), cos=1, sin=1)" for b in BATCHES] +
            [f"attend(c=cache({c}))" for c in CACHES] + [f"rope(c=cache({c}), cos=1, sin=1)" for c in CACHES])


def test_refused_arguments(fake_hip):  # noqa: F811
    names = ("cached", "fresh", "free_blocks", "free_count", "free_left", "table", "lengths", "starts", "rows", "positions", "slots")
    refused(fake_hip, [f"assign(batch({n}=None))" for n in names] +
            [f"attend(batch({n}=None))" for n in ("table", "lengths", "starts", "rows")] +
            [f"rope(batch({n}=None), cos=1, sin=1)" for n in ("positions", "slots")] +
            ["attend(heads=0)", "attend(heads=3)", "attend(q=4)", "attend(out=8)", "attend(q=-buffer.ptr)", "attend(out=-buffer.ptr)",
             "attend(batch(tokens=2**20), heads=4096)", "attend(batch(tokens=2**20), heads=130)", "rope(batch(tokens=2**20), heads=130, cos=1, sin=1)", "attend(workspace=buffer.ptr + 8, bytes=1 << 20)",
             "rope(heads=0, cos=1, sin=1)", "rope(heads=5, cos=1, sin=1)", "rope(cos=1)", "rope(sin=1)", "rope(rotary=3, cos=1, sin=1)",
             "rope(rotary=66, cos=1, sin=1)", "rope(positions=0, cos=1, sin=1)", "rope(positions=2**31, cos=1, sin=1)",
             "rope(qkv=4, cos=1, sin=1)", "rope(q=4, cos=1, sin=1)", "rope(cos=5, sin=1)", "rope(cos=1, sin=9)",
             "rope(qkv=-buffer.ptr, cos=1, sin=1)", "rope(q=-buffer.ptr, cos=1, sin=1)"])


def test_accepted_calls(fake_hip):  # noqa: F811
    results = fake_hip(CALLS + '''
result = [assign(batch()), rope(cos=1, sin=1), rope(rotary=0), attend(), attend(window=2**32 - 1), attend(c=cache(dim=256, format=1)),
          assign(batch(requests=4000, tokens=2**31 - 1)), attend(batch(requests=4000, tokens=2**20))]
''')
    assert all(code == 0 and launched >= 1 for code, _, launched in results), results


@pytest.mark.parametrize("sizes,heads,kernels", [
    ("requests=64, tokens=64, max_rows=1, width=64", 4, ["few_kernel", "few_merge"]),          # a decode step
    ("requests=64, tokens=64, max_rows=1, width=8", 4, ["few_kernel"]),                        # too short to be parted
    ("requests=1, tokens=300, max_rows=300, width=64", 4, ["rows_kernel", "rows_merge"]),      # a prompt
    ("requests=1, tokens=300, max_rows=300, width=20", 4, ["rows_kernel"]),
    ("requests=51, tokens=300, max_rows=200, width=64", 4, ["few_kernel", "rows_kernel", "few_merge", "rows_merge"]),
    ("requests=50, tokens=300, max_rows=200, width=64", 4, ["rows_kernel", "rows_merge"]),     # six new tokens a request
    ("requests=5, tokens=20, max_rows=8, width=64", 4, ["few_kernel", "few_merge"]),           # 16 rows of a KV head
    ("requests=5, tokens=20, max_rows=9, width=64", 4, ["few_kernel", "rows_kernel", "few_merge", "rows_merge"]),
    ("requests=64, tokens=64, max_rows=1, width=64", 34, ["rows_kernel", "rows_merge"])])      # groups of 17
def test_attention_routes(fake_hip, sizes, heads, kernels):  # noqa: F811
    launched = fake_hip(CALLS + f"""
code = lib.lh_attention_kv8(C.byref(batch({sizes})), C.byref(cache()), buffer.ptr, {heads}, 0, buffer.ptr, None, 0, None)
result = [code, kernels()]
""")
    assert launched[0] == 0 and len(launched[1]) == len(kernels)
    assert all(f"attention_kv8_{name}" in k for name, k in zip(kernels, launched[1])), launched


def test_assign_routes(fake_hip):  # noqa: F811
    small, large, many = fake_hip(CALLS + """
result = []
for changed in (dict(max_rows=4), dict(max_rows=5), dict(tokens=2049, max_rows=1)):
    assert lib.lh_kv_assign(C.byref(batch(**changed)), None) == 0
    result.append(kernels())
""")
    assert [len(k) for k in (small, large, many)] == [1, 1, 2]
    assert "ILb1ELb0ELb1E" in small[0] and "ILb1ELb0ELb0E" in large[0] and "ILb0ELb1ELb0E" in many[1]


def test_workspace_does_not_depend_on_lengths(fake_hip):  # noqa: F811
    # a decode step's parts are bounded by the GPU's size, not by the table's width
    sizes, error = fake_hip(CALLS + """
n, result = C.c_size_t(), []
for width in (64, 4096, 2**20):
    assert lib.lh_attention_kv8_workspace(C.byref(batch(requests=64, tokens=64, max_rows=1, width=width)), C.byref(cache(keys=None, values=None)), 8, C.byref(n)) == 0
    result.append(n.value)
result = [result, lib.lh_attention_kv8_workspace(C.byref(batch()), C.byref(cache()), 8, None)]
""")
    assert sizes[1] == sizes[2] <= 16 << 20 and sizes[0] <= sizes[1] and error == 1


# ---- the plain forms themselves
def test_e4m3_codes():
    values = ref.E4M3_VALUES
    assert values[0x7E] == 448 and values[1] == 2.0 ** -9 and values[0x08] == 2.0 ** -6 and np.isnan(values[0x7F])
    codes = np.array([c for c in range(256) if (c & 127) != 127], np.uint8)
    assert np.array_equal(ref.encode(values[codes], ref.E4M3), codes)
    # halfway between neighbours: the even code
    low, high = values[:126], values[1:127]
    assert np.array_equal(ref.encode((low + high) / 2, ref.E4M3) & 1, np.zeros(126))


def test_append_grows_a_scale():
    codes, scales = np.zeros((1, 1, 16, 16), np.uint8), np.zeros((1, 1), np.float32)
    x = np.zeros((2, 1, 16), np.float32)
    x[0, 0, :2], x[1, 0, 0] = (1.0, -0.5), 2.0
    ref.append(codes, scales, x[:1], np.array([0]), 16, ref.INT8, False)
    assert scales[0, 0] == np.float32(1 / 127) and list(codes[0, 0, 0, :2].view(np.int8)) == [127, -64]
    ref.append(codes, scales, x[1:], np.array([1]), 16, ref.INT8, False)
    # 127 / 2 and -64 / 2 to the nearest, ties to even
    assert scales[0, 0] == np.float32(2 / 127) and list(codes[0, 0, 0, :2].view(np.int8)) == [64, -32]
    assert codes[0, 0, 1, 0] == 127


def test_assign_turns_away_what_does_not_fit():
    table = np.full((4, 3), -1)
    table[0, :2], table[2, 0] = (5, 6), 7
    plan = ref.assign([17, 0, 16, 3], [-1, 20, 1, 40], table, np.array([1, 2, 0, 0, 0, 0, 0, 0]), 2, 16, 3, 8, 70, 50)
    assert list(plan["rows"]) == [0, 20, 1, 0] and list(plan["lengths"]) == [0, 20, 17, 3]
    assert list(plan["table"][1, :2]) == [6, 5] and plan["table"][2, 1] == 2 and plan["free_left"] == [1]
    assert list(plan["free_blocks"][:4]) == [1, 2, 5, 6] and plan["slots"][20] == 2 * 16
    assert (plan["slots"][21:] == -1).all()


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
def test_attention_form_sees_a_planted_mistake(form):
    # a scale taken from the neighbouring block moves the result far past any tolerance used here
    rng = np.random.default_rng(form)
    keys, values = (ref.encode(40 * rng.standard_normal(s), form) for s in ((3, 1, 16, 16), (3, 1, 16, 16)))
    ks, vs = (np.float32(2.0) ** rng.integers(-8, -4, (3, 1)).astype(np.float32) for _ in range(2))
    ks[1], ks[2] = ks[0] * 2, ks[0] * 4
    q, table = rng.standard_normal((2, 1, 16)).astype(np.float32), np.array([[0, 1, 2]])
    out = [np.zeros((1, 2, 16)) for _ in range(2)]
    for o, scales in zip(out, (ks, ks[[1, 0, 2]])):
        ref.attention(q, keys, values, scales, vs, table, [40], [0, 1], [1], 16, form, 0, o)
    assert np.abs(out[0] - out[1]).max() > 1e-2


def test_pool_waits_for_its_stream(fake_hip):
    # a step's new tokens are not overwritten before the last step's kernels have read them; none fills on another stream
    assert fake_hip("""
calls = []
class Spy:
    def __getattr__(self, name):
        if name.startswith("lh_") and name not in ("lh_device_alloc", "lh_device_free"): calls.append(name)
        return getattr(lib, name)
spy = Spy()
rt.library = lambda: spy
pool, stream = rt.BlockPool(3, 8, 16, 10, 4), rt.Stream()
made = sorted(set(calls))
del calls[:]
pool.step([1, 1, 1], stream.handle)
on_stream = calls[:]
del calls[:]
pool.step([1, -1, 1])
result = [made, on_stream, calls[:]]
""") == [["lh_copy_to_device", "lh_stream_create"], ["lh_stream_synchronize", "lh_copy_to_device", "lh_kv_assign"],
        ["lh_copy_to_device", "lh_kv_assign"]]
