"""Host checks of the serving step's limits, without a GPU: token counts that a launch does not take, rows that share memory."""
import ctypes
import random

from mlc_decode_amd import _lib
from mlc_decode_amd.serving import _apart_or_same, _rows_meet
from test_serving import BASE, cache_desc, lib, rope_desc  # noqa: F401


def test_more_tokens_than_a_launch_takes_are_refused(lib):
    """Up to the largest counts an int32 holds; the limits are those of the header."""
    c, r = cache_desc(), rope_desc()
    for tokens in ((1 << 26) - 3, 1 << 30, 2 ** 31 - 1):
        assert lib.mla_kv_gather(ctypes.byref(c), BASE, tokens, BASE, 576, None) == 4 and b"too many tokens" in lib.mla_last_error()
    a = _lib.MlaAppendSlotsArgs()
    a.kv_new, a.new_stride, a.slots = BASE, 576, BASE
    for a.tokens in ((1 << 27) - 7, 1 << 30, 2 ** 31 - 1):
        assert lib.mla_kv_append_slots(ctypes.byref(c), None, ctypes.byref(a), None) == 4 and b"too many tokens" in lib.mla_last_error()
    a = _lib.MlaRopeArgs()
    a.x, a.out, a.positions, a.heads, a.dim = BASE, 2 * BASE, BASE, 1, 1024
    for r.dim, per in ((64, 8), (128, 8), (256, 4), (1024, 1)):
        for a.tokens in (((1 << 24) - 1) * per + 1, 2 ** 31 - 1):
            assert lib.mla_apply_rope(ctypes.byref(r), ctypes.byref(a), None) == 4 and b"too many tokens" in lib.mla_last_error()


def test_rows_meet_as_counted_out():
    """Against every pair of rows: nested and interleaved strides, broadcast ones, single rows, shifts."""
    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        counts = rng.randint(1, 5), rng.randint(1, 5)
        strides = tuple(rng.choice((0, rng.randint(1, 12), 4 * rng.randint(1, 12), 20 * rng.randint(1, 4))) for _ in range(2))
        width, shift = rng.randint(1, 12), rng.choice((0, rng.randint(-60, 60)))
        at = [t * strides[0] + h * strides[1] for t in range(counts[0]) for h in range(counts[1])]
        want = any(abs(b + shift - a) < width for i, a in enumerate(at) for j, b in enumerate(at) if shift or i != j)
        assert _rows_meet(strides, counts, width, shift) == want, (strides, counts, width, shift)
        seen[want] += 1
    assert min(seen.values()) > 500
    assert _rows_meet((64, 64), (2, 2), 64) and not _rows_meet((150, 100), (2, 2), 50)
    # heads every 300, tokens every 1000: the fourth head and the next token are 100 apart
    assert not _apart_or_same(0, (1000, 300), 2 * 64, (1000, 300), (2, 4), 64, 2)
