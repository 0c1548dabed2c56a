"""Numbers that the library's argument types do not hold are refused, not cut to their low bits (fakehip.py)."""
from __future__ import annotations

from test_kv_pages import run, shim  # noqa: F401


def test_numbers_that_do_not_fit(shim):  # noqa: F811
    run(shim, """
        kv = cache()
        a = address(1 << 20)
        kv.extend([0], [3])
        rope = Rope(a, a, 10, 64, positions=a)
        more, much = 1 << 32, 1 << 64
        log()
        for call in (lambda: be.rope_into(a, a, 3, more + 4, 64, rope), lambda: be.rope_into(a, a, 3, 4, more + 64, rope),
                     lambda: be.rope_into(a, a, much + 3, 4, 64, rope), lambda: be.rope_into(a, a, 3, 4, 64, rope, x_stride=much + 256),
                     lambda: be.rope_into(a, a, 3, 4, 64, rope, out_stride=much), lambda: be.rope_into(a, a, 3, 4 - more, 64, rope),
                     lambda: Rope(a, a, 10, more + 64, positions=a), lambda: Rope(a, a, much + 10, 64, positions=a),
                     lambda: cache(pages=much + 12), lambda: cache(head_dim=more + 64),
                     lambda: kv.append(0, a, a, stride=much), lambda: kv.append(0, a, a, q_ptr=a, heads=4, q_stride=much),
                     lambda: kv.append(more, a, a), lambda: kv.append(0, a, a, q_ptr=a, heads=more + 4),
                     lambda: kv.attend(0, a, a, 2, q_stride=much, out_stride=much), lambda: kv.attend(0, a, a, more + 2),
                     lambda: kv.attend(0, a, a, 2, window=more), lambda: kv.read(0, [0], [0], much + 3, a, a), lambda: kv.read(0, [0], [much], 3, a, a)):
            assert refused(call) == "IllegalArgumentException", call.__code__.co_firstlineno
        assert not log("launch", "malloc")
        be.rope_into(a, a, np.int64(3), np.int32(4), np.int64(64), rope, x_stride=np.int64(256), out_stride=np.int32(256))
        kv.append(0, a, a, stride=np.int64(128))
        kv.attend(0, a, a, 2, q_stride=np.int32(128), out_stride=np.int64(128))
        assert len(launches()) >= 3
    """)
