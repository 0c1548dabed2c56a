"""Norms, routing and experts without a GPU (fakehip.py): what calls refuse, and what they launch, allocate and take for a workspace."""
from __future__ import annotations

from test_kv_pages import run, shim  # noqa: F401

MORE = """
        from jax4j_amd import Experts, Norm
        a = address(1 << 22)
        F, B, NONE = DType.F32, DType.BF16, "IllegalArgumentException"
        def matrices(up=QuantType.Q4_K, down=QuantType.Q6_K, experts=4, dim=256, ffn=512):
            return [zeros(up, experts * ffn, dim), zeros(up, experts * ffn, dim), zeros(down, experts * dim, ffn)]
        def quiet(calls):
            log()
            for i, (call, *words) in enumerate(calls):
                assert refused(call, *words) in ("IllegalArgumentException", "UnsupportedOperationException"), i
            assert not log("launch", "malloc"), log()
"""


def test_norm_refuses(shim):  # noqa: F811
    run(shim, MORE + """
        def norm(x=a, out=a + 65536, rows=4, dim=256, before=Norm(), **more):
            return lambda: be.norm_into(x, out, rows, dim, before, **more)
        quiet([(norm(x=0), "neither"), (norm(out=0, before=None), "neither"), (norm(out=0, residual_out_ptr=a + 131072), "together"), (norm(before=None), "together"),
               (norm(after=Norm()), "not there"), (norm(gate_ptr=a + 4096), "not there"), (norm(rows=0), "0 rows"), (norm(rows=-1), "negative"),
               (norm(rows=1 << 31),), (norm(dim=0),), (norm(dim=32769), "32768"), (norm(dim=1 << 32), "fit"), (norm(rows=1 << 64), "fit"),
               (norm(residual_stride=255), "apart"), (norm(out_stride=-1), "negative"), (norm(residual_stride=1 << 63), "fit"), (norm(x=a + 2), "aligned"),
               (norm(x=a + 1, residual_type=B), "aligned"), (norm(block_ptr=a + 131072, gate_ptr=a + 4096, gate_every=-1), "negative"),
               (norm(out=a, residual_type=B), "overlaps"), (norm(out=a + 4), "overlaps"), (norm(residual_stride=512, out=a), "overlaps"),
               (norm(out=a + 65536, residual_out_ptr=a + 65536), "overlaps"), (norm(before=Norm(a + 65536)), "overlaps"), (norm(before=Norm(a + 2)), "aligned"),
               (norm(before=Norm(eps=-1.0)), "eps"), (norm(before=Norm(eps=float("nan"))), "eps"), (lambda: Norm(kind="group"), "unknown"),
               (norm(residual_type=DType.F16),), (norm(x=a + (1 << 70)), "fit"), (lambda: Norm(1 << 64), "fit"), (norm(stream=-1), "fit")])
        norm(out=a)()
        norm(residual_out_ptr=a, block_ptr=a + 131072)()
        norm(rows=np.int64(3), dim=np.int32(256), residual_stride=np.int64(300))()
        assert len(launches()) == 3
    """)


def test_route_refuses(shim):  # noqa: F811
    run(shim, MORE + """
        def route(x=a, ids=a + 65536, weights=a + 131072, rows=4, experts=64, top=4, **more):
            return lambda: be.route_into(x, ids, weights, rows, experts, top, **more)
        quiet([(route(x=0), "NULL"), (route(ids=0), "NULL"), (route(weights=0), "NULL"), (route(rows=0),), (route(rows=-1),), (route(rows=1 << 64),),
               (route(experts=0),), (route(experts=1025), "1024"), (route(experts=1 << 32),), (route(top=0),), (route(top=65),), (route(experts=3), "3 experts"),
               (route(top=1 << 32),), (route(groups=65, experts=650), "groups"), (route(groups=5), "groups"), (route(groups=8, top_groups=9), "groups"),
               (route(groups=8, top_groups=0), "groups"), (route(groups=16, top_groups=1, top=5), "of 4"), (route(groups=8, top_groups=2, group_best=3), "best"),
               (route(stride=63), "apart"), (route(x=a + 1, dtype=B), "aligned"), (route(ids=a + 65537), "aligned"), (route(bias_ptr=a + 2), "aligned"),
               (route(ids=a), "apart"), (route(weights=a + 65536), "apart"), (route(bias_ptr=a + 65536), "apart"), (route(score="relu"), "unknown"),
               (route(x=1 << 70), "fit"), (route(stream=1 << 64), "fit")])
        route()()
        route(groups=8, top_groups=2, group_best=2, bias_ptr=a + 262144, score="sigmoid", renormalize=True, scale=2.5, dtype=B)()
        assert len(launches()) == 2
    """)


def test_experts_refuse(shim):  # noqa: F811
    run(shim, MORE + """
        gate, up, down = matrices()
        other = matrices(QuantType.Q8_0, QuantType.Q8_0)
        narrow = matrices(QuantType.Q8_0, QuantType.Q8_0, dim=96, ffn=64)
        quiet([(lambda: Experts(be, gate, up, down, experts=0),), (lambda: Experts(be, gate, up, down, experts=1025), "1024"),
               (lambda: Experts(be, gate, up, down, experts=1 << 32),), (lambda: Experts(be, gate, up, down, experts=3), "3 experts"),
               (lambda: Experts(be, gate, other[1], down, experts=4), "type"), (lambda: Experts(be, gate, down, up, experts=4),),
               (lambda: Experts(be, *narrow, experts=4), "multiple of 64"), (lambda: Experts(be, gate, up, down, experts=4, activation="tanh"), "unknown")])
        e = Experts(be, gate, up, down, experts=4)
        assert launches() and e.info()["bytes"] == 4 * (4 * 4 * 512 + 2 * 4 * 256 + 2 * 4)
        for m in (gate, up, down):
            assert refused(lambda: be.release(m), "live") == NONE
        def apply(x=a, ids=a + 262144, weights=a + 524288, out=a + 1048576, rows=4, top=2, dtype=F, **more):
            return lambda: e.apply(x, ids, weights, out, rows, top, dtype, **more)
        n = e.workspace(4, 2)
        space = (a + 2097152 + 255) // 256 * 256
        quiet([(apply(x=0), "NULL"), (apply(ids=0), "NULL"), (apply(weights=0), "NULL"), (apply(out=0), "NULL"), (apply(rows=0),), (apply(rows=-1), "negative"),
               (apply(top=0),), (apply(top=65), "64"), (apply(rows=(1 << 21) + 1), "pairs"), (apply(rows=1 << 62), "pairs"), (apply(top=1 << 32), "fit"),
               (apply(rows=1 << 64), "fit"), (apply(x_stride=255), "apart"), (apply(x_stride=257), "multiple of 16"), (apply(dtype=B, out_stride=260), "multiple of 16"),
               (apply(out_stride=1 << 63), "fit"), (apply(x=1 << 70), "fit"), (apply(stream=-1), "fit"), (apply(x_stride=1 << 41),), (apply(x=a + 4), "aligned"), (apply(out=a + 8), "aligned"), (apply(ids=a + 2), "aligned"),
               (apply(out=a), "apart"), (apply(out=a + 1024), "apart"), (apply(ids=a + 1048576), "apart"), (apply(weights=a + 1048576 + 64), "apart"),
               (apply(workspace_ptr=space, workspace_bytes=n - 1), "workspace"), (apply(workspace_ptr=space + 16, workspace_bytes=n), "workspace"),
               (apply(workspace_ptr=a // 256 * 256, workspace_bytes=n), "apart"), (apply(workspace_ptr=space, workspace_bytes=1 << 64), "fit"),
               (lambda: e.workspace(0, 2),), (lambda: e.workspace(4, 0),), (lambda: e.workspace(1 << 22, 2),), (lambda: e.workspace(1 << 63, 2),)])
        apply()()
        apply(workspace_ptr=space, workspace_bytes=n, dtype=B)()
        assert launches()
        handle = e.handle
        e.destroy()
        e.destroy()
        e.handle = handle
        quiet([(apply(), "destroyed"), (lambda: e.info(), "destroyed"), (lambda: e.workspace(4, 2), "destroyed"), (lambda: e.destroy(), "destroyed")])
        for m in (gate, up, down):
            be.release(m)
        again = Experts(be, *matrices(), experts=4)  # the slot, not the old handle
        quiet([(apply(), "destroyed")])
    """)


def test_a_call_s_launches_and_workspace(shim):  # noqa: F811
    """One row two launches, others four; calls of many rows as ranges of at most 2^17 pairs with a workspace that stops growing; nothing
    allocated once the engine's workspace is there."""
    run(shim, MORE + """
        e = Experts(be, *matrices(QuantType.Q8_0, QuantType.Q8_0, 4, 64, 64), experts=4)
        x = [1 << 40 | i << 36 for i in range(4)]  # never touched: nothing runs
        def launched(rows, top, dtype=F):
            e.apply(*x, rows, top, dtype)
            log()
            e.apply(*x, rows, top, dtype)
            calls = log("launch", "malloc")
            assert all(l.startswith("launch") for l in calls)
            return len(calls)
        assert launched(1, 4) == 2 and launched(2, 4) == 4 and launched(4096, 4, B) == 4
        assert launched(1 << 15, 4) == 4 and launched((1 << 15) + 1, 4) == 8 and launched(1 << 20, 4) == 128
        sizes = [e.workspace(rows, 4) for rows in (1, 2, 100, 1 << 15, (1 << 15) + 1, 1 << 20)]
        assert sizes[3] >= sizes[4] and sizes[5] == sizes[3], sizes
        # the last range of a call is smaller, and may be of another kind: its workspace counts too
        for rows in (32769, 40000, 65537, 98304):
            parts = -(-rows // 32768)
            low = rows // parts
            assert e.workspace(rows, 4) == max(e.workspace(low, 4), e.workspace(low + (rows % parts > 0), 4))
        wide = Experts(be, *matrices(QuantType.Q8_0, QuantType.Q8_0, 1, 32768, 64), experts=1)
        wide.apply(*x, 16384, 1)
        log()
        wide.apply(*x, 16384, 1)  # 2 GiB of x' in fp32
        assert len(launches()) == 8
    """)


def test_an_engine_stream_that_is_captured(shim):  # noqa: F811
    run(shim, MORE + """
        m = matrices()
        engine = be.stream()
        fake.fake_capture(C.c_void_p(engine), 1)
        quiet([(lambda: Experts(be, *m, experts=4), "captured")])
        fake.fake_capture(C.c_void_p(engine), 0)
        e = Experts(be, *m, experts=4)
        n = e.workspace(4, 2)
        space = (a + 2097152 + 255) // 256 * 256
        fake.fake_capture(C.c_void_p(engine), 1)
        log()
        e.apply(a, a + 262144, a + 524288, a + 1048576, 4, 2, workspace_ptr=space, workspace_bytes=n)
        lines = log("launch", "malloc", "wait", "record")
        assert [l.split()[0] for l in lines] == ["launch"] * 4, lines
        fake.fake_capture(C.c_void_p(engine), 0)
    """)


def test_a_workspace_is_of_a_call_s_own_rows(shim):  # noqa: F811
    """Where calls go from few pairs an expert to many, shares take fewer bytes: a workspace for more rows may be short for fewer, which is refused."""
    run(shim, MORE + """
        e = Experts(be, *matrices(QuantType.Q4_K, QuantType.Q6_K, 64, 256, 256), experts=64)
        sizes = {rows: e.workspace(rows, 8, B) for rows in (1, 2, 8, 100, 191, 192, 300)}
        assert sizes[192] < sizes[191], sizes
        x, ids, weights, out, space = (1 << 40 | i << 36 for i in range(5))
        def call(rows, n):
            return lambda: e.apply(x, ids, weights, out, rows, 8, B, workspace_ptr=space, workspace_bytes=n)
        quiet([(call(191, sizes[192]), "workspace")])
        for rows, n in sizes.items():
            call(rows, n)()
            call(rows, max(sizes.values()))()
            quiet([(call(rows, n - 1), "workspace")])
    """)
