"""The order of calls on one key/value cache over the streams that they come on, without a GPU (fakehip.py)."""
from __future__ import annotations

import subprocess

import pytest

import fakehip
from test_kv_pages import run, shim  # noqa: F401


@pytest.mark.parametrize("handle", [1, 2, 0x70], ids=["hipStreamLegacy", "hipStreamPerThread", "a stream's"])
def test_an_equal_handle_may_be_another_stream(shim, handle):  # noqa: F811
    """A thread's own stream has the same handle in every thread, a new stream may have that of one destroyed: a call waits for the
    call before it, unless that one is done."""
    run(shim, f"""
        kv = cache(pages=60, sequences=4, sequence_pages=60)
        a = address(1 << 20)
        kv.extend([0], [20], stream={handle})
        def waits(call):
            lines = log()
            call()
            return [l.split()[0] for l in log() if l.split()[0] in ("wait", "record", "launch")]
        calls = (lambda s: kv.append(0, a, a, stream=s), lambda s: kv.attend(0, a, a + 65536, 2, stream=s), lambda s: kv.read(0, [0], [0], 4, a, a, stream=s),
                 lambda s: kv.begin([0], [1], stream=s), lambda s: kv.fork([0], [1], stream=s), lambda s: kv.extend([0], [1], stream=s))
        for call in calls:
            for done in (0, 1):
                kv.truncate([1], [0])
                fake.fake_events_done(done)
                got = waits(lambda: call({handle}))
                assert got[:2] == (["launch"] if done else ["wait", "launch"])[:len(got)] and "record" not in got, got
        fake.fake_events_done(0)
        # the engine's own is one stream: nothing there, and what leaves it or comes to it waits
        got = [waits(lambda: kv.attend(0, a, a + 65536, 2, stream=s)) for s in (0, 0, {handle}, 0)]
        assert got == [["wait", "launch"], ["launch"], ["record", "wait", "launch"], ["wait", "launch"]], got
    """)


def test_no_event_goes_into_a_graph_of_the_engine_stream(shim):  # noqa: F811
    """The last call is on the engine stream, which is captured now: a call on another stream could only wait for an event of the
    graph, and would become part of it. It is refused before it changes anything, and goes through after the capture."""
    run(shim, """
        kv = cache(pages=60, sequences=4, sequence_pages=60)
        a = address(1 << 20)
        kv.extend([0, 3], [20, 40])
        kv.append(0, a, a)
        kv.truncate([3], [0])
        kv.extend([0], [30])
        engine = be.stream()
        calls = [lambda: kv.append(0, a, a, stream=0x70), lambda: kv.attend(0, a, a + 65536, 2, stream=0x70),
                 lambda: kv.read(0, [0], [0], 4, a, a, stream=0x70), lambda: kv.begin([0], [1], stream=0x70), lambda: kv.fork([0], [1], stream=0x70),
                 lambda: kv.extend([0], [1], stream=0x70), lambda: kv.compact(stream=0x70), lambda: kv.evict([0], 4, stream=0x70)]
        state = lambda: (kv.info(), kv.tables(range(4)).tolist(), kv.lengths(range(4)).tolist())
        for call in calls:
            kv.attend(0, a, a + 65536, 2)
            was = state()
            log()
            fake.fake_capture(C.c_void_p(engine), 1)
            assert refused(call, "engine stream", "captured") == "IllegalArgumentException"
            assert state() == was and not log("record", "wait", "launch")
            kv.attend(0, a, a + 65536, 2)  # into the graph
            assert launches()
            fake.fake_capture(C.c_void_p(engine), 0)
            call()
            lines = [l.split()[0] for l in log("record", "wait", "launch")]
            assert lines[:3] == ["record", "wait", "launch"] or not lines, lines
    """)


def changed_shim(folder, function, line, switch):
    """The same runtime, in one of whose functions this line comes first while fake_<switch>(1) holds."""
    text = (fakehip.TESTS / "fake_hip.cpp").read_text()
    head = f"F hipError_t {function}("
    at = text.index("LOCK;", text.index(head)) + len("LOCK;")
    text = text[:at] + f" if ({switch}) {{ {line} }}" + text[at:]
    at = text.index(head)
    text = text[:at] + f"static bool {switch} = false;\nF void fake_{switch}(int on) {{ {switch} = on != 0; }}\n" + text[at:]
    (folder / "fake_hip.cpp").write_text(text)
    lib = folder / "fake_hip.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", f"-I{fakehip.ROCM / 'include'}",
                    "-o", str(lib), str(folder / "fake_hip.cpp")], check=True)
    return lib


@pytest.fixture(scope="module")
def unsure_shim(tmp_path_factory):
    """It does not tell whether stream 0x70 is captured (as of hipStreamLegacy beside another's capture)."""
    return changed_shim(tmp_path_factory.mktemp("unsure_hip"), "hipStreamIsCapturing",
                        "if (s == (hipStream_t)0x70) return ret(hipErrorStreamCaptureImplicit);", "unsure")


def test_a_stream_that_may_be_captured_or_not(unsure_shim):
    """Neither kind of call would be right there: one without a wait would race, one with an event be part of a graph."""
    run(unsure_shim, """
        kv = cache(pages=60, sequences=4, sequence_pages=60)
        a = address(1 << 20)
        kv.extend([0], [20], stream=0x60)
        state = lambda: (kv.info(), kv.tables(range(4)).tolist(), kv.lengths(range(4)).tolist())
        for call in (lambda: kv.append(0, a, a, stream=0x70), lambda: kv.attend(0, a, a + 65536, 2, stream=0x70),
                     lambda: kv.read(0, [0], [0], 4, a, a, stream=0x70), lambda: kv.begin([0], [1], stream=0x70), lambda: kv.fork([0], [1], stream=0x70),
                     lambda: kv.extend([0], [1], stream=0x70), lambda: kv.compact(stream=0x70), lambda: kv.evict([0], 4, stream=0x70)):
            was = state()
            log()
            fake.fake_unsure(1)
            assert refused(call, "failed") == "RuntimeError"
            assert state() == was and not log("record", "wait", "launch")
            fake.fake_unsure(0)
            call()
    """)


@pytest.fixture(scope="module")
def no_wait_shim(tmp_path_factory):
    return changed_shim(tmp_path_factory.mktemp("no_wait_hip"), "hipStreamWaitEvent", "return ret(hipErrorInvalidHandle);", "no_wait")


def test_a_call_that_could_not_wait_is_not_waited_for(no_wait_shim):
    """Its stream is not behind the call before it: that one stays what the next call waits for."""
    run(no_wait_shim, """
        kv = cache(pages=60, sequences=4, sequence_pages=60)
        a = address(1 << 20)
        fake.fake_events_done(0)
        for first in (0x60, 0):
            for failing in (0x70, 0):
                if failing == first:
                    continue
                kv.extend([0], [5], stream=first)
                log()
                fake.fake_no_wait(1)
                assert refused(lambda: kv.attend(0, a, a + 65536, 2, stream=failing), "failed") == "RuntimeError"
                fake.fake_no_wait(0)
                assert [l.split()[-1] for l in log("record", "launch")] == ([hex(be.stream())] if first == 0 else [])
                kv.attend(0, a, a + 65536, 2, stream=first)
                assert bool(log("wait")) == (first != 0)
                fake.fake_no_wait(1)
                assert refused(lambda: kv.attend(0, a, a + 65536, 2, stream=failing), "failed") == "RuntimeError"
                fake.fake_no_wait(0)
                log()
                kv.attend(0, a, a + 65536, 2, stream=0x80)
                lines = [l.split() for l in log("record", "wait", "launch")]
                assert [l[0] for l in lines][:3] == ["record"] * (first == 0) + ["wait", "launch"] + ["launch"] * (first != 0 and len(lines) > 2), lines
                assert first or lines[0][-1] == hex(be.stream())
    """)
