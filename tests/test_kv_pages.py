"""The 8-bit key/value cache without a GPU (fakehip.py): which pages sequences hold after extend, fork, cut, evict and compact,
what calls refuse, and what they launch."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest

import fakehip
from jax4j_amd import _native as N


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    return fakehip.build_shim(tmp_path_factory.mktemp("fake_hip"))


SETUP = """
from jax4j_amd import KvCache, Rope
def cache(**more):
    return KvCache(be, **dict(dict(layers=2, kv_heads=2, head_dim=64, pages=12, page_tokens=16, sequences=4, sequence_pages=8), **more))
def refused(call, *words):
    try:
        call()
    except Exception as e:
        assert all(w in str(e) for w in words), str(e)
        return type(e).__name__
    return "nothing"
"""


def run(shim, body):
    return fakehip.run(shim, SETUP + "\n".join(line[8:] if line.startswith(" " * 8) else line for line in body.splitlines()))


@pytest.mark.parametrize("page", [16, 32, 64])
def test_pages_by_a_model(shim, page):
    """Random calls against lists of pages and counts of their holders, the lowest free page first."""
    steps = run(shim, f"""
        import random
        P, pages, S, width = {page}, 24, 6, 10
        kv = cache(pages=pages, page_tokens=P, sequences=S, sequence_pages=width)
        rng = random.Random({page})
        held, length, refs = [[] for _ in range(S)], [0] * S, [0] * pages
        def take():
            p = refs.index(0)
            refs[p] = 1
            return p
        def drop(p):
            if p >= 0:
                refs[p] -= 1
        done = 0
        for _ in range(600):
            what = rng.choice(["extend"] * 4 + ["fork", "copy", "cut", "free", "evict", "compact"])
            seqs = rng.sample(range(S), rng.randint(1, 3))
            before = ([list(h) for h in held], list(length), list(refs))
            short = False
            try:
                if what == "extend":
                    tokens = [rng.choice([1, 1, 5, P, 3 * P]) for _ in seqs]
                    if any(length[s] + t > width * P for s, t in zip(seqs, tokens)):
                        assert refused(lambda: kv.extend(seqs, tokens), "table") == "IllegalArgumentException"
                        continue
                    for s, t in zip(seqs, tokens):
                        if length[s] % P and refs[held[s][-1]] > 1:
                            old = held[s][-1]
                            held[s][-1] = take()
                            drop(old)
                        length[s] += t
                        while len(held[s]) * P < length[s]:
                            held[s].append(take())
                    call = lambda: kv.extend(seqs, tokens)
                elif what in ("fork", "copy"):
                    dst = [s for s in range(S) if not length[s]][:2]
                    src = [rng.choice([s for s in range(S) if s not in dst] or [0]) for _ in dst]
                    if not dst:
                        continue
                    for a, b in zip(src, dst):
                        length[b] = length[a]
                        held[b] = [p if p < 0 else take() if what == "copy" else p for p in held[a]]
                        if what == "fork":
                            for p in held[b]:
                                if p >= 0:
                                    refs[p] += 1
                    call = lambda: kv.fork(src, dst, share=what == "fork")
                elif what in ("cut", "free"):
                    to = [0 if what == "free" else rng.randint(0, length[s]) for s in seqs]
                    if any(t % P and held[s][t // P] < 0 for s, t in zip(seqs, to)):
                        assert refused(lambda: kv.truncate(seqs, to), "evicted") == "IllegalArgumentException"
                        continue
                    for s, t in zip(seqs, to):
                        while len(held[s]) * P >= t + P:
                            drop(held[s].pop())
                        length[s] = t
                    call = lambda: kv.truncate(seqs, to)
                elif what == "evict":
                    w, k = rng.randint(1, 3 * P), rng.choice([0, 4, P + 1])
                    for s in seqs:
                        for j, p in enumerate(held[s]):
                            if p >= 0 and j * P >= k and (j + 1) * P - 1 <= length[s] - w:
                                drop(p)
                                held[s][j] = -1
                    call = lambda: kv.evict(seqs, w, k)
                else:
                    live = sum(r > 0 for r in refs)
                    for p in range(live, pages):
                        if refs[p]:
                            h = refs.index(0)
                            refs[h], refs[p] = refs[p], 0
                            held = [[h if x == p else x for x in t] for t in held]
                    call = kv.compact
            except ValueError:  # no page is free
                held, length, refs = before
                call = {{"extend": lambda: kv.extend(seqs, tokens), "copy": lambda: kv.fork(src, dst, share=False)}}[what]
                assert refused(call, "pages needed") == "RuntimeError"
                short = True
            if not short:
                call()
            done += not short
            assert kv.tables(range(S)).tolist() == [h + [-1] * (width - len(h)) for h in held], what
            assert [kv.length(s) for s in range(S)] == length
            assert kv.info()["pages_free"] == refs.count(0)
        kv.truncate(range(S), [0] * S)
        assert kv.info()["pages_free"] == pages
        kv.destroy()
        result = done
    """)
    assert steps > 200


def test_refusals(shim):
    run(shim, """
        bad = "IllegalArgumentException"
        for name, value in dict(layers=0, kv_heads=0, head_dim=80, page_tokens=24, pages=0, sequences=0, sequence_pages=0).items():
            assert refused(lambda: cache(**{name: value}), "kv cache") == bad, name
        assert refused(lambda: cache(pages=1 << 40)) == bad and refused(lambda: cache(sequences=1 << 20, sequence_pages=1 << 20)) == bad
        kv = cache()
        a = address(1 << 20)
        r = lambda **k: Rope(a, a, 10, 64, **k)
        assert refused(lambda: kv.append(0, a, a), "no step") == bad and refused(lambda: kv.attend(0, a, a, 2), "no step") == bad
        for seqs, tokens in (([], []), ([4], [1]), ([-1], [1]), ([1, 1], [1, 1]), ([0], [0]), ([0], [-3]), ([0], [129])):
            assert refused(lambda: kv.extend(seqs, tokens), "kv extend") == bad, (seqs, tokens)
        assert refused(lambda: kv.extend([0], [1, 2]), "counts") == bad and refused(lambda: kv.extend([0], [1 << 40]), "32 bits") == bad
        assert refused(lambda: kv.begin([0], [1]), "kv begin") == bad
        assert refused(lambda: kv.extend([0, 1, 2, 3], [64, 64, 64, 1]), "13 pages needed, 12 free") == "RuntimeError"
        assert kv.info()["pages_free"] == 12 and kv.info()["step_rows"] == 0
        kv.extend([2, 0], [20, 3])
        assert kv.info()["step_sequences"] == 2 and kv.info()["step_rows"] == 23
        for call in (lambda: kv.append(2, a, a), lambda: kv.append(-1, a, a), lambda: kv.append(0, 0, a), lambda: kv.append(0, a, 0),
                     lambda: kv.append(0, a + 4, a), lambda: kv.append(0, a, a, stride=127), lambda: kv.append(0, a, a, stride=130),
                     lambda: kv.append(0, a, a, DType.BF16, stride=132), lambda: kv.append(0, a, a, q_ptr=a), lambda: kv.append(0, a, a, DType.I8),
                     lambda: kv.append(0, a, a, rope=Rope(a, a, 0, 64)), lambda: kv.append(0, a, a, rope=Rope(a, a, 10, 66)),
                     lambda: kv.append(0, a, a, rope=Rope(a, a, 10, 63)), lambda: kv.append(0, a, a, rope=Rope(0, a, 10, 64)),
                     lambda: kv.append(0, a, a, rope=r(sections=(16, 16))), lambda: r(sections=(16, 15)), lambda: r(pair_axis=[256] * 32),
                     lambda: r(sections=(32,), pair_axis=[0] * 32), lambda: kv.append(0, a, a, rope=r(positions=a + 2)),
                     lambda: kv.attend(2, a, a, 2), lambda: kv.attend(0, a, a, 3), lambda: kv.attend(0, a, a, 0), lambda: kv.attend(0, 0, a, 2),
                     lambda: kv.attend(0, a, 0, 2), lambda: kv.attend(0, a + 8, a, 2), lambda: kv.attend(0, a, a, 2, q_type=DType.I8),
                     lambda: kv.attend(0, a, a, 2, out_stride=100), lambda: kv.attend(0, a, a, 2, window=-1), lambda: kv.attend(0, a, a, 2, sinks=-1),
                     lambda: kv.attend(0, a, a, 2, scale=-1.0), lambda: kv.attend(0, a, a, 2, scale=float("nan")),
                     lambda: kv.fork([0], [2]), lambda: kv.fork([0, 0], [1, 1]), lambda: kv.fork([9], [1]), lambda: kv.fork([0], [1, 3]),
                     lambda: kv.truncate([2], [21]), lambda: kv.truncate([2], [-1]), lambda: kv.truncate([2, 2], [1, 1]),
                     lambda: kv.evict([0], 0, 0), lambda: kv.evict([0], 5, -1), lambda: kv.evict([7], 5, 1),
                     lambda: kv.read(0, [0], [-1], 4, a, a), lambda: kv.read(0, [0], [0], 0, a, a), lambda: kv.read(0, [0], [0], 4, 0, 0),
                     lambda: kv.read(0, [0], [0], 4, a + 4, 0), lambda: kv.read(3, [0], [0], 4, a, a), lambda: kv.read(0, [0, 1], [0], 4, a, a),
                     lambda: be.rope_into(a, a, 1, 1, 64, r()), lambda: be.rope_into(a, a + 256, 3, 1, 64, r(positions=a)),
                     lambda: be.rope_into(a, a, 1, 1, 63, r(positions=a)), lambda: be.rope_into(a, a, 0, 1, 64, r(positions=a)),
                     lambda: be.rope_into(a, a, 1, 1, 32, r(positions=a)), lambda: be.rope_into(a, a, 2, 2, 64, r(positions=a), x_stride=127),
                     lambda: be.rope_into(0, a, 1, 1, 64, r(positions=a)), lambda: be.rope_into(a + 2, a + 2, 1, 1, 64, r(positions=a)),
                     lambda: be.rope_into(a, a, 1, 1, 64, r(positions=a), DType.I8)):
            assert refused(call) == bad, call.__code__.co_firstlineno
        assert len(launches()) == 2 and kv.length(0) == 3  # of the cache's making and the one extend
        for call in (lambda: kv.fork([0], [1], stream=0x70), lambda: kv.extend([0], [1], stream=0x70), lambda: kv.begin([0], [1], stream=0x70),
                     lambda: kv.compact(stream=0x70), lambda: kv.evict([0], 1, stream=0x70), lambda: kv.read(0, [0], [0], 4, a, a, stream=0x70)):
            fake.fake_capture(0x70, 1)
            assert refused(call, "captured") == bad
            fake.fake_capture(0x70, 0)
        h = kv.handle
        kv.destroy()
        kv.destroy()
        kv.handle = h
        assert refused(lambda: kv.extend([0], [1]), "destroyed") == bad and refused(kv.destroy, "destroyed") == bad
        assert cache().handle != h
    """)


def test_shared_and_evicted_pages_are_not_written(shim):
    run(shim, """
        kv = cache()
        a = address(1 << 20)
        kv.extend([0], [20])
        kv.append(0, a, a)
        kv.fork([0], [1])
        assert refused(lambda: kv.append(1, a, a), "shared") == "IllegalArgumentException"
        kv.begin([0], [1])
        assert refused(lambda: kv.append(0, a, a), "shared") == "IllegalArgumentException"
        kv.attend(0, a, a, 2)
        kv.extend([1, 0], [1, 1])  # the first takes a page of its own, the other keeps the one they had
        assert kv.tables([0, 1])[:, :2].tolist() == [[0, 1], [0, 2]]
        kv.append(0, a, a)
        kv.begin([0], [21])  # from the page that they share on
        assert refused(lambda: kv.append(0, a, a), "shared") == "IllegalArgumentException"
        kv.truncate([1], [0])
        kv.append(0, a, a)
        kv.extend([0], [60])
        kv.evict([0], 1)
        assert refused(lambda: kv.append(0, a, a), "evicted") == "IllegalArgumentException"
        kv.truncate([0], [80])
        assert kv.info()["step_rows"] == 0 and refused(lambda: kv.attend(0, a, a, 2), "no step") == "IllegalArgumentException"
    """)


def test_what_a_step_launches(shim):
    """One launch for a step's tables, one a layer to append, one or two to attend; no allocation, and a wait only where
    the stream is another than the call's before."""
    counts = run(shim, """
        kv = cache(layers=4, pages=2000, sequence_pages=400, sequences=64)
        a = address(1 << 22)
        kv.extend(range(64), [100] * 64)
        log()
        result = []
        kv.extend(range(64), [1] * 64)
        result.append(len(launches()))
        kv.append(1, a, a)
        result.append(len(launches()))
        kv.attend(1, a, a, 8)
        result.append(len(launches()))
        kv.attend(1, a, a, 8, stream=0x70)
        kv.attend(1, a, a, 8, stream=0x70)
        kv.attend(1, a, a, 8)
        lines = log()
        result.append(sum(l.split()[0] == "wait" for l in lines))
        result.append(sum(l.split()[0] in ("malloc", "mallocasync", "free") for l in lines))
    """)
    assert counts[:2] == [1, 1] and counts[2] <= 2 and counts[3:] == [2, 0]


def test_captured_append_reaches_every_block_of_a_replay(shim):
    """16 tokens at the beginning of a block are one block's, in a replay two blocks'; 400 uneven ones are up to 26 and 1."""
    run(shim, """
        kv = cache(pages=200, sequences=10, sequence_pages=100)
        a = address(1 << 22)
        def groups(stream):
            log()
            kv.append(0, a, a, stream=stream)
            return int(launches()[0][3])
        kv.extend([0, 1], [16, 16])
        assert groups(0) == 2 * 2
        fake.fake_capture(0x70, 1)
        assert groups(0x70) == 2 * 2 * 2
        fake.fake_capture(0x70, 0)
        kv.extend(range(10), [400] + [1] * 9)
        assert groups(0) == 2 * (25 + 9)
        fake.fake_capture(0x70, 1)
        assert groups(0x70) == 2 * (26 + 9)
        fake.fake_capture(0x70, 0)
    """)


def test_memory_of_a_cache_is_given_back(shim):
    run(shim, """
        before = fake.fake_used()
        kv = cache()
        assert fake.fake_used() > before
        kv.destroy()
        assert fake.fake_used() == before
        fake.fake_capacity(before + (1 << 20))  # room for the pool and not for the rest
        assert refused(cache, "kv cache failed") == "RuntimeError"
        assert fake.fake_used() == before
    """)


def test_a_fork_of_what_the_call_itself_makes_is_refused(shim):
    """Sequence 1 is empty when the call begins and would be a copy of 0 when it is copied: pages that nobody counted."""
    run(shim, """
        kv = cache(pages=8)
        kv.extend([0], [4 * 16])
        for share in (True, False):
            assert refused(lambda: kv.fork([0, 1], [1, 2], share=share), "made by this call") == "IllegalArgumentException"
            assert refused(lambda: kv.fork([3], [3], share=share), "made by this call") == "IllegalArgumentException"
        assert kv.info()["pages_free"] == 4 and [kv.length(s) for s in range(4)] == [64, 0, 0, 0]
    """)


def test_outputs_over_inputs(shim):
    """In place or apart, columns of the same rows being apart; what lies across is refused."""
    run(shim, """
        kv = cache()
        kv.extend([0, 1], [3, 20])  # 23 rows; heads of 64 floats: k, v 128 a row, q of 4 heads 256
        a = address(1 << 20)
        bad = "IllegalArgumentException"
        row = 4 * (256 + 128 + 128)  # q, k, v of a fused product
        append = lambda q_out, q=0: kv.append(0, a + 4 * 256, a + 4 * 384, q_ptr=a + q, q_out_ptr=a + q_out, heads=4, stride=512, q_stride=512)
        append(0)
        append(23 * row)
        for q_out in (16, 4 * 256, 4 * 255 * 4, row, 3 * row + 1024, 22 * row):
            assert refused(lambda: append(q_out), "overlaps") == bad, q_out
        attend = lambda out, **k: kv.attend(0, a, a + out, 4, q_stride=512, **k)
        attend(0, out_stride=512)
        attend(4 * 256, out_stride=512)
        attend(5 * row + 4 * 256, out_stride=512)
        attend(23 * row)
        for out, k in ((0, {}), (0, dict(out_stride=512, out_type=DType.BF16)), (16, dict(out_stride=512)), (4 * 256, {}), (row, dict(out_stride=512))):
            assert refused(lambda: attend(out, **k), "overlaps") == bad, (out, k)
        rope = Rope(a, a, 10, 64, positions=a)
        turn = lambda out: be.rope_into(a, a + out, 23, 4, 64, rope, x_stride=512, out_stride=512)
        turn(0)
        turn(1024)
        for out in (16, 1028, row, row - 16):
            assert refused(lambda: turn(out), "overlaps") == bad, out
    """)


def test_no_host_memory(shim, monkeypatch):
    """Every call that finds too little host memory for its lists says so, and leaves the cache as it was."""
    monkeypatch.setenv("MALLOC_ARENA_MAX", "1")  # long lists neither from another thread's heap nor from what was freed
    monkeypatch.setenv("MALLOC_MMAP_THRESHOLD_", str(1 << 17))
    run(shim, """
        import resource
        be.upload_quantized(np.zeros(34, np.uint8), QuantType.Q8_0, (1, 32))
        def limited(call, more=1 << 20):
            used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
            resource.setrlimit(resource.RLIMIT_AS, (used + more, resource.RLIM_INFINITY))
            try:
                return refused(call, "failed", "out of host memory")
            finally:
                resource.setrlimit(resource.RLIMIT_AS, (resource.RLIM_INFINITY, resource.RLIM_INFINITY))
        before = fake.fake_used()
        assert limited(lambda: cache(pages=1 << 26), 64 << 20) == "RuntimeError"
        assert fake.fake_used() == before
        # pages of 1 KiB here: tables large against the pool
        kv = cache(layers=1, kv_heads=1, pages=1 << 20, sequences=3, sequence_pages=1 << 20)
        tokens = 1 << 23
        def state():
            return kv.info(), [kv.length(s) for s in range(3)]
        def held(call):
            was = state()
            assert limited(call) == "RuntimeError"
            assert state() == was
            call()
        held(lambda: kv.extend([0], [tokens]))
        table = kv.tables([0]).tobytes()
        assert limited(lambda: kv.fork([0], [1])) == "RuntimeError" and kv.tables([0]).tobytes() == table and kv.length(1) == 0
        kv.extend([1], [16])
        kv.truncate([0], [tokens // 2])
        held(kv.compact)
    """)


@pytest.fixture(scope="module")
def failing_shim(tmp_path_factory):
    """The same runtime, whose launches fail while fake_fail_launches(1) holds."""
    folder = tmp_path_factory.mktemp("failing_hip")
    text = (fakehip.TESTS / "fake_hip.cpp").read_text()
    for name in ("hipLaunchKernel", "hipExtLaunchKernel"):
        head = f"F hipError_t {name}("
        at = text.index("LOCK;", text.index(head)) + len("LOCK;")
        text = text[:at] + " if (launches_fail) return ret(hipErrorLaunchFailure);" + text[at:]
    at = text.index("F hipError_t hipLaunchKernel(")
    text = text[:at] + "static bool launches_fail = false;\nF void fake_fail_launches(int on) { launches_fail = on != 0; }\n" + text[at:]
    (folder / "fake_hip.cpp").write_text(text)
    lib = folder / "fake_hip.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", f"-I{fakehip.ROCM / 'include'}",
                    "-o", str(lib), str(folder / "fake_hip.cpp")], check=True)
    return lib


def test_a_change_that_the_device_did_not_get(failing_shim):
    """Its tables are then not the host's: the cache is refused, and can be looked at and destroyed."""
    run(failing_shim, """
        a = address(1 << 20)
        for change in (lambda kv: kv.extend([1], [16]), lambda kv: kv.begin([0], [1]), lambda kv: kv.fork([0], [2]), lambda kv: kv.evict([0], 1),
                       lambda kv: (kv.truncate([3], [0]), kv.compact())):
            kv = cache()
            kv.extend([3, 0], [20, 40])
            kv.append(0, a, a)
            fake.fake_fail_launches(1)
            assert refused(lambda: kv.append(0, a, a), "kv append failed") == "RuntimeError"  # changes nothing here
            assert refused(lambda: change(kv), "failed") == "RuntimeError"
            fake.fake_fail_launches(0)
            for call in (lambda: kv.extend([0], [1]), lambda: kv.append(0, a, a), lambda: kv.attend(0, a, a, 2), lambda: kv.read(0, [0], [0], 4, a, a)):
                assert refused(call, "an earlier call") == "RuntimeError"
            kv.info()
            kv.destroy()
    """)


def test_binding_matches_the_header(tmp_path):
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    names = {"j4q_kv_config": N.KvConfig, "j4q_kv_desc": N.KvDesc, "j4q_rope": N.RopeArgs, "j4q_kv_append_args": N.KvAppendArgs,
             "j4q_kv_attend_args": N.KvAttendArgs}
    lines = [f'printf("%zu\\n", sizeof({c}));' for c in names]
    for c, t in names.items():
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in t._fields_]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "jax4j_mi355x.h"\nint main(void) {' + "".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c11", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    want = [C.sizeof(t) for t in names.values()] + [getattr(t, f[0]).offset for t in names.values() for f in t._fields_]
    assert got == want
