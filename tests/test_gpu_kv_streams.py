"""Calls on one key/value cache over streams whose handles do not tell them apart: every result is that of the calls in order."""
from __future__ import annotations

import ctypes as C
import threading

import numpy as np
import pytest
import torch

from jax4j_amd import IllegalArgumentException
from jax4j_amd import _native as N
from test_gpu_kept_memory import Hip
from test_gpu_kv import dev, model  # noqa: F401

pytestmark = pytest.mark.gpu


class Steps:
    """Tokens of one sequence, appended and attended to."""

    def __init__(self, model):  # noqa: F811
        self.kv = model(kv_heads=2, head_dim=128, pages=100, page_tokens=16, sequences=1, sequence_pages=100).kv
        rng = np.random.default_rng(7)
        self.k, self.v, self.q = (dev(rng.standard_normal((12, 100, h, 128)).astype(np.float32)) for h in (2, 2, 8))
        self.out = torch.zeros_like(self.q)
        torch.cuda.synchronize()

    def append(self, i, stream):
        self.kv.extend([0], [100], stream=stream)
        self.kv.append(0, self.k[i].data_ptr(), self.v[i].data_ptr(), stream=stream)

    def attend(self, i, stream):
        self.kv.attend(0, self.q[i].data_ptr(), self.out[i].data_ptr(), 8, stream=stream)

    def check(self, n):
        torch.cuda.synchronize()
        got = self.out.clone()
        self.kv.truncate([0], [0])
        for i in range(n):
            self.append(i, 0)
            self.attend(i, 0)
        torch.cuda.synchronize()
        assert torch.equal(got[:n], self.out[:n]) and bool(self.out[:n].abs().amax((1, 2, 3)).min() > 0)


@pytest.mark.parametrize("handle", [1, 2], ids=["hipStreamLegacy", "hipStreamPerThread"])
def test_one_handle_in_two_threads(model, handle):  # noqa: F811
    """A stream of each thread's own, or one for both: appended behind a long kernel in one thread, attended to in another, and back."""
    steps, lib = Steps(model), N.load()
    turn, failed = [threading.Event() for _ in range(14)], []

    def work(me):
        try:
            for i in range(12):
                if i % 2 == me:
                    assert turn[i].wait(60)
                    if i:
                        steps.attend(i - 1, handle)
                    assert lib.j4q_spin(500, handle) == 0
                    steps.append(i, handle)
                    turn[i + 1].set()
            assert turn[13].wait(60)  # its stream lives until all is done
        except BaseException as e:
            failed.append(e)
        finally:
            for t in turn:
                t.set()

    threads = [threading.Thread(target=work, args=(me,)) for me in (0, 1)]
    for t in threads:
        t.start()
    turn[0].set()
    assert turn[12].wait(60)
    steps.attend(11, 0)
    torch.cuda.synchronize()
    turn[13].set()
    for t in threads:
        t.join(60)
    assert not failed, failed
    steps.check(12)


def test_a_stream_created_where_one_was_destroyed(model):  # noqa: F811
    steps, lib, hip = Steps(model), N.load(), Hip()
    for i in range(12):
        assert lib.j4q_spin(500, hip.stream) == 0
        steps.append(i, hip.stream.value)
        hip.ok("hipStreamDestroy", hip.stream)  # its calls are still queued
        hip = Hip()
        steps.attend(i, hip.stream.value)
    hip.close()
    steps.check(12)


def test_the_engine_stream_captured(model, backend):  # noqa: F811
    """Attention captured on the engine stream: a call on another stream is refused meanwhile and goes through afterwards, and every
    replay gives what the same call gives."""
    steps, hip = Steps(model), Hip()
    st, graph, run = C.c_void_p(backend.stream()), C.c_void_p(), C.c_void_p()
    steps.append(0, 0)
    steps.append(1, 0)
    steps.kv.begin([0], [100])
    steps.attend(1, 0)
    torch.cuda.synchronize()
    hip.ok("hipStreamBeginCapture", st, 2)  # relaxed
    steps.attend(0, 0)
    with pytest.raises(IllegalArgumentException, match="engine stream"):
        steps.append(2, hip.stream.value)
    with pytest.raises(IllegalArgumentException, match="engine stream"):
        steps.attend(2, hip.stream.value)
    hip.ok("hipStreamEndCapture", st, C.byref(graph))
    hip.ok("hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
    assert steps.kv.lengths([0]).tolist() == [200]
    for _ in range(4):
        steps.out[0].zero_()
        torch.cuda.synchronize()
        hip.ok("hipGraphLaunch", run, st)
        hip.wait()
        got = steps.out[0].clone()
        steps.attend(0, hip.stream.value)
        torch.cuda.synchronize()
        assert torch.allclose(got, steps.out[0], rtol=0, atol=4e-5) and bool(got.abs().max() > 0)  # perhaps in other ranges of the tokens
    hip.ok("hipGraphExecDestroy", run)
    hip.ok("hipGraphDestroy", graph)
    hip.close()
