"""Results of HipBackend's calls (CPU, with a stand-in for the library): each caller gets those of its own call, whatever other
threads and backends do during it."""
import ctypes as C
import threading

import pytest

from rosylnalive_amd import gpu_core
from rosylnalive_amd.gpu_core import Completion, HipBackend


class _Library:
    """Submissions and waits that write their results, and then let the other thread make its call before they return."""

    def __init__(self):
        self.turn = threading.Barrier(2, timeout=30)

    def lrm_hip_submit(self, device, commands, repeat, fence):
        C.cast(fence, C.POINTER(C.c_uint64))[0] = repeat
        self.turn.wait()
        self.turn.wait()
        return 0

    def lrm_hip_wait(self, device, submission, dispatches, timers):
        C.cast(dispatches, C.POINTER(C.c_int))[0] = submission + 100
        C.cast(timers, C.POINTER(C.c_int))[0] = 0
        self.turn.wait()
        self.turn.wait()
        return 0


class _List:
    _h = None


def _backend():
    b = HipBackend.__new__(HipBackend)
    b._h, b._borrowed = None, True
    return b


@pytest.mark.parametrize("shared", [True, False], ids=["one backend", "two backends"])
def test_results_of_calls_in_two_threads(monkeypatch, shared):
    library = _Library()
    monkeypatch.setattr(gpu_core, "lib", lambda: library)
    first = _backend()
    second = first if shared else _backend()
    got = {}

    def steps(name, backend, numbers):
        got[name] = [(int(backend.submit(_List(), n)), backend.wait(n)) for n in numbers]

    other = threading.Thread(target=steps, args=("b", second, range(50, 60)))
    other.start()
    steps("a", first, range(1, 11))
    other.join()
    assert got["a"] == [(n, Completion(n, n + 100, [])) for n in range(1, 11)]
    assert got["b"] == [(n, Completion(n, n + 100, [])) for n in range(50, 60)]
