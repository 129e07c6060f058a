"""Submissions that share a completion event: short lists made right behind each other, waited for in any order; and replays of
short reusable lists, which are launched again rather than captured, next to captured ones."""
import ctypes as C
import time

import numpy as np
import pytest

from gpu_session import Session
from rosylnalive_amd import _native
from rosylnalive_amd.gpu_core import DType, GpuContractException

pytestmark = pytest.mark.gpu

F32 = DType.F32
N = 5000


@pytest.fixture()
def sess():
    x = np.arange(N, dtype=np.float32)
    s = Session({"x": (F32, (N,), 0, x), "y": (F32, (N,), 0, None), "z": (F32, (N,), 0, None)})
    yield s
    s.close()


def _scale(s, cl, a, times=1, src="x", dst="y"):
    for _ in range(times):
        cl.dispatch("scale_f32", s.fields("scale_f32", x=src, y=dst, n=N, a=a))


@pytest.mark.parametrize("order", ["first to last", "last to first", "shuffled"])
def test_waits_in_any_order(sess, order):
    lists, fences = [], []
    for i in range(150):
        cl = sess.backend.begin()
        _scale(sess, cl, float(i), times=1 + i % 3)
        fences.append(sess.backend.submit(cl))
        lists.append(cl)
    assert fences == sorted(set(fences))
    turn = list(range(150))
    if order == "last to first":
        turn.reverse()
    elif order == "shuffled":
        np.random.default_rng(4).shuffle(turn)
    for i in turn:
        c = sess.backend.wait(fences[i])
        assert c.submission == fences[i] and c.dispatches == 1 + i % 3
        if i == 149:  # the newest: its result is there once its wait returns
            assert np.array_equal(sess.read("y"), np.arange(N, dtype=np.float32) * np.float32(149))
    assert sess.backend.wait(fences[3]).dispatches == 1  # again
    with pytest.raises(GpuContractException, match="never made"):
        sess.backend.wait(int(fences[-1]) + 1)
    for cl in lists:
        cl.release()


def test_a_wait_between_submissions(sess):
    """A program that keeps two submissions under way: each waited-for one is complete when its wait returns."""
    prev = None
    for i in range(1, 60):
        cl = sess.backend.begin()
        _scale(sess, cl, float(i))
        _scale(sess, cl, 2.0, src="y", dst="z")
        fence = sess.backend.submit(cl)
        if prev is not None:
            assert sess.backend.wait(prev[0]).dispatches == 2
            prev[1].release()
        prev = (fence, cl)
    sess.backend.wait(prev[0])
    assert np.array_equal(sess.read("z"), np.arange(N, dtype=np.float32) * np.float32(118))


@pytest.mark.parametrize("launches", [1, 6, 7, 20])
def test_replays_of_short_and_long_lists(sess, launches):
    """z = x 2^launches by doubling in place, replayed `repeat` times with new inputs between, however the list is replayed; no
    change after the first submission."""
    cl = sess.backend.begin(reusable=True)
    for _ in range(launches):
        cl.dispatch("scale_f32", sess.fields("scale_f32", x="z", y="z", n=N, a=2.0))
    for repeat in (1, 3, 2):
        x = np.random.default_rng(repeat).standard_normal(N).astype(np.float32)
        sess.write("z", x)
        c = sess.backend.wait(sess.backend.submit(cl, repeat))
        assert c.dispatches == launches * repeat
        assert np.array_equal(sess.read("z"), x * np.float32(2.0 ** (launches * repeat)))
        with pytest.raises(GpuContractException, match="cannot be changed"):
            _scale(sess, cl, 1.0)
    cl.release()
    cl = sess.backend.begin(reusable=True)
    cl.begin_timer("t")
    _scale(sess, cl, 1.0)
    cl.end_timer(0)
    with pytest.raises(GpuContractException, match="timers"):
        sess.backend.submit(cl)
    cl.release()


@pytest.fixture()
def long():
    """A session whose one launch over 32 million values takes about 60 us, and small tensors beside them."""
    n = 1 << 25
    s = Session({"big": (F32, (n,), 0, np.zeros(n, np.float32)), "x": (F32, (N,), 0, np.ones(N, np.float32)),
                 "y": (F32, (N,), 0, None)})
    s.n_big = n
    yield s
    s.close()


def _long_list(s, launches, reusable):
    cl = s.backend.begin(reusable=reusable)
    for _ in range(launches):
        cl.dispatch("scale_f32", s.fields("scale_f32", x="big", y="big", n=s.n_big, a=1.0))
    return cl


@pytest.mark.parametrize("form", ["direct", "captured", "one shot"])
@pytest.mark.parametrize("pause", [0.0, 1e-3])
def test_a_wait_does_not_cover_long_work_submitted_later(long, form, pause):
    """Two short submissions right behind each other, so that the second has no completion event of its own, then a long one, at
    once or a millisecond later: the wait for the second returns while the long one still runs, which the wait for that one
    then shows."""
    s = long
    launches = {"direct": 4, "captured": 40, "one shot": 400}[form]
    repeat = 400 // launches
    short = s.backend.begin(reusable=True)
    _scale(s, short, 2.0)
    s.backend.wait(s.backend.submit(short))
    late = _long_list(s, launches, form != "one shot")
    if form != "one shot":
        s.backend.wait(s.backend.submit(late))  # (the first submission captures)
    good = 0
    for _ in range(5):
        time.sleep(1e-3)
        a, b = s.backend.submit(short), s.backend.submit(short)
        if pause:
            s.backend.wait(a)
            time.sleep(pause)
        c = s.backend.submit(late, repeat if form != "one shot" else 1)
        t0 = time.perf_counter()
        s.backend.wait(b)
        t1 = time.perf_counter()
        s.backend.wait(c)
        t2 = time.perf_counter()
        good += t1 - t0 < t2 - t1
        if form == "one shot":
            late.release()
            late = _long_list(s, launches, False)
    assert good >= 4  # (the host may be held up once)
    short.release()
    late.release()


@pytest.mark.parametrize("order", ["first to last", "last to first", "every third", "shuffled"])
@pytest.mark.parametrize("launches", [5, 6, 40])
def test_results_are_there_when_a_wait_returns(launches, order):
    """Submissions that take the GPU much longer than the host, right behind each other (those of up to six launches share events,
    longer ones have their own), each with a result of its own as its last launch: when a wait returns, a copy that nothing
    orders behind the device's stream (the null stream's, from the tensor's address) finds the result, and those of all
    submissions before it."""
    n, count = 1 << 25, 12
    x = np.arange(1, N + 1, dtype=np.float32)
    s = Session({"big": (F32, (n,), 0, np.zeros(n, np.float32)), "x": (F32, (N,), 0, x),
                 **{f"out{i}": (F32, (N,), 0, None) for i in range(count)}})
    copy = C.CDLL(_native.LIB_PATH).hipMemcpy  # of the runtime that the library runs on
    copy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    lists = []
    for i in range(count):
        cl = s.backend.begin(reusable=i % 2 == 1)
        for _ in range(launches - 1):
            cl.dispatch("scale_f32", s.fields("scale_f32", x="big", y="big", n=n, a=1.0))
        _scale(s, cl, float(i + 2), dst=f"out{i}")
        lists.append(cl)
    turn = list(range(count))
    if order == "last to first":
        turn.reverse()
    elif order == "every third":
        turn = turn[2::3] + turn[0::3] + turn[1::3]
    elif order == "shuffled":
        np.random.default_rng(6).shuffle(turn)
    at = [s.heap.view(s.tok[f"out{i}"]).address for i in range(count)]
    got = np.empty(N, np.float32)
    try:
        fences = [s.backend.submit(cl) for cl in lists]
        for i in turn:
            assert s.backend.wait(fences[i]).dispatches == launches
            for j in range(i + 1):
                assert copy(got.ctypes.data, at[j], got.nbytes, 2) == 0
                assert np.array_equal(got, x * np.float32(j + 2)), (i, j)
    finally:
        for cl in lists:
            cl.release()
        s.close()
