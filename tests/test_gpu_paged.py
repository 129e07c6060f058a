"""The paged key/value cache on the GPU against float64 (paged_oracle.py): the step's plan by equality, the append and the
attention within bounds formed from their roundings, alone and as a program runs them one after the other."""
import ctypes as C

import numpy as np
import pytest

import paged_oracle as O
from gpu_session import POISON_16, Session
from rosylnalive_amd import _native
from rosylnalive_amd.gpu_core import (PAGED_NONE, Arena, ArgBlock, DType, GpuContractException, HeapPlanner, HipBackend,
                                      TensorFlags, TensorTable, attention_paged_workspace_words)

pytestmark = pytest.mark.gpu

F32, BF16, F16, U32 = DType.F32, DType.BF16, DType.F16, DType.U32
RO = TensorFlags.READ_ONLY
DT = {"f16": F16, "bf16": BF16}


def _rank4(v_cache):
    """[pages, kv_heads, page / 8, head_dim, 8] as the rank that a table row takes."""
    return v_cache.shape[:3] + (v_cache.shape[3] * 8,)


# ---------------------------------------------------------------- plan

def _plan_case(past, fresh, page, blocks, pages, free, tokens, seed=0):
    r = np.random.default_rng(seed)
    past, fresh = np.array(past, np.int64), np.array(fresh, np.int64)
    R = len(past)
    table = np.full((R, blocks), PAGED_NONE, np.uint32)
    for i in range(R):
        n = -(-min(int(past[i]), blocks * page) // page)
        table[i, :n] = r.integers(0, pages, n)
    free = np.array(free, np.uint32)
    init = {"positions": r.integers(0, 99, tokens).astype(np.uint32), "slots": r.integers(0, 99, tokens).astype(np.uint32)}
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    s = Session({"past": u(past), "fresh": u(fresh), "free": u(free if len(free) else [0]), "table": u(table),
                 "starts": (U32, (R + 1,), 0, None), "context": (U32, (R,), 0, None), "positions": u(init["positions"]),
                 "slots": u(init["slots"]), "counts": (U32, (3,), 0, None)})
    names = ("table", "starts", "context", "positions", "slots", "counts")
    try:
        for _ in range(2):  # a step planned again gives the same
            cl = s.backend.begin()
            cl.dispatch("paged_plan", s.fields("paged_plan", **{n: n for n in s.spec}, requests=R, blocks=blocks, page=page,
                                               pages=pages, free_count=len(free), tokens=tokens))
            s.backend.wait(s.backend.submit(cl))
            cl.release()
            got = {n: s.read(n) for n in names}
            want = O.plan(past, fresh, free, table, blocks, page, pages, tokens, init["positions"], init["slots"])
            for n, w in zip(names, want):
                assert np.array_equal(got[n], w), (n, got[n], w)
    finally:
        s.close()


PLANS = {
    "one_token_first": dict(past=[0], fresh=[1], page=16, blocks=1, pages=1, free=[0], tokens=1),
    "edges_of_a_page": dict(past=[15, 16, 17, 0, 31, 32], fresh=[1, 1, 1, 0, 2, 16], page=16, blocks=4, pages=40,
                            free=range(30, 40), tokens=21),
    "padding_rows_stay": dict(past=[3, 100], fresh=[5, 70], page=64, blocks=5, pages=9, free=[8, 1, 7], tokens=300),
    "nothing_new": dict(past=[3, 0, 64], fresh=[0, 0, 0], page=64, blocks=2, pages=9, free=[], tokens=4),
    "free_pages_run_out": dict(past=[10, 60, 0], fresh=[40, 10, 33], page=16, blocks=8, pages=50, free=[4, 49, 7], tokens=83),
    "page_ids_past_the_cache": dict(past=[16, 0], fresh=[20, 20], page=16, blocks=4, pages=5, free=[77, 4, 5, 0], tokens=40),
    "longer_than_the_table": dict(past=[60, 4, 200], fresh=[10, 1, 3], page=16, blocks=4, pages=30, free=range(20, 30), tokens=14),
    "more_rows_than_planned": dict(past=[5, 6, 7], fresh=[9, 9, 9], page=32, blocks=3, pages=30, free=range(10), tokens=13),
}


@pytest.mark.parametrize("name", list(PLANS))
def test_plan(name):
    _plan_case(**PLANS[name])


@pytest.mark.parametrize("R,page,most_fresh", [(1, 256, 700), (255, 16, 3), (257, 32, 40), (1000, 16, 30), (4096, 64, 5)])
def test_plan_many(R, page, most_fresh):
    r = np.random.default_rng(R)
    past, fresh = r.integers(0, 900, R), r.integers(0, most_fresh + 1, R)
    blocks = 1700 // page + 1
    _plan_case(past, fresh, page, blocks, 60000, r.permutation(60000)[:20000], int(fresh.sum()) + 7, seed=R)


def test_plan_lengths_near_2_32():
    """Sums of lengths past 2^32 saturate; what has a place in table and rows keeps it."""
    big = 0xFFFFFFF0
    s = {"past": np.array([5, big, 7, big], np.uint32), "fresh": np.array([3, 100, big, big], np.uint32)}
    table = np.full((4, 2), PAGED_NONE, np.uint32)
    table[:, 0] = [1, 2, 3, 4]
    table[1:4, 1] = [9, PAGED_NONE, 8]
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    ses = Session({"past": u(s["past"]), "fresh": u(s["fresh"]), "free": u([0, 10, 11]), "table": u(table),
                   "starts": (U32, (5,), 0, None), "context": (U32, (4,), 0, None), "positions": (U32, (200,), 0, None),
                   "slots": (U32, (200,), 0, None), "counts": (U32, (3,), 0, None)})
    try:
        got = ses.run("paged_plan", ["starts", "context", "positions", "slots", "counts"], **{n: n for n in ses.spec},
                      requests=4, blocks=2, page=16, pages=12, free_count=3, tokens=200)
        tab = ses.read("table")
    finally:
        ses.close()
    assert got["starts"].tolist() == [0, 3, 103, 200, 200]
    assert got["context"].tolist() == [8, 32, 32, 32]
    assert tab.tolist() == [[1, PAGED_NONE], [2, 9], [3, 0], [4, 8]]
    assert got["counts"].tolist() == [0xFFFFFFFF, 1, 3]
    assert got["positions"][:3].tolist() == [5, 6, 7] and got["slots"][:3].tolist() == [21, 22, 23]
    assert (got["slots"][3:103] == PAGED_NONE).all()
    assert got["positions"][103:].tolist() == list(range(7, 104))
    assert got["slots"][103:128].tolist() == [3 * 16 + p for p in range(7, 16)] + list(range(16))
    assert (got["slots"][128:] == PAGED_NONE).all()


# ---------------------------------------------------------------- append

def _append_case(dtype, qkv_dtype, qh, kvh, hd, page, rows, pad, seed, max_pos=500, scale=1.5):
    """rows: (position, slot) of each row."""
    r = np.random.default_rng(seed)
    T = len(rows) + pad
    slots = np.array([x[1] for x in rows] + [3] * pad, np.uint32)
    positions = np.array([x[0] for x in rows] + [1] * pad, np.uint32)
    pages = 23
    w = qh + 2 * kvh
    qkv = O.to_bits(qkv_dtype, r.standard_normal((T, w * hd)) * scale)
    qn, kn = (O.to_bits(BF16, 1 + 0.2 * r.standard_normal(hd)) for _ in range(2))
    ang = np.arange(max_pos)[:, None] * 1e4 ** (-np.arange(0, hd, 2) / hd)[None]
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    kc, vc = (O.to_bits(dtype, r.standard_normal(n)) for n in ((pages, kvh, page, hd), (pages, kvh, page // 8, hd, 8)))
    q0 = np.full((T, qh * hd), POISON_16, np.uint16)
    starts = np.array([0, len(rows) // 2, len(rows)], np.uint32)
    s = Session({"qkv": (qkv_dtype, qkv.shape, RO, qkv), "q_norm": (BF16, (hd,), RO, qn), "k_norm": (BF16, (hd,), RO, kn),
                 "cos_table": (F32, cos.shape, RO, cos), "sin_table": (F32, sin.shape, RO, sin),
                 "starts": (U32, (3,), 0, starts), "positions": (U32, (T,), 0, positions), "slots": (U32, (T,), 0, slots),
                 "q": (dtype, q0.shape, 0, q0), "k_cache": (dtype, kc.shape, 0, kc), "v_cache": (dtype, _rank4(vc), 0, vc)})
    try:
        cl = s.backend.begin()
        cl.dispatch("qk_norm_rope_append_paged", s.fields(
            "qk_norm_rope_append_paged", **{n: n for n in s.spec}, requests=2, tokens=T, q_heads=qh, kv_heads=kvh,
            head_dim=hd, max_pos=max_pos, page=page, pages=pages, eps=1e-6))
        s.backend.wait(s.backend.submit(cl))
        cl.release()
        gq, gk, gv = s.read("q"), s.read("k_cache"), s.read("v_cache").reshape(vc.shape)
    finally:
        s.close()
    f = O.from_bits
    q, k, v, bq, bk = O.append(f(qkv_dtype, qkv), f(BF16, qn), f(BF16, kn), cos.astype(np.float64), sin.astype(np.float64),
                               positions, slots, len(rows), qh, kvh, hd, page, pages, max_pos, 1e-6, np.zeros(q0.shape),
                               f(dtype, kc), f(dtype, vc))
    u = O.EPS_HALF[dtype]
    # float32's error, its rounding to the type, the type's smallest step
    assert np.all(np.abs(f(dtype, gq)[:len(rows)] - q[:len(rows)]) <= (bq + u * np.abs(q) + 2.0 ** -25)[:len(rows)])
    assert np.all(gq[len(rows):] == POISON_16)
    assert np.all(np.abs(f(dtype, gk) - k) <= bk + u * np.abs(k) + 2.0 ** -25)
    assert np.all((gk == kc) | (bk > 0))  # nothing else was touched
    assert np.array_equal(gv, O.to_bits(dtype, v))  # rounded once: every bit


def _rows(*runs):
    """(position, slot) rows of runs (first position, first slot, count)."""
    return [(p + i, s + i) for p, s, n in runs for i in range(n)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("qh,kvh,hd", [(16, 8, 128), (4, 4, 64), (7, 1, 128), (14, 2, 64), (1, 1, 64), (32, 8, 128)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_append_heads(dtype, qh, kvh, hd, page):
    rows = _rows((0, page * 3, 1), (40, page * 5 + 9, 7), (7, page * 2 + 8, 8), (130, page * 20 + 3, page - 3), (300, 0, 5))
    for qkv in (F32, DT[dtype]):
        _append_case(DT[dtype], qkv, qh, kvh, hd, page, rows, 3, seed=qh + hd)


@pytest.mark.parametrize("run", [(0, 1), (0, 8), (0, 16), (1, 16), (5, 3), (5, 4), (7, 1), (7, 2), (7, 9), (8, 15), (3, 61), (0, 64),
                                 (0, 65), (13, 128), (1, 300)])
def test_append_runs(run):
    """Runs of slots that begin and end anywhere in the values' tiles of 8 and in the rows that a workgroup takes."""
    off, n = run
    for qkv in (F32, F16):
        _append_case(F16, qkv, 4, 2, 128, 32, _rows((off, 32 * 4 + off, n), (9, 32 * 20 + 1, 1), (2, 5, 40)), 2, seed=n)


def test_append_rows_without_a_slot():
    """No slot, a slot past the cache, slots backwards and with gaps, a position past the tables: the q row is written (zeros
    without a rotation), the caches only where there is a place."""
    rows = [(5, PAGED_NONE), (6, 23 * 16), (7, 23 * 16 - 1), (8, 40), (9, 39), (10, 38), (11, 37), (12, 36), (13, 35), (14, 34),
            (15, 33), (16, 32), (20, 48), (21, 49), (22, 50), (23, PAGED_NONE), (24, 52), (25, 53), (26, 54), (27, 55),
            (499, 100), (500, 101), (4000000000, 102), (3, 104)]
    for dtype in (F16, BF16):
        _append_case(dtype, F32, 4, 2, 128, 16, rows, 1, seed=9)


@pytest.mark.parametrize("T", [4095, 4096, 4097])
@pytest.mark.parametrize("dtype,qkv,qh,kvh,hd", [("f16", "f32", 16, 8, 128), ("bf16", "bf16", 14, 2, 64), ("f16", "f16", 1, 1, 64)])
def test_append_thousands_of_rows(T, dtype, qkv, qh, kvh, hd):
    """On both sides of the rows from which a wave takes a row's heads whole."""
    rows = _rows((0, 256, 2000), (5, 256 * 9 + 3, 1001), (0, 256 * 14, 256), (40, 256 * 16 + 77, 800))
    rows += [(i, 1 + 7 * i) for i in range(T - 3 - len(rows))]
    assert len({slot for _, slot in rows}) == len(rows)
    _append_case(DT[dtype], F32 if qkv == "f32" else DT[qkv], qh, kvh, hd, 256, rows, 3, seed=T, max_pos=2100)


def test_append_more_workgroups_than_a_grid_row():
    """240,001 rows take 67,502 workgroups, more than the 65,535 of a grid's row."""
    r = np.random.default_rng(40)
    T, hd, page, pages, MP = 240001, 64, 256, 940, 512
    qkv = r.standard_normal((T, 3 * hd)).astype(np.float16)
    ang = np.arange(MP)[:, None] * 1e4 ** (-np.arange(0, hd, 2) / hd)[None]
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qn, kn = (O.to_bits(BF16, 1 + 0.2 * r.standard_normal(hd)) for _ in range(2))
    slots, positions = np.arange(T) + 7, np.arange(T) % MP
    slots[100000:] = np.concatenate([r.permutation(slots[100000:150000]), slots[150000:]])
    kc, vc = (np.full(n, POISON_16, np.uint16) for n in ((pages, 1, page, hd), (pages, 1, page // 8, hd, 8)))
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    s = Session({"qkv": (F16, qkv.shape, RO, qkv), "q_norm": (BF16, (hd,), RO, qn), "k_norm": (BF16, (hd,), RO, kn),
                 "cos_table": (F32, cos.shape, RO, cos), "sin_table": (F32, sin.shape, RO, sin), "starts": u([0, T - 2]),
                 "positions": u(positions), "slots": u(slots), "q": (F16, (T, hd), 0, None), "k_cache": (F16, kc.shape, 0, kc),
                 "v_cache": (F16, _rank4(vc), 0, vc)})
    try:
        got = s.run("qk_norm_rope_append_paged", ["q"], **{n: n for n in s.spec}, requests=1, tokens=T, q_heads=1, kv_heads=1,
                    head_dim=hd, max_pos=MP, page=page, pages=pages, eps=1e-6)
        gk, gv = s.read("k_cache").reshape(-1, hd), s.read("v_cache").reshape(-1, hd, 8)
    finally:
        s.close()
    x = qkv.astype(np.float64).reshape(T, 3, hd)
    w = np.stack([O.from_bits(BF16, qn), O.from_bits(BF16, kn)])
    h = w * x[:, :2] / np.sqrt((x[:, :2] ** 2).mean(2, keepdims=True) + 1e-6)
    a, b, c, d = h[..., :hd // 2], h[..., hd // 2:], cos[positions][:, None], sin[positions][:, None]
    want = np.concatenate([a * c - b * d, b * c + a * d], 2)
    # (the bound of paged_oracle.append, half a step of fp16 and its smallest)
    bound = np.tile(np.abs(a) + np.abs(b), 2) * 16 * O.U24 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    mine, at = np.arange(T) < T - 2, slots[:T - 2]
    f = O.from_bits
    assert np.all(np.abs(f(F16, got["q"]) - want[:, 0])[mine] <= bound[:, 0][mine]) and np.all(got["q"][~mine] == POISON_16)
    assert np.all(np.abs(f(F16, gk[at]) - want[mine, 1]) <= bound[mine, 1])
    assert np.array_equal(gv[at // 8, :, at % 8], qkv.view(np.uint16).reshape(T, 3, hd)[mine, 2])
    rest = np.setdiff1d(np.arange(pages * page), at)
    assert np.all(gk[rest] == POISON_16) and np.all(gv[rest // 8, :, rest % 8] == POISON_16)


def test_append_no_rows():
    for pad in (1, 70):
        _append_case(F16, F32, 4, 2, 128, 16, [], pad, seed=10)


def test_append_extreme_values():
    """Heads whose squares are small next to eps, and large ones whose values overflow fp16 (infinities, as IEEE narrowing)."""
    _append_case(BF16, F32, 4, 2, 64, 16, _rows((0, 16, 20)), 0, seed=12, scale=1e-6)
    _append_case(BF16, F32, 4, 2, 64, 16, _rows((0, 16, 20)), 0, seed=13, scale=3e5)


# ---------------------------------------------------------------- attention

def _attn_case(dtype, qh, kvh, hd, page, lens, *, pad=0, max_fresh=0, context=None, spoil=None, std=1.0, seed=0, spare=3,
               scale=None, values=None, twice=True, check=True):
    """lens: (cached, new) of each request. Every position that no request may read (spare pages, the end of the last page)
    holds NaN. spoil(table, pages): changes the table's entries. values(q, kc, vc, table): changes the inputs."""
    r = np.random.default_rng([seed, len(lens), hd, qh])
    past, fresh = (np.array(x, np.int64) for x in zip(*lens))
    end = past + fresh
    ctx = end if context is None else np.array(context, np.int64)
    R, total = len(lens), int(fresh.sum())
    T = total + pad
    assert T >= 1
    need = -(-np.minimum(np.maximum(end, ctx), end.max() + 40) // page)
    blocks, pages = max(1, int(need.max())) + 1, int(need.sum()) + spare
    ids, table, at = r.permutation(pages), np.full((R, blocks), PAGED_NONE, np.uint32), 0
    kc, vc = np.full((pages, kvh, page, hd), np.nan), np.full((pages, kvh, page // 8, hd, 8), np.nan)
    for i in range(R):
        table[i, :need[i]] = ids[at:at + need[i]]
        at += need[i]
        pos = np.arange(min(ctx[i], need[i] * page))
        pid = table[i, pos // page]
        kc[pid, :, pos % page] = r.standard_normal((len(pos), kvh, hd)) * std
        vc[pid, :, (pos % page) // 8, :, pos % 8] = r.standard_normal((len(pos), kvh, hd))
    if spoil:
        spoil(table, pages)
    starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.uint32)
    q = r.standard_normal((T, qh * hd)) * std
    q[total:] = np.nan
    if values:
        values(q, kc, vc, table)
    f, b = O.from_bits, O.to_bits
    qb, kb, vb = b(dtype, q), b(dtype, kc), b(dtype, vc)
    y0 = np.full((T, qh * hd), POISON_16, np.uint16)
    words = attention_paged_workspace_words(R, T, qh, kvh, hd)
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    s = Session({"q": (dtype, qb.shape, RO, qb), "k_cache": (dtype, kb.shape, RO, kb), "v_cache": (dtype, _rank4(vb), RO, vb),
                 "table": u(table), "starts": u(starts), "context": u(ctx), "y": (dtype, y0.shape, 0, y0),
                 "workspace": u(np.zeros(words))})
    sc = hd ** -0.5 if scale is None else scale
    runs = []
    try:
        for _ in range(2 if twice else 1):
            s.write("y", y0)
            cl = s.backend.begin()
            cl.dispatch("attention_paged", s.fields(
                "attention_paged", **{n: n for n in s.spec}, requests=R, tokens=T, max_fresh=max_fresh, q_heads=qh,
                kv_heads=kvh, head_dim=hd, blocks=blocks, page=page, pages=pages, scale=sc))
            s.backend.wait(s.backend.submit(cl))
            cl.release()
            runs.append(s.read("y"))
    finally:
        s.close()
    assert all(x.tobytes() == runs[0].tobytes() for x in runs)
    if not check:
        return f(dtype, runs[0])
    want, bound = O.attention(f(dtype, qb), f(dtype, kb), f(dtype, vb), table, starts, ctx, qh, kvh, hd, page, pages, blocks, T,
                              max_fresh or T, float(np.float32(sc)), dtype, np.zeros(y0.shape))
    mine = bound >= 0
    got = f(dtype, runs[0])
    off = np.abs(got - want)
    bad = mine & ~((off <= bound) | (np.isnan(got) & np.isnan(want)) | (got == want))
    assert not bad.any(), (np.argwhere(bad)[:5], off[bad][:5], bound[bad][:5], got[bad][:5], want[bad][:5])
    assert np.all(runs[0][~mine] == POISON_16)  # rows behind the last sequence, and rows past max_fresh
    return got


HEADS = [(16, 8, 128), (4, 4, 64), (8, 1, 128), (14, 2, 64), (6, 2, 128), (40, 1, 64), (1, 1, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("qh,kvh,hd", HEADS)
def test_attention_single_tokens(dtype, qh, kvh, hd):
    """One token each over contexts on both sides of every tile, page and split border."""
    lens = [(n, 1) for n in (0, 1, 7, 14, 15, 16, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128, 129, 255, 256, 400, 777)]
    _attn_case(DT[dtype], qh, kvh, hd, 16, lens, pad=2, max_fresh=1)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_pages(page, hd):
    lens = [(300, 1), (0, 5), (page - 1, 2), (page, 1), (2 * page - 3, 40), (11, 0), (500, 3)]
    for dtype in (F16, BF16):
        _attn_case(dtype, 4, 2, hd, page, lens, pad=1)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("qh,kvh,hd", HEADS)
def test_attention_chunks(dtype, qh, kvh, hd):
    lens = [(0, 1), (0, 2), (0, 70), (33, 17), (100, 64), (63, 65), (250, 130), (5, 31), (0, 0), (129, 1)]
    _attn_case(DT[dtype], qh, kvh, hd, 32, lens, pad=3)


@pytest.mark.parametrize("n", [1, 2, 3, 8, 9, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 96, 127, 128, 129, 200, 255, 256, 257])
def test_attention_chunk_lengths(n):
    _attn_case(F16, 4, 2, 128, 16, [(0, n)])
    _attn_case(BF16, 2, 2, 64, 64, [(77, n), (n, 1)])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_long_context(dtype):
    """One token over 20,011 keys, then with seven others: many splits of one row joined, and few."""
    _attn_case(DT[dtype], 4, 2, 128, 16, [(20010, 1)], max_fresh=1)
    _attn_case(DT[dtype], 4, 2, 64, 64, [(9000, 1), (5, 1), (0, 1), (700, 1), (2047, 1), (2048, 1), (4000, 1), (64, 1)])


def test_attention_many_requests():
    r = np.random.default_rng(3)
    _attn_case(F16, 2, 1, 64, 16, [(int(x), 1) for x in r.integers(0, 90, 700)], max_fresh=1)
    _attn_case(BF16, 2, 1, 64, 16, [(int(x), int(f)) for x, f in zip(r.integers(0, 40, 300), r.integers(0, 4, 300))])


@pytest.mark.parametrize("requests", [1, 4096])
def test_attention_request_limits(requests):
    _attn_case(F16, 1, 1, 64, 16, [(i % 5, i % 2) for i in range(1, requests + 1)], pad=1)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("qh,kvh,hd", [(16, 8, 128), (14, 2, 64), (200, 1, 64), (130, 1, 128), (24, 2, 128)])
def test_attention_mixed_batches(dtype, qh, kvh, hd):
    """Single tokens and chunks together: most requests with one row, of very different contexts, none that has rows first and
    last."""
    r = np.random.default_rng(12)
    lens = [(30, 0)] + [(int(x), 1) for x in r.integers(0, 1500, 17)] + [(700, 90), (0, 40), (0, 0), (1000, 33), (64, 0)]
    _attn_case(DT[dtype], qh, kvh, hd, 16, lens, pad=5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("qh,kvh,hd", [(16, 8, 128), (12, 12, 64), (32, 8, 128)])
def test_attention_many_items(dtype, qh, kvh, hd):
    """More items than workgroups: pieces of several, the parts of others, requests without rows between them."""
    r = np.random.default_rng(13)
    lens = [(int(x), int(f)) for x, f in zip(r.integers(0, 700, 90), r.choice([0, 1, 1, 1, 2, 20], 90))] + [(300, 150), (1400, 40)]
    _attn_case(DT[dtype], qh, kvh, hd, 32, lens, pad=2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("qh,kvh,hd", [(16, 8, 128), (32, 8, 128), (4, 4, 64)])
@pytest.mark.parametrize("batch", ["own", "uneven", "many"])
def test_attention_mixed_batches_in_wide_tables(dtype, qh, kvh, hd, batch):
    """Batches of at least 16 requests that bring few rows each, in tables of more than 2048 positions (a launch of its own joins
    the split items): workgroups of their own per item, too few of them for the long ones, and more items than workgroups."""
    r = np.random.default_rng(14)
    single = lambda n, top: [(int(x), 1) for x in r.integers(0, top, n)]  # noqa: E731
    lens = {"own": single(17, 1500) + [(2200, 40), (0, 70), (1000, 5)],
            "uneven": single(57, 60) + [(4000, 30), (2900, 17), (3100, 2)],
            "many": single(40, 500) + [(30, 0), (2300, 33)] + single(40, 300) + [(0, 0), (70, 90)]}[batch]
    _attn_case(DT[dtype], qh, kvh, hd, 32, lens, pad=4)


@pytest.mark.parametrize("qh,kvh,hd", [(256, 1, 64), (100, 1, 128), (34, 2, 64), (17, 1, 128)])
def test_attention_large_groups(qh, kvh, hd):
    """Query heads per KV head that fill a tile with one row, leave columns over, and just miss the form for few."""
    _attn_case(F16, qh, kvh, hd, 16, [(50, 1), (0, 5), (130, 3)], pad=1)
    _attn_case(BF16, qh, kvh, hd, 32, [(70, 1), (0, 1)], max_fresh=1)


@pytest.mark.parametrize("short", [9, 24])
def test_attention_uneven_requests(short):
    """Few items of very different lengths: with workgroups of their own each, and with too few left for the long ones."""
    _attn_case(F16, 8, 8, 64, 32, [(3 * i, 2) for i in range(short)] + [(4000, 30), (3900, 17), (4100, 1)], pad=3)


def test_attention_rows_without_keys():
    """A context shorter than the new rows: the first of them see nothing and give zeros; a request with no context; a
    context past the table."""
    lens = [(0, 9), (3, 1), (40, 30), (0, 1), (16, 2)]
    for dtype in (F16, BF16):
        y = _attn_case(dtype, 4, 2, 128, 16, lens, context=[4, 0, 25, 1, 0xFFFFFFF0], pad=1)
        assert np.all(y[:5] == 0) and np.all(y[9] == 0)


def test_attention_no_rows():
    _attn_case(F16, 4, 2, 64, 16, [(0, 0), (30, 0)], pad=3)


def test_attention_max_fresh():
    """Rows of a request past max_fresh are left as they were; those before it see the keys of their places."""
    for most in (1, 2, 16, 64):
        _attn_case(F16, 4, 2, 128, 16, [(20, 1), (0, 90), (33, 2), (5, 70)], max_fresh=most, pad=2)


def test_attention_pages_that_are_none():
    """Entries without a page, or past the cache, hide their keys; a request with no page at all gives zeros."""
    def spoil(table, pages):
        table[0, 1] = PAGED_NONE
        table[1, 0] = pages
        table[2, 2] = PAGED_NONE - 1
        table[3, :] = PAGED_NONE
        table[4, 3] = 0x80000000
    for dtype in (F16, BF16):
        for fresh in (1, 40):
            _attn_case(dtype, 4, 2, 64, 16, [(60, fresh), (60, fresh), (70, fresh), (20, fresh), (100, fresh)], spoil=spoil)


def test_attention_shared_pages():
    """Two requests over the same pages (a shared prefix): the same row of both gives the same bits."""
    def values(q, kc, vc, table):
        table[1] = table[0]
        q[1] = q[0]
    for ctx in (100, 700):
        y = _attn_case(F16, 16, 8, 128, 16, [(ctx, 1), (ctx, 1)], values=values, max_fresh=1)
        assert y[0].tobytes() == y[1].tobytes()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fresh", [1, 3, 90])
def test_attention_scores(dtype, fresh):
    """Scores in the hundreds, a maximum that rises in every tile, one key that outweighs the others first or last, equal
    ones."""
    lens = [(300, fresh), (0, fresh), (130, fresh)]

    def rising(q, kc, vc, table):
        q[:], kc[~np.isnan(kc)] = 1.0, 0.0
        for i, (p, f) in enumerate(lens):
            pos = np.arange(p + f)
            kc[table[i, pos // 16], :, pos % 16] = (pos / 64.0)[:, None, None]

    def dominant(at):
        def change(q, kc, vc, table):
            q[:] = 2.0
            for i, (p, f) in enumerate(lens):
                pos = (p + f - 1) if at < 0 else 0
                kc[table[i, pos // 16], :, pos % 16] = 4.0
        return change

    def equal(q, kc, vc, table):
        q[:] = 0.0

    d = DT[dtype]
    _attn_case(d, 4, 2, 128, 16, lens, std=6.0, seed=1)
    for change in (rising, dominant(0), dominant(-1), equal):
        _attn_case(d, 4, 2, 128, 16, lens, values=change)
    _attn_case(d, 4, 2, 64, 16, lens, scale=30.0, seed=2)
    _attn_case(d, 4, 2, 64, 16, lens, scale=1e-4, seed=2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [[(40, 2), (0, 3), (130, 4)], [(300, 90), (0, 77), (63, 5)], [(1900, 129), (5, 20)],
                                  [(100, 200)] * 40, [(500, 1)] * 17 + [(40, 90), (700, 150)]],
                         ids=["few", "chunks", "long", "many", "mixed"])
def test_attention_values_that_are_not_finite(dtype, hd, lens):
    """Infinities and NaN among a chunk's own values reach the rows that see them, in their dim of their head, and change no
    bit of any other row: what a row gives does not depend on the tokens after it."""
    qh, kvh, page, at = 4, 2, 16, []
    r = np.random.default_rng(5)
    for i, (past, new) in enumerate(lens):
        for j in {0, 1, new // 2, new - 1}:
            for x in (np.inf, -np.inf, np.nan):
                at.append((i, past + j, int(r.integers(kvh)), int(r.integers(hd)), x))
        at.append((i, past + new - 1, 0, at[-1][3], np.inf))

    def put(odd):
        def change(q, kc, vc, table):
            for i, pos, h, d, x in at:
                vc[table[i, pos // page], h, pos % page // 8, d, pos % 8] = x if odd else 0.0
        return change

    d = DT[dtype]
    plain = _attn_case(d, qh, kvh, hd, page, lens, std=0.3, values=put(False), twice=False)
    got = _attn_case(d, qh, kvh, hd, page, lens, std=0.3, values=put(True), check=False)
    add = np.zeros(plain.shape)
    first = np.concatenate([[0], np.cumsum([n for _, n in lens])])
    last = {(i, pos, h, dim): x for i, pos, h, dim, x in at}  # (a later entry takes the place of an earlier one)
    with np.errstate(invalid="ignore"):
        for (i, pos, h, dim), x in last.items():
            for g in range(2 * h, 2 * h + 2):
                add[first[i] + pos - lens[i][0]:first[i + 1], g * hd + dim] += x
    want = np.where(add == 0, plain, add)
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | (np.isnan(got) & np.isnan(want))))[:5]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[(40, 2), (0, 3), (130, 4)], [(300, 90), (0, 77), (1900, 129)]], ids=["few", "chunks"])
@pytest.mark.parametrize("x", [np.nan, np.inf])
def test_attention_keys_that_are_not_finite(dtype, lens, x):
    """A chunk's last key, if it is NaN or infinite, changes no bit of the rows before it."""
    def put(x):
        def change(q, kc, vc, table):
            for i, (past, new) in enumerate(lens):
                pos = past + new - 1
                kc[table[i, pos // 16], :, pos % 16] = x
        return change

    d = DT[dtype]
    plain = _attn_case(d, 4, 2, 128, 16, lens, values=put(0.0), twice=False)
    got = _attn_case(d, 4, 2, 128, 16, lens, values=put(x), check=False)
    ends = np.cumsum([n for _, n in lens])
    before = np.setdiff1d(np.arange(ends[-1]), ends - 1)
    assert np.array_equal(got[before], plain[before])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fresh", [1, 20])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_many_small_weights(dtype, fresh, hd):
    """A few keys that outweigh all others, with values of zero, before tens of thousands of weights of 2^-25 (in fp16 half of its
    smallest step) whose values alone make the result: none may be lost to the type's underflow. So many requests over the
    same pages that a workgroup has whole contexts."""
    page, blocks, R, d = 64, 1000, 600 // fresh, DT[dtype]
    n = blocks * page
    k, v = np.zeros((n, hd)), np.full((n, hd), 1000.0)
    top = 25.4 * np.log(2)
    k[:512:32], v[:512:32] = 2.0, 0.0  # (every wave's first keys)
    q = np.full((R * fresh, hd), 0.5)
    sc = top / hd  # the score of the large keys is hd * sc, of the others 0
    kb, vb = O.to_bits(d, k.reshape(blocks, 1, page, hd)), O.to_bits(d, v.reshape(blocks, 1, page // 8, 8, hd).swapaxes(3, 4))
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    s = Session({"q": (d, q.shape, RO, O.to_bits(d, q)), "k_cache": (d, kb.shape, RO, kb), "v_cache": (d, _rank4(vb), RO, vb),
                 "table": u(np.tile(np.arange(blocks), (R, 1))), "starts": u(np.arange(R + 1) * fresh),
                 "context": u(np.full(R, n)), "y": (d, q.shape, 0, None),
                 "workspace": u(np.zeros(attention_paged_workspace_words(R, R * fresh, 1, 1, hd)))})
    try:
        y = O.from_bits(d, s.run("attention_paged", ["y"], **{m: m for m in s.spec}, requests=R, tokens=R * fresh,
                                 max_fresh=fresh, q_heads=1, kv_heads=1, head_dim=hd, blocks=blocks, page=page, pages=blocks,
                                 scale=sc)["y"])
    finally:
        s.close()
    seen = n - fresh + 1 + np.tile(np.arange(fresh), R)
    small = np.exp(-hd * float(np.float32(sc)))
    want = (1000 * (seen - 16) * small / (16 + (seen - 16) * small))[:, None]
    # a score's float32 error (its product, the scale, the reference), a weight's rounding and the result's to the type, the float32
    # sums over the keys, and the weights that may still fall below the type's smallest step: in fp16 2^-32 of the largest each
    rel = 2 * O.EPS_HALF[d] + 2 * (hd + 8) * O.U24 * top + (n + 16) * O.U24
    tiny = 1000 * n * 2.0 ** -32 / 16 if d == F16 else 0.0
    assert np.all(np.abs(y - want) <= rel * want + tiny), (np.abs(y - want).max(), want.max())


@pytest.mark.parametrize("fresh,blocks", [(1, 4), (1, 40), (2, 40), (9, 40), (40, 30)])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_values_at_the_end_of_fp16(hd, fresh, blocks):
    """Values of +-65,504 at every key: the result is that value whatever the weights, never an infinity, though the rounded
    weights may be 2^-11 more than their sum (half of that passes fp16's last step). The first keys score less, so that the
    reference stays at theirs and the other weights are no powers of two."""
    page, R, group = 64, 1200 if fresh < 9 else 300, 16
    n, r = blocks * page, np.random.default_rng(31)
    k = np.full((n, hd), 4.0 / hd)
    k[:128] = 0.0
    end = np.where(np.arange(hd) % 3 == 0, -65504.0, 65504.0)
    q = np.abs(r.standard_normal((R * fresh, group * hd))) * 1.2  # (scores of 3 to 5 in the exponent's powers of two)
    b = lambda a: O.to_bits(F16, a)  # noqa: E731
    kb, vb = b(k.reshape(blocks, 1, page, hd)), b(np.tile(end[None, None, None, :, None], (blocks, 1, page // 8, 1, 8)))
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    s = Session({"q": (F16, q.shape, RO, b(q)), "k_cache": (F16, kb.shape, RO, kb), "v_cache": (F16, _rank4(vb), RO, vb),
                 "table": u(np.tile(np.arange(blocks), (R, 1))), "starts": u(np.arange(R + 1) * fresh),
                 "context": u(np.full(R, n)), "y": (F16, q.shape, 0, None),
                 "workspace": u(np.zeros(attention_paged_workspace_words(R, R * fresh, group, 1, hd)))})
    try:
        y = O.from_bits(F16, s.run("attention_paged", ["y"], **{m: m for m in s.spec}, requests=R, tokens=R * fresh,
                                   max_fresh=fresh, q_heads=group, kv_heads=1, head_dim=hd, blocks=blocks, page=page,
                                   pages=blocks, scale=1.0)["y"])
    finally:
        s.close()
    # a weight's rounding, the float32 sums over the keys, the result's rounding to a step of 32
    bound = 65504 * (2.0 ** -11 + 2 * (n + 16) * O.U24) + 16
    assert np.all(np.abs(y - np.tile(end, group)) <= bound), np.unique(y)


def test_attention_replayed_with_other_lengths():
    """One recorded list, replayed as the lengths, the table and the queries on the device change, with the shorter and the
    longer in either order: a launch leaves nothing in the workspace that the next could take for its own."""
    r = np.random.default_rng(8)
    qh, kvh, hd, page, pages, blocks, R, T = 4, 2, 128, 16, 400, 130, 6, 90
    kb, vb = O.to_bits(F16, r.standard_normal((pages, kvh, page, hd))), O.to_bits(F16, r.standard_normal((pages, kvh, page // 8, hd, 8)))
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    s = Session({"q": (F16, (T, qh * hd), 0, None), "k_cache": (F16, kb.shape, RO, kb), "v_cache": (F16, _rank4(vb), RO, vb),
                 "table": u(np.zeros((R, blocks))), "starts": u(np.zeros(R + 1)), "context": u(np.zeros(R)),
                 "y": (F16, (T, qh * hd), 0, None), "workspace": u(np.zeros(attention_paged_workspace_words(R, T, qh, kvh, hd)))})
    cl = s.backend.begin(reusable=True)
    try:
        cl.dispatch("attention_paged", s.fields(
            "attention_paged", **{n: n for n in s.spec}, requests=R, tokens=T, max_fresh=0, q_heads=qh, kv_heads=kvh, head_dim=hd,
            blocks=blocks, page=page, pages=pages, scale=hd ** -0.5))
        for lens in ([(2000, 1)] * 6, [(5, 1), (0, 80), (3, 0), (1, 1), (900, 4), (17, 3)], [(0, 1)] * 6, [(1500, 60), (0, 0)] * 3,
                     [(2000, 1)] * 6):
            lens = [(p, min(f, T // 6 if len(set(lens)) < 3 else f)) for p, f in lens]
            past, fresh = (np.array(x) for x in zip(*lens))
            starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.uint32)
            table = r.integers(0, pages, (R, blocks)).astype(np.uint32)
            qb = O.to_bits(F16, r.standard_normal((T, qh * hd)))
            for n, a in (("q", qb), ("table", table), ("starts", starts), ("context", (past + fresh).astype(np.uint32)),
                         ("y", s.poison("y"))):
                s.write(n, a)
            s.backend.wait(s.backend.submit(cl))
            y = s.read("y")
            want, bound = O.attention(O.from_bits(F16, qb), O.from_bits(F16, kb), O.from_bits(F16, vb), table, starts, past + fresh,
                                      qh, kvh, hd, page, pages, blocks, T, T, float(np.float32(hd ** -0.5)), F16,
                                      np.zeros((T, qh * hd)))
            mine = bound >= 0
            assert np.all((np.abs(O.from_bits(F16, y) - want) <= bound)[mine]), lens
            assert np.all(y[~mine] == POISON_16)
    finally:
        cl.release()
        s.close()


@pytest.mark.parametrize("hd,wide", [(128, 0), (64, 0), (128, 200)])
def test_attention_starts_that_decrease(hd, wide):
    """Starts that decrease somewhere (requests whose rows would overlap) compute nothing, in either form and however split
    items are joined; the next dispatch with good ones finds the workspace as it has to be."""
    qh, kvh, page, R, T = 4, 2, 16, 300, 90
    r = np.random.default_rng(17)
    past, fresh = r.integers(0, 60, R), np.zeros(R, np.int64)
    fresh[r.permutation(R)[:45]] = 2
    blocks, pages = 5 + wide, 99
    good = np.concatenate([[0], np.cumsum(fresh)]).astype(np.uint32)
    kb, vb = O.to_bits(F16, r.standard_normal((pages, kvh, page, hd))), O.to_bits(F16, r.standard_normal((pages, kvh, page // 8, hd, 8)))
    qb = O.to_bits(F16, r.standard_normal((T, qh * hd)))
    table = r.integers(0, pages, (R, blocks)).astype(np.uint32)
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    words = attention_paged_workspace_words(R, T, qh, kvh, hd)
    s = Session({"q": (F16, qb.shape, RO, qb), "k_cache": (F16, kb.shape, RO, kb), "v_cache": (F16, _rank4(vb), RO, vb),
                 "table": u(table), "starts": u(good), "context": u(past + fresh), "y": (F16, qb.shape, 0, None),
                 "workspace": u(np.zeros(words))})
    f = O.from_bits
    want, bound = O.attention(f(F16, qb), f(F16, kb), f(F16, vb), table, good, past + fresh, qh, kvh, hd, page, pages, blocks, T, T,
                              float(np.float32(hd ** -0.5)), F16, np.zeros(qb.shape))

    def run(starts, most):
        s.write("starts", starts.astype(np.uint32))
        s.write("y", s.poison("y"))
        cl = s.backend.begin()
        cl.dispatch("attention_paged", s.fields(
            "attention_paged", **{n: n for n in s.spec}, requests=R, tokens=T, max_fresh=most, q_heads=qh, kv_heads=kvh,
            head_dim=hd, blocks=blocks, page=page, pages=pages, scale=hd ** -0.5))
        s.backend.wait(s.backend.submit(cl))
        cl.release()
        return s.read("y")

    turns = np.zeros(R + 1, np.int64)
    turns[1::2] = T
    last, first = good.copy(), good.copy()
    last[R] = T - 1 - last[R] % 2
    last[R - 1] = T
    first[0] = 1
    first[1] = 0
    far = np.where(np.arange(R + 1) == 7, 0xFFFFFFFF, good)
    try:
        for most in (2, 0):
            for starts in (turns, turns[::-1], last, first, far):
                assert np.all(run(starts, most) == POISON_16)
            assert np.all(s.read("workspace")[:512] == 0)
            y = run(good, most)
            assert np.all((np.abs(f(F16, y) - want) <= bound)[bound >= 0]) and np.all(y[bound < 0] == POISON_16)
    finally:
        s.close()


def _batch(seed, lens, qh, kvh, hd, page, outputs, workspaces, tokens):
    """A session with one ragged batch in it and as many results and workspaces, and the dispatch's fields for each form."""
    r = np.random.default_rng(seed)
    past, fresh = (np.array(x) for x in zip(*lens))
    R, blocks = len(lens), int((past + fresh).max()) // page + 1
    pages = R * blocks
    kb, vb = O.to_bits(F16, r.standard_normal((pages, kvh, page, hd))), O.to_bits(F16, r.standard_normal((pages, kvh, page // 8, hd, 8)))
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    words = attention_paged_workspace_words(R, tokens, qh, kvh, hd)
    q = O.to_bits(F16, r.standard_normal((tokens, qh * hd)))
    s = Session({"q": (F16, q.shape, 0, q), "k_cache": (F16, kb.shape, RO, kb), "v_cache": (F16, _rank4(vb), RO, vb),
                 "table": u(r.permutation(pages).reshape(R, blocks)), "starts": u(np.concatenate([[0], np.cumsum(fresh)])),
                 "context": u(past + fresh), **{f"y{i}": (F16, q.shape, 0, None) for i in range(outputs)},
                 **{f"ws{i}": u(np.zeros(words)) for i in range(workspaces)}})
    common = ("q", "k_cache", "v_cache", "table", "starts", "context")

    def fields(y, ws, max_fresh):
        return s.fields("attention_paged", **{n: n for n in common}, y=y, workspace=ws, requests=R, tokens=tokens,
                        max_fresh=max_fresh, q_heads=qh, kv_heads=kvh, head_dim=hd, blocks=blocks, page=page, pages=pages,
                        scale=hd ** -0.5)
    return s, fields


def _eager(s, fields, *args):
    cl = s.backend.begin()
    cl.dispatch("attention_paged", fields(*args))
    s.backend.wait(s.backend.submit(cl))
    cl.release()
    return s.read(args[0])


@pytest.mark.parametrize("count", [2, 10])
def test_attention_forms_take_turns_in_one_workspace(count):
    """A reusable list of few dispatches (launched one by one) and of many (a captured graph) in which the form for single
    tokens and the tiles use one workspace in turn, replayed with eager work and other lists between: every replay gives the
    eager dispatch's bits."""
    lens = [(700, 1), (0, 1), (1500, 1), (63, 1), (64, 1), (2000, 1)]
    s, fields = _batch(3, lens, 4, 2, 128, 16, count, 1, 40)
    cl, other = s.backend.begin(reusable=True), s.backend.begin(reusable=True)
    try:
        want = [_eager(s, fields, "y0", "ws0", f) for f in (1, 0)]
        for i in range(count):
            cl.dispatch("attention_paged", fields(f"y{i}", "ws0", 1 - i % 2))
        other.dispatch("attention_paged", fields("y0", "ws0", 0))
        for replay in range(4):
            for i in range(count):
                s.write(f"y{i}", s.poison(f"y{i}"))
            s.backend.wait(s.backend.submit(cl, repeat=1 + replay % 2))
            for i in range(count):
                assert s.read(f"y{i}").tobytes() == want[i % 2].tobytes(), (replay, i)
            s.backend.wait(s.backend.submit(other))
            assert s.read("y0").tobytes() == want[1].tobytes()
    finally:
        cl.release()
        other.release()
        s.close()


@pytest.mark.parametrize("first,second", [(1, 1), (1, 0), (0, 0)])
def test_attention_overlapped(first, second):
    """Two dispatches that may run at once, each with a workspace of its own."""
    s, fields = _batch(4, [(1200, 1), (300, 1), (5, 1)], 8, 4, 64, 32, 2, 2, 20)
    try:
        want = [_eager(s, fields, "y0", "ws0", f) for f in (first, second)]
        for _ in range(3):
            for n in ("y0", "y1"):
                s.write(n, s.poison(n))
            cl = s.backend.begin()
            cl.dispatch_overlapped("attention_paged", fields("y0", "ws0", first))
            cl.dispatch("attention_paged", fields("y1", "ws1", second))
            cl.barrier()
            s.backend.wait(s.backend.submit(cl))
            cl.release()
            assert [s.read(n).tobytes() for n in ("y0", "y1")] == [w.tobytes() for w in want]
    finally:
        s.close()


def test_attention_pages_missing_far_back():
    """Pages that are none in the middle of long contexts, in some groups of sixteen blocks and not in others."""
    def spoil(table, pages):
        r = np.random.default_rng(2)
        for i in range(len(table)):
            table[i, r.integers(0, 3000 // 16, 4)] = [PAGED_NONE, pages, pages + 7, PAGED_NONE]

    for lens in ([(3000, 40), (2900, 100)], [(3000, 1)] * 3 + [(2990, 2)]):
        _attn_case(F16, 4, 2, 128, 16, lens, spoil=spoil)
        _attn_case(BF16, 2, 2, 64, 16, lens, spoil=spoil)


def test_append_two_rows_of_one_slot():
    """Two rows that name one slot: each part of the entry is one row's or the other's, and nothing else changes."""
    r = np.random.default_rng(6)
    qh, kvh, hd, page, pages, T = 2, 2, 64, 16, 3, 4
    qkv = r.standard_normal((T, (qh + 2 * kvh) * hd)).astype(np.float32)
    ones, cos = O.to_bits(BF16, np.ones(hd)), np.ones((9, hd // 2), np.float32)
    kc, vc = (np.full(n, POISON_16, np.uint16) for n in ((pages, kvh, page, hd), (pages, kvh, page // 8, hd, 8)))
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    s = Session({"qkv": (F32, qkv.shape, RO, qkv), "q_norm": (BF16, (hd,), RO, ones), "k_norm": (BF16, (hd,), RO, ones),
                 "cos_table": (F32, cos.shape, RO, cos), "sin_table": (F32, cos.shape, RO, cos * 0), "starts": u([0, T]),
                 "positions": u([1, 2, 3, 4]), "slots": u([5, 21, 5, 21]), "q": (F16, (T, qh * hd), 0, None),
                 "k_cache": (F16, kc.shape, 0, kc), "v_cache": (F16, _rank4(vc), 0, vc)})
    try:
        cl = s.backend.begin()
        cl.dispatch("qk_norm_rope_append_paged", s.fields(
            "qk_norm_rope_append_paged", **{n: n for n in s.spec}, requests=1, tokens=T, q_heads=qh, kv_heads=kvh, head_dim=hd,
            max_pos=9, page=page, pages=pages, eps=0.0))
        s.backend.wait(s.backend.submit(cl))
        cl.release()
        gk, gv = s.read("k_cache"), s.read("v_cache").reshape(vc.shape)
    finally:
        s.close()
    x = qkv.reshape(T, qh + 2 * kvh, hd)
    v = O.to_bits(F16, x[:, qh + kvh:])
    k = x[:, qh:qh + kvh].astype(np.float64)
    k = k / np.sqrt((k * k).mean(-1, keepdims=True))
    touched_k, touched_v = np.zeros(kc.shape, bool), np.zeros(vc.shape, bool)
    for slot, rows in ((5, (0, 2)), (21, (1, 3))):
        at, off = divmod(slot, page)
        touched_k[at, :, off], touched_v[at, :, off // 8, :, off % 8] = True, True
        g = O.from_bits(F16, gk[at, :, off])
        # float32's sum of squares, root and products, then half a step of fp16
        assert np.all(np.min([np.abs(g - k[t]) - (2.0 ** -11 + 16 * O.U24) * np.abs(k[t]) for t in rows], axis=0) <= 2.0 ** -25)
        assert np.all((gv[at, :, off // 8, :, off % 8] == v[rows[0]]) | (gv[at, :, off // 8, :, off % 8] == v[rows[1]]))
    assert np.all(gk[~touched_k] == POISON_16) and np.all(gv[~touched_v] == POISON_16)


# ---------------------------------------------------------------- together

def test_a_serving_loop():
    """Four requests through plan, append and attention on one recorded list: their prompts, a chunk for two of them, single
    tokens, one that ends; each step's lengths are uploaded, everything else stays on the device. The queries' rows, both
    caches and the attention of each step against float64 on what the device's own cache holds."""
    r = np.random.default_rng(21)
    qh, kvh, hd, page, pages, blocks, R, T, MP = 4, 2, 64, 16, 60, 20, 4, 120, 320
    ang = np.arange(MP)[:, None] * 1e4 ** (-np.arange(0, hd, 2) / hd)[None]
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qn, kn = (O.to_bits(BF16, 1 + 0.2 * r.standard_normal(hd)) for _ in range(2))
    u = lambda a: (U32, np.shape(a), 0, np.asarray(a, np.uint32))  # noqa: E731
    half = lambda *shape: (F16, shape, 0, np.zeros(shape, np.uint16))  # noqa: E731
    s = Session({"past": u(np.zeros(R)), "fresh": u(np.zeros(R)), "free": u(np.zeros(pages)),
                 "table": u(np.full((R, blocks), PAGED_NONE)), "starts": u(np.zeros(R + 1)), "context": u(np.zeros(R)),
                 "positions": u(np.zeros(T)), "slots": u(np.zeros(T)), "counts": u(np.zeros(3)),
                 "qkv": (F32, (T, (qh + 2 * kvh) * hd), 0, None), "q_norm": (BF16, (hd,), RO, qn), "k_norm": (BF16, (hd,), RO, kn),
                 "cos_table": (F32, cos.shape, RO, cos), "sin_table": (F32, sin.shape, RO, sin), "q": half(T, qh * hd),
                 "k_cache": half(pages, kvh, page, hd), "v_cache": half(pages, kvh, page // 8, hd * 8), "y": half(T, qh * hd),
                 "workspace": u(np.zeros(attention_paged_workspace_words(R, T, qh, kvh, hd)))})
    free = r.permutation(pages).astype(np.uint32)
    cl = s.backend.begin(reusable=True)
    pick = lambda *names: {n: n for n in names}  # noqa: E731
    try:
        cl.dispatch("paged_plan", s.fields(
            "paged_plan", **pick("past", "fresh", "free", "table", "starts", "context", "positions", "slots", "counts"),
            requests=R, blocks=blocks, page=page, pages=pages, free_count=pages, tokens=T))
        cl.dispatch("qk_norm_rope_append_paged", s.fields(
            "qk_norm_rope_append_paged", **pick("qkv", "q_norm", "k_norm", "cos_table", "sin_table", "starts", "positions",
                                                "slots", "q", "k_cache", "v_cache"), requests=R, tokens=T, q_heads=qh,
            kv_heads=kvh, head_dim=hd, max_pos=MP, page=page, pages=pages, eps=1e-6))
        cl.dispatch("attention_paged", s.fields(
            "attention_paged", **pick("q", "k_cache", "v_cache", "table", "starts", "context", "y", "workspace"), requests=R,
            tokens=T, max_fresh=0, q_heads=qh, kv_heads=kvh, head_dim=hd, blocks=blocks, page=page, pages=pages,
            scale=hd ** -0.5))
        past = np.zeros(R, np.int64)
        table = np.full((R, blocks), PAGED_NONE, np.uint32)
        for fresh in ([17, 40, 1, 33], [1, 50, 1, 60], [1, 1, 1, 1], [1, 0, 1, 1], [2, 0, 90, 1]):
            fresh = np.array(fresh, np.int64)
            qkv = (r.standard_normal((T, (qh + 2 * kvh) * hd)) * 1.5).astype(np.float32)
            for n, a in (("past", past), ("fresh", fresh)):
                s.write(n, a.astype(np.uint32))
            s.write("free", np.concatenate([free, np.zeros(pages - len(free), np.uint32)]))
            s.write("qkv", qkv)
            k0, v0 = (O.from_bits(F16, s.read(n)) for n in ("k_cache", "v_cache"))
            v0 = v0.reshape(pages, kvh, page // 8, hd, 8)
            s.backend.wait(s.backend.submit(cl))
            g = {n: s.read(n) for n in ("table", "starts", "context", "positions", "slots", "counts", "q", "k_cache", "v_cache", "y")}
            g["v_cache"] = g["v_cache"].reshape(v0.shape)
            total = int(fresh.sum())
            want = O.plan(past, fresh, free, table, blocks, page, pages, T, g["positions"].copy(), g["slots"].copy())
            for n, w in zip(("table", "starts", "context", "positions", "slots", "counts"), want):
                assert np.array_equal(g[n], w), n
            table = want[0]
            q, k, v, bq, bk = O.append(qkv.astype(np.float64), O.from_bits(BF16, qn), O.from_bits(BF16, kn), cos.astype(np.float64),
                                       sin.astype(np.float64), want[3], want[4], total, qh, kvh, hd, page, pages, MP, 1e-6,
                                       np.zeros((T, qh * hd)), k0, v0)
            step = 2.0 ** -11
            gq, gk = O.from_bits(F16, g["q"]), O.from_bits(F16, g["k_cache"])
            assert np.all((np.abs(gq - q) <= bq + step * np.abs(q) + 2.0 ** -25)[:total])
            assert np.all(np.abs(gk - k) <= bk + step * np.abs(k) + 2.0 ** -25)
            assert np.array_equal(g["v_cache"], O.to_bits(F16, v))
            y, bound = O.attention(gq, gk, O.from_bits(F16, g["v_cache"]), table, want[1], want[2], qh, kvh, hd, page, pages,
                                   blocks, T, T, float(np.float32(hd ** -0.5)), F16, np.zeros((T, qh * hd)))
            mine = bound >= 0
            assert mine.sum() == total * qh * hd
            assert np.all((np.abs(O.from_bits(F16, g["y"]) - y) <= bound)[mine])
            past += fresh
            free = free[int(want[5][1]):]
    finally:
        cl.release()
        s.close()


# ---------------------------------------------------------------- heap tensors shared with other libraries

def test_heap_views():
    """A heap tensor as another library on the GPU finds it (address, shape, type), read and written there through the HIP
    runtime; what is no page's range is refused."""
    planner = HeapPlanner()
    space = {"a": (F32, (3, 5)), "b": (BF16, (8,)), "c": (U32, (4,)), "d": (F16, (2, 2, 2))}
    place = {n: planner.allocate(Arena.ACTIVATIONS, int(np.prod(sh)) * DType.SIZE[d]) for n, (d, sh) in space.items()}
    layout = planner.build()
    copy = C.CDLL(_native.LIB_PATH).hipMemcpy  # of the runtime that the library runs on
    copy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    b = HipBackend(0)
    try:
        heap = b.create_heap(layout)
        with pytest.raises(GpuContractException, match="table"):
            heap.view(1)
        table = TensorTable(layout)
        tok = {n: table.add_placed(n, place[n], d, list(sh), RO if n == "d" else 0) for n, (d, sh) in space.items()}
        heap.write_table(table.seal())
        rows = {n: heap.table.row(t) for n, t in tok.items()}
        for n, kind in (("a", "<f4"), ("b", "<i2"), ("c", "<i4"), ("d", "<f2")):
            view = heap.view(tok[n])
            face = view.__cuda_array_interface__
            assert face["shape"] == space[n][1] and face["typestr"] == kind and face["strides"] is None
            assert face["data"] == (view.address, n == "d")
            assert view.address == heap.address(rows[n][0], rows[n][1], 4)
        x, y = np.arange(15, dtype=np.float32).reshape(3, 5), np.zeros((3, 5), np.float32)
        heap.upload(rows["a"][0], rows["a"][1], x)
        assert copy(y.ctypes.data, heap.view(tok["a"]).address, 60, 2) == 0 and np.array_equal(x, y)
        assert copy(heap.view(tok["a"]).address, (x + 1).ctypes.data, 60, 1) == 0
        assert np.array_equal(np.frombuffer(heap.download(rows["a"][0], rows["a"][1], 60), np.float32), (x + 1).ravel())
        with pytest.raises(GpuContractException, match="slot 0"):
            heap.address(0, 0, 64)
        page = layout.pages[0].bytes
        heap.address(1, 0, page)
        for off, n in ((0, page + 1), (page + 1, 0), (1 << 63, 1 << 63), (page, 1)):
            with pytest.raises(GpuContractException, match="past the page"):
                heap.address(1, off, n)
        for slot in (2, -1, 64):
            with pytest.raises(GpuContractException, match="slot"):
                heap.address(slot, 0, 4)
        for token in (0, 9):
            with pytest.raises(GpuContractException, match="token"):
                heap.view(token)
    finally:
        b.close()


def test_paged_ids_belong_to_the_fast_set():
    ref, fast = HipBackend(0), HipBackend(0)
    try:
        ref.load_kernels()
        fast.load_kernels("fast")
        ids = [47, 48, 49]
        assert not any(ref.contains(i) for i in ids) and all(fast.contains(i) for i in ids)
        assert all(ref.contains(i) for i in range(41, 47)) and not fast.contains(50) and not ref.contains(50)
    finally:
        ref.close()
        fast.close()
