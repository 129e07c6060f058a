"""Refusals of the paged key/value cache's dispatches (CPU): every size, type and range that the kernels rely on is checked
when a dispatch is recorded."""
import pytest

from rosylnalive_amd import _native
from rosylnalive_amd.gpu_core import (Arena, ArgBlock, Catalog, DType, GpuContractException, HeapPlanner, TensorTable,
                                      attention_paged_workspace_words, prepare)

F32, BF16, F16, U32 = DType.F32, DType.BF16, DType.F16, DType.U32

# the least tensors of a dispatch: 3 requests, 10 tokens, 4/2 heads of 64, 5 blocks a request, 7 pages of 16
R, T, QH, KVH, HD, B, P, N, MP = 3, 10, 4, 2, 64, 5, 16, 7, 90
PLAN = {"past": (U32, R), "fresh": (U32, R), "free": (U32, 6), "table": (U32, R * B), "starts": (U32, R + 1),
        "context": (U32, R), "positions": (U32, T), "slots": (U32, T), "counts": (U32, 3)}
PLAN_S = dict(requests=R, blocks=B, page=P, pages=N, free_count=6, tokens=T)
APPEND = {"qkv": (F32, T * (QH + 2 * KVH) * HD), "q_norm": (BF16, HD), "k_norm": (BF16, HD), "cos_table": (F32, MP * HD // 2),
          "sin_table": (F32, MP * HD // 2), "starts": (U32, R + 1), "positions": (U32, T), "slots": (U32, T),
          "q": (F16, T * QH * HD), "k_cache": (F16, N * P * KVH * HD), "v_cache": (F16, N * P * KVH * HD)}
APPEND_S = dict(requests=R, tokens=T, q_heads=QH, kv_heads=KVH, head_dim=HD, max_pos=MP, page=P, pages=N, eps=1e-6)
ATTN = {"q": (BF16, T * QH * HD), "k_cache": (BF16, N * P * KVH * HD), "v_cache": (BF16, N * P * KVH * HD), "table": (U32, R * B),
        "starts": (U32, R + 1), "context": (U32, R), "y": (BF16, T * QH * HD)}
ATTN_S = dict(requests=R, tokens=T, max_fresh=0, q_heads=QH, kv_heads=KVH, head_dim=HD, blocks=B, page=P, pages=N, scale=0.125)
CALLS = {"paged_plan": (PLAN, PLAN_S), "qk_norm_rope_append_paged": (APPEND, APPEND_S), "attention_paged": (ATTN, ATTN_S)}


def _prepare(kernel, tensors=None, alias=None, **scalars):
    base, s = CALLS[kernel]
    space = dict(base, **(tensors or {}))
    if kernel == "attention_paged":
        space.setdefault("workspace", (U32, attention_paged_workspace_words(R, T, QH, KVH, HD)))
    planner = HeapPlanner()
    places = {n: planner.allocate(Arena.ACTIVATIONS, (c * DType.SIZE[dt] + 3) // 4 * 4) for n, (dt, c) in space.items()}
    table = TensorTable(planner.build())
    tok = {n: table.add_placed(n, places[n], dt, [c], 0) for n, (dt, c) in space.items()}
    for a, b in (alias or {}).items():
        tok[a] = tok[b]
    return prepare(table.seal(), Catalog.find(kernel).id, ArgBlock.encode(kernel, **tok, **dict(s, **scalars)))


@pytest.mark.parametrize("kernel", list(CALLS))
def test_least_tensors_are_enough(kernel):
    _prepare(kernel)


@pytest.mark.parametrize("kernel,name", [(k, n) for k, (t, _) in CALLS.items() for n in t if n != "free"])
def test_one_element_less_is_refused(kernel, name):
    dt, c = CALLS[kernel][0][name]
    with pytest.raises(GpuContractException, match="elements"):
        _prepare(kernel, {name: (dt, c - 1)})


def test_free_list_may_be_longer_or_unused():
    _prepare("paged_plan", free_count=0)
    with pytest.raises(GpuContractException, match="free"):
        _prepare("paged_plan", free_count=7)


def test_workspace_too_small():
    n = attention_paged_workspace_words(R, T, QH, KVH, HD)
    with pytest.raises(GpuContractException, match="workspace"):
        _prepare("attention_paged", {"workspace": (U32, n - 1)})


BAD = [("requests", 0, "requests"), ("requests", 4097, "requests"), ("tokens", 0, "tokens|grid"), ("page", 8, "page"),
       ("page", 24, "page"), ("page", 512, "page"), ("page", 0, "page"), ("pages", 0, "pages"),
       ("pages", 1 << 28, "pages"), ("blocks", 0, "blocks"), ("blocks", 1 << 28, "blocks"), ("kv_heads", 0, "kv_heads"),
       ("kv_heads", 3, "kv_heads"), ("q_heads", 0, "kv_heads|grid"), ("head_dim", 32, "head_dim"), ("head_dim", 0, "head_dim|grid"),
       ("max_pos", 0, "max_pos"), ("scale", 0.0, "scale"), ("scale", -1.0, "scale"), ("scale", float("nan"), "scale"),
       ("scale", float("inf"), "scale"),
       # sizes whose products wrap 32 or 64 bits
       ("tokens", 0xFFFFFFFF, "elements|grid"), ("q_heads", 0xFFFFFFFE, "elements|grid|query heads"), ("q_heads", 514, "elements|query heads"), ("max_pos", 0xFFFFFFFF, "elements"),
       ("pages", 0x0FFFFFFF, "elements|pages")]


@pytest.mark.parametrize("kernel,field,value,match", [(k, f, v, m) for k, (_, s) in CALLS.items() for f, v, m in BAD
                                                      if f in s and (k, v) != ("paged_plan", 0x0FFFFFFF)])
def test_scalars_out_of_range_are_refused(kernel, field, value, match):
    with pytest.raises(GpuContractException, match=match):
        _prepare(kernel, **{field: value})


def _typed(kernel, names, dtype):
    return {n: (dtype, CALLS[kernel][0][n][1]) for n in names}


@pytest.mark.parametrize("names", [("q",), ("k_cache",), ("v_cache",), ("y",), ("q", "y"), ("k_cache", "v_cache")])
def test_attention_types_are_not_mixed(names):
    with pytest.raises(GpuContractException, match="mixed"):
        _prepare("attention_paged", _typed("attention_paged", names, F16))


def test_attention_takes_fp16_and_bf16_throughout():
    for dt in (F16, BF16):
        _prepare("attention_paged", _typed("attention_paged", ("q", "k_cache", "v_cache", "y"), dt))
    with pytest.raises(GpuContractException, match="does not accept"):
        _prepare("attention_paged", _typed("attention_paged", ("q", "k_cache", "v_cache", "y"), F32))


def test_append_types():
    name = "qk_norm_rope_append_paged"
    for dt in (F16, BF16):
        _prepare(name, _typed(name, ("q", "k_cache", "v_cache"), dt))
        _prepare(name, _typed(name, ("qkv", "q", "k_cache", "v_cache"), dt))
    for names, dt in ((("q",), BF16), (("k_cache",), BF16), (("v_cache",), BF16), (("qkv",), BF16)):
        with pytest.raises(GpuContractException, match="mixed"):
            _prepare(name, _typed(name, names, dt))
    with pytest.raises(GpuContractException, match="does not accept"):
        _prepare(name, _typed(name, ("q_norm",), F16))


@pytest.mark.parametrize("kernel,a,b", [("attention_paged", "y", "q"), ("attention_paged", "v_cache", "k_cache"),
                                        ("qk_norm_rope_append_paged", "v_cache", "k_cache"),
                                        ("paged_plan", "context", "past"), ("paged_plan", "slots", "positions")])
def test_aliases(kernel, a, b):
    if (a, b) == ("v_cache", "k_cache") and kernel == "attention_paged":
        _prepare(kernel, alias={a: b})  # both only read
        return
    with pytest.raises(GpuContractException, match="overlap"):
        _prepare(kernel, alias={a: b})


def test_workspace_entry_point():
    assert attention_paged_workspace_words(1, 1, 1, 1, 64) >= 1
    assert _native.lib().lrm_attention_paged_workspace(1, 1, 1, 1, 64, None) == _native.LRM_E_ARG
    # no less for more of anything
    base = attention_paged_workspace_words(8, 100, 16, 8, 128)
    for more in ((9, 100, 16, 8, 128), (8, 3000, 16, 8, 128), (8, 100, 32, 8, 128)):
        assert attention_paged_workspace_words(*more) >= base
