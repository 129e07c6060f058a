"""The operators of a key/value cache in pages, as a program that serves many requests calls them, one step at a time:

  plan        from each request's cached and new token counts, on the GPU: the pages that the new tokens need (taken from a
              list of free ones into the block table), and for each new token its position and its slot in the cache
  append      the projections of the new tokens: RMSNorm of each query and key head, the rotation by position, the keys and
              values into their slots, the queries to the attention
  attention   the new tokens of every request (a prompt, a chunk of one, one token, any mix) over the request's pages,
              causal, query heads in groups on shared KV heads

A page holds `page` positions of every KV head: keys as [kv_heads, page, head_dim], values as [kv_heads, page / 8,
head_dim, 8]. A request's table row lists its pages in order. 0xFFFFFFFF (-1 here) stands for no page and no slot.

A case is a call with its lengths: `requests` of them, of which the first `chunks` bring chunk_lo .. chunk_hi new tokens and
the others one, over past_lo .. past_hi cached ones, drawn from `mix`. Rows of padding follow the last token's (a program
that records its step once records it for a fixed number of rows). The values of the inputs come from the seed.
"""
import collections
import math
import random

import numpy as np
import torch

own = False

NONE = -1  # 0xFFFFFFFF as the int32 that holds its bits
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, **kw):
    c = {"name": name, "op": op, "requests": 1, "chunks": 0, "chunk_lo": 1, "chunk_hi": 1, "past_lo": 0, "past_hi": 0,
         "mix": 1, "pad": 0, "page": 64, "q_heads": 16, "kv_heads": 8, "head_dim": 128, "dtype": "f16", "qkv": "f32"}
    c.update(kw)
    return c


def listed():
    return [
        # the bookkeeping of a decode step: 64 requests, one token each, some of them at the start of a page
        _case("plan_step64", "plan", requests=64, past_lo=1, past_hi=8192),
        # the same for a step that admits prompts: 60 of 700 requests bring some hundreds of tokens, small pages
        _case("plan_prompts700", "plan", requests=700, chunks=60, chunk_lo=100, chunk_hi=700, past_hi=2000, mix=2, page=16,
              pad=37),
        # the new rows of a 16-request decode step
        _case("append_step16", "append", requests=16, past_lo=100, past_hi=8192),
        # a 512-token chunk of a long document, at an odd position
        _case("append_chunk512", "append", chunks=1, chunk_lo=512, chunk_hi=512, past_lo=7681, past_hi=7681),
        # ragged prompts together, bf16 projections and cache, four query heads a KV head
        _case("append_prompts23", "append", requests=23, chunks=23, chunk_lo=3, chunk_hi=790, past_hi=300, mix=3, pad=5,
              page=16, q_heads=32, dtype="bf16", qkv="bf16"),
        # one request's token at a short context: the smallest attention
        _case("attn_step700", "attention", past_lo=700, past_hi=700),
        # one request's token at a very long context
        _case("attn_step65k", "attention", past_lo=65701, past_hi=65701, page=16, q_heads=32, dtype="bf16"),
        # a full decode batch at 8K context
        _case("attn_batch16_8k", "attention", requests=16, past_lo=8192, past_hi=8192),
        # many requests of uneven context, one token each
        _case("attn_batch200", "attention", requests=200, past_lo=1, past_hi=4000, mix=4, page=16, dtype="bf16", pad=3),
        # a whole prompt
        _case("attn_prompt2048", "attention", chunks=1, chunk_lo=2048, chunk_hi=2048),
        # a chunk far into a long document: the matrix cores carry the weight
        _case("attn_chunk4096_at28k", "attention", chunks=1, chunk_lo=4096, chunk_hi=4096, past_lo=28672, past_hi=28672,
              page=32),
        # decoding requests and chunks of prompts in one step, seven query heads a KV head, heads of 64
        _case("attn_mixed40", "attention", requests=40, chunks=3, chunk_lo=200, chunk_hi=900, past_hi=6000, mix=5, page=16,
              q_heads=14, kv_heads=2, head_dim=64, dtype="bf16", pad=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "append", "append", "step", "step", "prompt", "mixed"))
    kw = {"mix": rng.randrange(1 << 30), "page": rng.choice((16, 32, 64, 128)), "pad": rng.choice((0, 0, rng.randint(1, 40)))}
    heads = rng.choice(((16, 8, 128), (16, 8, 128), (32, 8, 128), (14, 2, 64), (12, 12, 64), (8, 1, 128)))
    kw.update(zip(("q_heads", "kv_heads", "head_dim"), heads))
    kw["dtype"] = rng.choice(("f16", "bf16"))
    if kind == "plan":
        n = _log(rng, 1, 1000)
        return _draw("plan", requests=n, chunks=rng.randint(0, min(n, 60)), chunk_hi=_log(rng, 2, 700),
                     past_hi=_log(rng, 64, 8000), **kw)
    if kind == "append":
        n = _log(rng, 1, 64)
        return _draw("append", requests=n, chunks=rng.choice((0, rng.randint(0, min(n, 16)))), chunk_hi=_log(rng, 2, 700),
                     past_hi=_log(rng, 2, 4000), qkv=rng.choice(("f32", "f32", kw["dtype"])), **kw)
    if kind == "step":  # one token each; about 2^18 cached ones at most
        n = _log(rng, 1, 256)
        past = _log(rng, 2, min(65536, (1 << 18) // n))
        return _draw("attention", requests=n, past_lo=rng.choice((past, 0, past // 2)), past_hi=past, **kw)
    if kind == "prompt":
        new = _log(rng, 2, 4096)
        past = rng.choice((0, 0, _log(rng, 2, 16384)))
        return _draw("attention", chunks=1, chunk_lo=new, chunk_hi=new, past_lo=past, past_hi=past, **kw)
    n = rng.randint(2, 48)
    return _draw("attention", requests=n, chunks=rng.randint(1, min(n, 4)), chunk_hi=_log(rng, 4, 900),
                 past_hi=_log(rng, 16, 4000), **kw)


def _draw(op, **kw):
    c = _case("", op, **kw)
    del c["name"]
    return c


# ---------------------------------------------------------------- lengths and inputs

def _lengths(case):
    """Cached and new tokens of each request: the case alone decides."""
    r = random.Random(case["mix"])
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["requests"])]
    fresh = [r.randint(case["chunk_lo"], case["chunk_hi"]) if i < case["chunks"] else 1 for i in range(case["requests"])]
    order = list(range(case["requests"]))
    r.shuffle(order)  # the chunks stand anywhere in the batch
    return [past[i] for i in order], [fresh[i] for i in order]


def _pages(tokens, page):
    return -(-tokens // page)


def _layout(case, seed):
    """What a serving program has decided: lengths, and for append and attention the table and the slots."""
    page = case["page"]
    past, fresh = (np.array(v, np.int64) for v in _lengths(case))
    end = past + fresh
    r = np.random.default_rng([seed, 11])
    need = _pages(end, page)
    blocks = int(need.max()) + 2
    pages = int(need.sum()) + 8
    ids = r.permutation(pages)
    table = np.full((case["requests"], blocks), NONE, np.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(fresh)])
    owner = np.repeat(np.arange(case["requests"]), fresh)
    position = past[owner] + np.arange(starts[-1]) - starts[owner]
    slot = table[owner, position // page] * page + position % page
    return {"past": past, "fresh": fresh, "end": end, "table": table, "pages": pages, "blocks": blocks, "starts": starts,
            "position": position, "slot": slot, "spare": ids[at:], "total": int(starts[-1])}


def _int(a, *more):
    return torch.from_numpy(np.concatenate([np.asarray(a, np.int64).reshape(-1), *more]).astype(np.int32)).cuda()


def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(TYPES[dtype])


def _caches(case, lay, g):
    kvh, page, hd = case["kv_heads"], case["page"], case["head_dim"]
    return (_normal(g, (lay["pages"], kvh, page, hd), case["dtype"]),
            _normal(g, (lay["pages"], kvh, page // 8, hd, 8), case["dtype"]))


def _inputs(case, seed):
    """(tensors, scalars, facts the host knows) of the call."""
    lay = _layout(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    R, T, hd, page = case["requests"], lay["total"] + case["pad"], case["head_dim"], case["page"]
    qh, kvh = case["q_heads"], case["kv_heads"]
    if case["op"] == "plan":
        # the table before the step: the pages of the cached tokens; the free list: the others, in any order
        have = _pages(lay["past"], page)
        cols = np.arange(lay["blocks"])[None, :]
        before = np.where(cols < have[:, None], lay["table"], NONE)
        free = np.concatenate([lay["table"][(cols >= have[:, None]) & (lay["table"] != NONE)], lay["spare"]])
        free = np.random.default_rng([seed, 12]).permutation(free)
        t = {"past": _int(lay["past"]), "fresh": _int(lay["fresh"]), "free": _int(free), "table": _int(before).view(R, -1),
             "starts": _int(np.zeros(R + 1)), "context": _int(np.zeros(R)), "positions": _int(np.zeros(T)),
             "slots": _int(np.full(T, NONE)), "counts": _int(np.zeros(3))}
        scalars = {"requests": R, "blocks": lay["blocks"], "page": page, "pages": lay["pages"], "free_count": len(free),
                   "tokens": T}
    elif case["op"] == "append":
        end = int(lay["end"].max())
        angle = np.arange(end)[:, None] * (1e6 ** (-np.arange(0, hd, 2) / hd))[None, :]
        k_cache, v_cache = _caches(case, lay, g)
        pad = np.zeros(case["pad"], np.int64)
        norm = lambda: (1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(torch.bfloat16)  # noqa: E731
        t = {"qkv": _normal(g, (T, (qh + 2 * kvh) * hd), case["qkv"], 1.5), "q_norm": norm(), "k_norm": norm(),
             "cos_table": torch.from_numpy(np.cos(angle).astype(np.float32)).cuda(),
             "sin_table": torch.from_numpy(np.sin(angle).astype(np.float32)).cuda(),
             "starts": _int(lay["starts"]), "positions": _int(lay["position"], pad),
             "slots": _int(lay["slot"], pad + NONE), "q": torch.zeros((T, qh * hd), dtype=TYPES[case["dtype"]], device="cuda"),
             "k_cache": k_cache, "v_cache": v_cache}
        scalars = {"requests": R, "tokens": T, "q_heads": qh, "kv_heads": kvh, "head_dim": hd, "max_pos": end, "page": page,
                   "pages": lay["pages"], "eps": EPS}
    else:
        k_cache, v_cache = _caches(case, lay, g)
        t = {"q": _normal(g, (T, qh * hd), case["dtype"], 1.5), "k_cache": k_cache, "v_cache": v_cache,
             "table": _int(lay["table"]).view(R, -1), "starts": _int(lay["starts"]), "context": _int(lay["end"]),
             "y": torch.zeros((T, qh * hd), dtype=TYPES[case["dtype"]], device="cuda")}
        scalars = {"requests": R, "tokens": T, "max_fresh": int(lay["fresh"].max()), "q_heads": qh, "kv_heads": kvh,
                   "head_dim": hd, "blocks": lay["blocks"], "page": page, "pages": lay["pages"], "scale": hd ** -0.5}
    facts = {"total": lay["total"], "most": int(lay["end"].max()), "fresh": int(lay["fresh"].max())}
    return t, scalars, facts


OUTPUTS = {"plan": ("table", "starts", "context", "positions", "slots", "counts"), "append": ("q", "k_cache", "v_cache"),
           "attention": ("y",)}
KERNELS = {"plan": "paged_plan", "append": "qk_norm_rope_append_paged", "attention": "attention_paged"}


def prepare(case, seed):
    t, scalars, facts = _inputs(case, seed)
    state = {"case": case, "t": t, "scalars": scalars, "facts": facts}
    if own:  # the same tensors in the heap of a device, and the operator on a list, as the framework's programs hold them
        state["call"] = _Call(case["op"], state.pop("t"), scalars)
    return state


def run(state):
    if own:
        return state["call"].run()
    return PLAIN[state["case"]["op"]](state["t"], state["scalars"], state["facts"])


def work(case):
    """plan: the lengths, the new pages' ids and the table entries that hold new tokens, read or written, positions and
    slots written. append: the projections read, the queries, keys and values written, the tables' rows and the indices.
    attention: every cached key and value of each request once, queries and results, the table; a multiply-add is two."""
    past, fresh = _lengths(case)
    page, hd, qh, kvh = case["page"], case["head_dim"], case["q_heads"], case["kv_heads"]
    tokens = sum(fresh)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "plan":
        new = sum(_pages(p + f, page) - _pages(p, page) for p, f in zip(past, fresh))
        touched = sum(_pages(p + f, page) - p // page for p, f in zip(past, fresh))
        return {"bytes": 4 * (4 * len(past) + 4 + new + touched + 2 * tokens), "flops": 0}
    if case["op"] == "append":
        rows = max(p + f for p, f in zip(past, fresh)) if case["requests"] == 1 else tokens
        return {"bytes": tokens * (qh + 2 * kvh) * hd * (size[case["qkv"]] + size[case["dtype"]])
                + 4 * min(rows, tokens) * hd + 8 * tokens, "flops": tokens * (qh + kvh) * hd * 9}
    keys = sum(p + f for p, f in zip(past, fresh))
    pairs = sum(f * p + f * (f + 1) // 2 for p, f in zip(past, fresh))
    blocks = sum(_pages(p + f, page) for p, f in zip(past, fresh))
    return {"bytes": 2 * (2 * keys * kvh + 2 * tokens * qh) * hd + 4 * blocks, "flops": 4 * pairs * qh * hd}


# ---------------------------------------------------------------- the framework's calls

class _Device:
    """The device, gone with the last tensor that shares its memory."""

    def __init__(self, backend):
        self.backend = backend

    def __del__(self):
        self.backend.close()


class _Shared:
    """A tensor of the heap to torch, which holds this object for as long as it uses the memory."""

    def __init__(self, view, device):
        self.__cuda_array_interface__ = view.__cuda_array_interface__
        self.device = device


class _Call:
    def __init__(self, op, tensors, scalars):
        from rosylnalive_amd import gpu_core as G

        types = {torch.float32: G.DType.F32, torch.float16: G.DType.F16, torch.bfloat16: G.DType.BF16,
                 torch.int32: G.DType.U32}
        space = {n: (types[t.dtype], tuple(t.shape[:3]) + (t.shape[3:].numel(),) if t.dim() > 4 else tuple(t.shape))
                 for n, t in tensors.items()}  # a table row holds four dims
        if op == "attention":
            space["workspace"] = (G.DType.U32, (G.attention_paged_workspace_words(
                scalars["requests"], scalars["tokens"], scalars["q_heads"], scalars["kv_heads"], scalars["head_dim"]),))
        planner = G.HeapPlanner()
        place = {n: planner.allocate(G.Arena.ACTIVATIONS, -(-math.prod(s) * G.DType.SIZE[d] // 4) * 4)
                 for n, (d, s) in space.items()}
        layout = planner.build()
        backend = G.HipBackend(0)
        self.device = _Device(backend)
        backend.load_kernels("fast")
        heap = backend.create_heap(layout)
        table = G.TensorTable(layout)
        token = {n: table.add_placed(n, place[n], d, s) for n, (d, s) in space.items()}
        heap.write_table(table.seal())
        views = {n: torch.as_tensor(_Shared(heap.view(token[n]), self.device), device="cuda").view(t.dtype).view(t.shape)
                 for n, t in tensors.items()}
        for n, t in tensors.items():
            views[n].copy_(t)
        torch.cuda.synchronize()  # torch's stream is not the device's
        self.outputs = {n: views[n] for n in OUTPUTS[op]}
        self.list = backend.begin(reusable=True)
        self.list.dispatch(KERNELS[op], G.ArgBlock.encode(KERNELS[op], **token, **scalars))
        self.pending = collections.deque()

    def run(self):
        backend = self.device.backend
        self.pending.append(backend.submit(self.list))
        if len(self.pending) > 64:  # a program keeps the work under way bounded
            backend.wait(self.pending.popleft())
        return self.outputs


# ---------------------------------------------------------------- the plain forms

def _plan(t, a, facts):
    page, most, dev = a["page"], a["blocks"] * a["page"], t["past"].device
    past, fresh, free = t["past"].long(), t["fresh"].long(), t["free"].long()
    begin, end = past.clamp(max=most), (past + fresh).clamp(max=most)
    have, want = (begin + page - 1) // page, (end + page - 1) // page
    first = torch.cumsum(want - have, 0) - (want - have)
    col = torch.arange(a["blocks"], device=dev)[None, :]
    at = first[:, None] + col - have[:, None]
    taken = torch.where(at < a["free_count"], free[at.clamp(0, max(0, a["free_count"] - 1))], NONE)
    table = torch.where((col >= have[:, None]) & (col < want[:, None]), taken, t["table"].long())
    ends = torch.cumsum(fresh, 0)
    total = ends[-1].clamp(max=a["tokens"])
    row = torch.arange(a["tokens"], device=dev)
    owner = torch.searchsorted(ends, row, right=True).clamp(max=a["requests"] - 1)
    position = past[owner] + row - (ends - fresh)[owner]
    entry = table[owner, (position // page).clamp(max=a["blocks"] - 1)]
    good = (position < most) & (entry >= 0) & (entry < a["pages"])
    slot = torch.where(good, entry * page + position % page, NONE)
    valid = row < total
    needed = (want - have).sum()
    status = (ends[-1] > a["tokens"]).long() + 2 * (past + fresh > most).any() + 4 * (needed > a["free_count"])
    t["table"].copy_(table)
    t["starts"].copy_(torch.cat([torch.zeros(1, dtype=torch.long, device=dev), ends]).clamp(max=a["tokens"]))
    t["context"].copy_(end)
    t["positions"].copy_(torch.where(valid, position, t["positions"].long()))
    t["slots"].copy_(torch.where(valid, slot, t["slots"].long()))
    t["counts"].copy_(torch.stack([ends[-1], needed, status]))
    return {n: t[n] for n in OUTPUTS["plan"]}


def _append(t, a, facts):
    n, hd, qh, kvh, page = facts["total"], a["head_dim"], a["q_heads"], a["kv_heads"], a["page"]
    x = t["qkv"][:n].float().view(n, qh + 2 * kvh, hd)
    position, slot = t["positions"][:n].long(), t["slots"][:n].long()
    w = torch.cat([t["q_norm"].float().expand(qh, hd), t["k_norm"].float().expand(kvh, hd)])
    h = x[:, :qh + kvh]
    h = w * (h / torch.sqrt((h * h).mean(-1, keepdim=True) + a["eps"]))
    cos, sin = t["cos_table"][position][:, None, :], t["sin_table"][position][:, None, :]
    lo, hi = h[..., :hd // 2], h[..., hd // 2:]
    h = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(t["q"].dtype)
    t["q"][:n] = h[:, :qh].reshape(n, qh * hd)
    at, off = slot // page, slot % page
    t["k_cache"][at, :, off] = h[:, qh:]
    t["v_cache"][at, :, off // 8, :, off % 8] = x[:, qh + kvh:].to(t["v_cache"].dtype)
    return {n: t[n] for n in OUTPUTS["append"]}


def _attention(t, a, facts):
    R, hd, qh, kvh, page, n = a["requests"], a["head_dim"], a["q_heads"], a["kv_heads"], a["page"], facts["total"]
    group, rows, dev = qh // kvh, facts["fresh"], t["q"].device
    starts, context = t["starts"].long(), t["context"].long()
    fresh = starts[1:] - starts[:-1]
    # keys and values of every request side by side, in order of position
    table = t["table"].long()[:, :_pages(facts["most"], page)].clamp(min=0)
    most = table.shape[1] * page
    k = t["k_cache"][table].float().permute(0, 2, 4, 1, 3).reshape(R, kvh, hd, most).contiguous()
    v = t["v_cache"][table].float().permute(0, 2, 1, 3, 5, 4).reshape(R, kvh, most, hd).contiguous()
    i = torch.arange(rows, device=dev)
    at = (starts[:-1, None] + i).clamp(max=n - 1)
    q = t["q"].float()[at].view(R, rows, kvh, group, hd).permute(0, 2, 3, 1, 4).reshape(R, kvh, group * rows, hd).contiguous()
    s = torch.matmul(q, k).mul_(a["scale"]).view(R, kvh, group, rows, most)
    last = (context - fresh)[:, None] + i  # the last key that row i of a request sees
    hidden = (torch.arange(most, device=dev) > last[:, :, None])[:, None, None]
    s.masked_fill_(hidden, -math.inf)
    s.sub_(s.max(-1, keepdim=True).values).exp_()
    s.div_(s.sum(-1, keepdim=True))
    o = torch.matmul(s.view(R, kvh, group * rows, most), v).view(R, kvh, group, rows, hd).permute(0, 3, 1, 2, 4)
    row = torch.arange(n, device=dev)
    owner = torch.searchsorted(starts[1:], row, right=True)
    t["y"][:n] = o[owner, row - starts[owner]].reshape(n, qh * hd).to(t["y"].dtype)
    return {"y": t["y"]}


PLAIN = {"plan": _plan, "append": _append, "attention": _attention}


# ---------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    t, a, facts = _inputs(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attention": _exact_attention}[case["op"]](t, a)


def _requests(t):
    """(first row, rows) of each request."""
    s = t["starts"].tolist()
    return [(lo, hi - lo) for lo, hi in zip(s, s[1:])]


def _exact_plan(t, a):
    t = {n: v.cpu().numpy().astype(np.int64) for n, v in t.items()}
    page, used, row = a["page"], 0, 0
    t["counts"][2] = 0
    for r in range(a["requests"]):
        t["starts"][r] = row
        length = int(t["past"][r])
        for _ in range(int(t["fresh"][r])):
            if length % page == 0:
                t["table"][r, length // page] = t["free"][used]
                used += 1
            t["positions"][row] = length
            t["slots"][row] = t["table"][r, length // page] * page + length % page
            length, row = length + 1, row + 1
        t["context"][r] = length
    t["starts"][-1] = row
    t["counts"][:2] = row, used
    return {n: t[n].astype(np.int32) for n in OUTPUTS["plan"]}


def _exact_append(t, a):
    hd, qh, kvh, page = a["head_dim"], a["q_heads"], a["kv_heads"], a["page"]
    out = {n: t[n].double().cpu().numpy() for n in OUTPUTS["append"]}
    qkv, cos, sin = (t[n].double().cpu().numpy() for n in ("qkv", "cos_table", "sin_table"))
    norms = [t["q_norm"].double().cpu().numpy()] * qh + [t["k_norm"].double().cpu().numpy()] * kvh
    positions, slots = t["positions"].tolist(), t["slots"].tolist()
    for row in range(t["starts"][-1].item()):
        heads = qkv[row].reshape(qh + 2 * kvh, hd)
        c, s = cos[positions[row]], sin[positions[row]]
        at, off = divmod(slots[row], page)
        turned = heads[:qh + kvh] * np.stack(norms)
        turned *= 1 / np.sqrt(np.square(heads[:qh + kvh]).sum(1, keepdims=True) / hd + a["eps"])
        pair = turned.reshape(-1, 2, hd // 2)
        turned = np.stack([pair[:, 0] * c - pair[:, 1] * s, pair[:, 0] * s + pair[:, 1] * c], 1).reshape(-1, hd)
        out["q"][row] = turned[:qh].reshape(-1)
        out["k_cache"][at, :, off] = turned[qh:]
        out["v_cache"][at, :, off // 8, :, off % 8] = heads[qh + kvh:]
    return out


def _exact_attention(t, a):
    hd, qh, kvh, page = a["head_dim"], a["q_heads"], a["kv_heads"], a["page"]
    y = t["y"].double()
    for r, (lo, rows) in enumerate(_requests(t)):
        keys = t["context"][r].item()
        ids = t["table"][r, :_pages(keys, page)].long()
        q = t["q"][lo:lo + rows].double().view(rows, qh, hd)
        first = keys - rows
        for h in range(kvh):
            k = t["k_cache"][ids, h].double().reshape(-1, hd)[:keys].t().contiguous()
            v = t["v_cache"][ids, h].double().transpose(2, 3).reshape(-1, hd)[:keys].contiguous()
            for g in range(h * qh // kvh, (h + 1) * qh // kvh):
                for i in range(0, rows, 2048):
                    j = min(rows, i + 2048)
                    s = torch.mm(q[i:j, g].contiguous(), k) * a["scale"]
                    seen = first + torch.arange(i, j, device=s.device)
                    s.masked_fill_(torch.arange(keys, device=s.device)[None] > seen[:, None], -math.inf)
                    y[lo + i:lo + j, g * hd:(g + 1) * hd] = torch.mm(torch.softmax(s, 1), v)
    return {"y": y.cpu().numpy()}
