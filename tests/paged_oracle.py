"""The paged key/value cache in float64, for its tests: the step's plan by counting, the append by formula, the attention over
pages gathered one by one; and how far a kernel may be from them (each bound's terms are named where it is formed)."""
import numpy as np

from oracle import cpuref
from rosylnalive_amd.gpu_core import PAGED_NONE, DType

EPS_HALF = {DType.F16: 2.0 ** -11, DType.BF16: 2.0 ** -8, DType.F32: 2.0 ** -24}
U24 = 2.0 ** -24


def to_bits(dtype, a):
    a = np.asarray(a, np.float32)
    if dtype == DType.F16:
        with np.errstate(over="ignore"):
            return a.astype(np.float16).view(np.uint16)
    return a if dtype == DType.F32 else cpuref.bf16_narrow(a)


def from_bits(dtype, b):
    if dtype == DType.F16:
        return b.view(np.float16).astype(np.float64)
    if dtype == DType.F32:
        return b.view(np.float32).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def plan(past, fresh, free, table, blocks, page, pages, tokens, positions, slots):
    """(table, starts, context, positions, slots, counts) after paged_plan, given what the tensors held."""
    R, most = len(past), blocks * page
    table, positions, slots = table.copy(), positions.copy(), slots.copy()
    starts, context = np.zeros(R + 1, np.uint32), np.zeros(R, np.uint32)
    used, row, over = 0, 0, False
    for r in range(R):
        begin, end = min(past[r], most), min(past[r] + fresh[r], most)
        over |= past[r] + fresh[r] > most
        for b in range(-(-begin // page), -(-end // page)):
            table[r, b] = free[used] if used < len(free) else PAGED_NONE
            used += 1
        starts[r] = min(row, tokens)
        context[r] = end
        for j in range(fresh[r]):
            if row < tokens:
                pos = past[r] + j
                positions[row] = pos
                slots[row] = PAGED_NONE
                if pos < most and table[r, pos // page] < pages:
                    slots[row] = table[r, pos // page] * page + pos % page
            row += 1
    starts[R] = min(row, tokens)
    counts = np.array([row, used, (row > tokens) + 2 * over + 4 * (used > len(free))], np.uint32)
    return table, starts, context, positions, slots, counts


def append(qkv, qn, kn, cos, sin, positions, slots, total, qh, kvh, hd, page, pages, max_pos, eps, q, kc, vc):
    """(q, kc, vc) in float64 after the append, and the bounds of q and kc; values go in unrounded."""
    q, kc, vc = q.copy(), kc.copy(), vc.copy()
    bq, bk = np.zeros_like(q), np.zeros_like(kc)
    for t in range(total):
        x = qkv[t].reshape(qh + 2 * kvh, hd)
        h = x[:qh + kvh]
        w = np.concatenate([np.tile(qn, (qh, 1)), np.tile(kn, (kvh, 1))])
        n = w * h / np.sqrt((h * h).mean(1, keepdims=True) + eps)
        pos, slot = int(positions[t]), int(slots[t])
        if pos < max_pos:
            a, b = n[:, :hd // 2], n[:, hd // 2:]
            r = np.concatenate([a * cos[pos] - b * sin[pos], b * cos[pos] + a * sin[pos]], 1)
            # float32: the sum of squares in a tree, its root, three products, two products and a sum per rotated value
            m = np.tile(np.abs(a) + np.abs(b), (1, 2)) * (16 * U24)
        else:
            r, m = np.zeros_like(n), np.zeros_like(n)
        q[t], bq[t] = r[:qh].reshape(-1), m[:qh].reshape(-1)
        if slot // page < pages and pos < max_pos:
            at, off = divmod(slot, page)
            kc[at, :, off], bk[at, :, off] = r[qh:], m[qh:]
            vc[at, :, off // 8, :, off % 8] = x[qh + kvh:]
    return q, kc, vc, bq, bk


def attention(q, kc, vc, table, starts, context, qh, kvh, hd, page, pages, blocks, tokens, max_fresh, scale, dtype, y):
    """(y, bound) after attention_paged over tensors of float64; rows that it does not own keep y's values and get a bound
    of -1. A masked key or value is never touched, so it may hold anything."""
    y, bound = y.copy(), np.full(y.shape, -1.0)
    u = EPS_HALF[dtype]
    group = qh // kvh
    for r in range(len(context)):
        first, end = min(int(starts[r]), tokens), min(int(starts[r + 1]), tokens)
        ctx = min(int(context[r]), blocks * page)
        for i in range(min(end - first, max_fresh)):
            seen = ctx - (end - first) + i + 1
            pos = np.arange(max(seen, 0))
            ids = table[r, pos // page]
            pos, ids = pos[ids < pages], ids[ids < pages].astype(np.int64)
            for h in range(kvh):
                k, v = kc[ids, h, pos % page], vc[ids, h, (pos % page) // 8, :, pos % 8]
                for g in range(h * group, (h + 1) * group):
                    o = slice(g * hd, (g + 1) * hd)
                    if not len(pos):
                        y[first + i, o], bound[first + i, o] = 0, 0
                        continue
                    qr = q[first + i, o]
                    with np.errstate(all="ignore"):
                        s = k @ qr * scale
                        p = np.exp(s - s.max())
                        l = p.sum()
                        y[first + i, o] = p @ v / l
                        # the exponent's float32: the dot over hd, the scaling and the running reference
                        ds = (hd + 8) * U24 * (np.abs(k) @ np.abs(qr) * scale).max() + 4 * U24 * np.abs(s).max()
                        # a weight's rounding to the type, the float32 sums over the keys, and the weights that the type's
                        # own underflow takes (2^-25 of the largest each, fp16 only)
                        rel = u + 2 * ds + (len(pos) + 16) * U24
                        tiny = len(pos) * 2.0 ** -25 * np.abs(v).max() / l if dtype == DType.F16 else 0.0
                        bound[first + i, o] = p @ np.abs(v) / l * rel + tiny + u * np.abs(y[first + i, o]) + 2.0 ** -25
    return y, bound
