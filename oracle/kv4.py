"""Float64 oracle of the paged 4-bit KV cache (csrc/fn_kv4.h): page records, planning, storing, loading, attention.

Written from the definitions, one request, one block and one row at a time (numpy, no torch), for
tests/test_kv4_gpu.py and tests/test_kv4_cpu.py.
"""

from __future__ import annotations

import numpy as np

GROUP = 64


def record_bytes(hd, bs):
    return 2 * bs * (hd // 2 + hd // GROUP * 2)


def quantise(x):
    """Blocks of 64 (last axis, fp32) -> (codes uint8 0..15, scale fp16), fp32 arithmetic as the definition gives it."""
    x = np.asarray(x, np.float32)
    big, small = x.max(-1, keepdims=True), x.min(-1, keepdims=True)
    with np.errstate(all="ignore"):
        d = np.where(big >= -small, big, small) * np.float32(-0.125)
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d).astype(np.float32)
        t = np.trunc((x * inv).astype(np.float32) + np.float32(8.5))
        c = np.clip(np.where(np.isnan(t), 0, t), 0, 15).astype(np.uint8)
        bad = ~np.isfinite(x).all(-1, keepdims=True) | (np.abs(d) > 65504)
        s = np.where(bad, np.float32(np.nan), d).astype(np.float16)
    return c, s[..., 0]


def values(c, s):
    return (c.astype(np.float64) - 8) * s.astype(np.float64)[..., None]


def _parts(rec, hd, bs):
    """Views of one record: K codes, V codes [ng][bs][32], K scales, V scales [ng][bs]."""
    ng, kb, sb = hd // GROUP, bs * hd // 2, bs * (hd // GROUP) * 2
    return (rec[:kb].reshape(ng, bs, 32), rec[kb:2 * kb].reshape(ng, bs, 32),
            rec[2 * kb:2 * kb + sb].view(np.float16).reshape(ng, bs),
            rec[2 * kb + sb:].view(np.float16).reshape(ng, bs))


def store(pages, hd, bs, k, v, slots):
    """pages uint8 [pages][nkv][record], updated; k, v [rows][nkv][hd] fp32."""
    for t, slot in enumerate(slots):
        if not 0 <= slot < pages.shape[0] * bs:
            continue
        for h in range(pages.shape[1]):
            p = _parts(pages[slot // bs, h], hd, bs)
            for part, x in enumerate((k, v)):
                c, s = quantise(x[t, h].reshape(-1, GROUP))
                p[part][:, slot % bs] = c[:, 0::2] | (c[:, 1::2] << 4)
                p[2 + part][:, slot % bs] = s


def load(pages, hd, bs, slots):
    """float64 k, v [rows][nkv][hd]."""
    out = np.zeros((2, len(slots), pages.shape[1], hd))
    for t, slot in enumerate(slots):
        if not 0 <= slot < pages.shape[0] * bs:
            continue
        for h in range(pages.shape[1]):
            p = _parts(pages[slot // bs, h], hd, bs)
            for part in range(2):
                b = p[part][:, slot % bs]
                c = np.stack([b & 15, b >> 4], -1).reshape(-1, GROUP)
                out[part, t, h] = values(c, p[2 + part][:, slot % bs]).reshape(-1)
    return out[0], out[1]


def attn(pages, hd, bs, q, cu, kv_len, table, scale=None, gate=None):
    """float64 [rows][nh][hd]; rows of no request, and rows that see no key, are zero."""
    q = np.asarray(q, np.float64)
    rows, nh = q.shape[:2]
    nkv = pages.shape[1]
    scale = 1 / np.sqrt(hd) if scale is None else scale
    out = np.zeros((rows, nh, hd))
    for r in range(len(kv_len)):
        n, new = int(kv_len[r]), int(cu[r + 1] - cu[r])
        if n <= 0 or new <= 0:
            continue
        k, v = load(pages, hd, bs, [int(table[r][t // bs]) * bs + t % bs for t in range(n)])
        for i in range(new):
            see = n - new + i + 1
            if see <= 0:
                continue
            for h in range(nh):
                kk, vv = k[:see, h // (nh // nkv)], v[:see, h // (nh // nkv)]
                s = kk @ q[cu[r] + i, h] * scale
                p = np.exp(s - s.max())
                y = p @ vv / p.sum()
                if gate is not None:
                    y = y / (1 + np.exp(-np.asarray(gate[cu[r] + i, h], np.float64)))
                out[cu[r] + i, h] = y
    return out


def plan(ctx, add, table, bs, free, free_count, n_pages, max_tokens):
    """One request after the other. Returns a dict of the outputs (table and free as copies)."""
    n, width = table.shape
    table, free = table.copy(), free.copy()
    stack = [int(x) for x in free[:free_count]]
    need_of = lambda t: -(-t // bs)  # noqa: E731
    for r in range(n):
        if add[r] < 0:
            stack += [int(x) for x in table[r, :min(need_of(max(int(ctx[r]), 0)), width)]]
    stack = stack[:n_pages]
    free[:len(stack)] = stack
    cu, kv_len, rows, refused, dry = [0], [], [], 0, False
    for r in range(n):
        c, new = max(int(ctx[r]), 0), max(int(add[r]), 0)
        have, want, first = need_of(c), need_of(c + new), cu[-1]
        cu.append(first + new)
        ok = new == 0 or (want <= width and first + new <= max_tokens)
        if ok and want > have and new:
            if dry or want - have > len(stack):
                ok, dry = False, True  # nobody overtakes a request that waits for pages
            else:
                for j in range(have, want):
                    table[r, j] = stack.pop()
        refused += not ok
        kv_len.append(c + new if ok and add[r] >= 0 else 0)
        for i in range(new):
            if first + i < max_tokens:
                rows.append((int(table[r, (c + i) // bs]) * bs + (c + i) % bs, c + i, r) if ok else (-1, -1, r))
    rows += [(-1, -1, -1)] * (max_tokens - len(rows))
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    return {"table": table, "free": free, "free_count": len(stack), "cu": i32([min(x, max_tokens) for x in cu]),
            "kv_len": i32(kv_len), "slots": np.array([x[0] for x in rows], np.int64), "positions": i32([x[1] for x in rows]),
            "requests": i32([x[2] for x in rows]), "status": refused}
