"""The paged cache from its definition in float64 (any device).  Test-only."""
from __future__ import annotations

import torch

from . import softmax


def place(table, page_size, pages, s, p):
    """(page, row) of position p of sequence s, None where there is none."""
    if not 0 <= p < table.shape[1] * page_size:
        return None
    page = int(table[s, p // page_size])
    return (page, p % page_size) if 0 <= page < pages else None


def rows_of(s, lengths, rows, starts=None, counts=None):
    """(batch entry, first row, rows, position of the first) of sequence s."""
    if starts is not None:
        a = min(max(int(starts[s]), 0), rows)
        return 0, a, min(max(int(starts[s + 1]), a), rows) - a, int(lengths[s])
    n = rows if counts is None else min(max(int(counts[s]), 0), rows)
    return s, 0, n, int(lengths[s])


def held(pool, table, s, n):
    """The first n positions of sequence s: (kv_heads, n, width), zeros where the table has no page."""
    pages, hk, size, w = pool.shape
    idx = table[s].long().cpu()
    idx = idx[: -(-n // size)] if n else idx[:0]
    ok = (idx >= 0) & (idx < pages)
    x = pool[idx.clamp(0, pages - 1).to(pool.device)] * 1
    x[~ok.to(pool.device)] = 0
    return x.transpose(0, 1).reshape(hk, -1, w)[:, :n]


def attend(q1, q2, pools, lam, table, lengths, scale=None, starts=None, counts=None, u=0.0):
    """out and out_off (softmax.attention's bound) of every row; zeros for rows of no sequence."""
    lead, h, rows, d = q1.shape
    dv = pools[2].shape[3]
    cap = table.shape[1] * pools[0].shape[2]
    res = {n: torch.zeros((lead, h, rows, dv), dtype=torch.float64, device=q1.device) for n in ("out", "out_off")}
    lam = softmax.lambda_rows(lam, lead, h, rows, q1.device)[..., 0]
    for s in range(table.shape[0]):
        b, r0, n, at = rows_of(s, lengths, rows, starts, counts)
        length = min(max(at + n, 0), cap)
        if n == 0 or length == 0:
            continue
        k1, k2, v = (held(p, table, s, length)[None] for p in pools)
        sel = slice(r0, r0 + n)
        got = softmax.attention(q1[b:b + 1, :, sel], q2[b:b + 1, :, sel], k1, k2, v, lam[b:b + 1, :, sel], scale, q_offset=at, u=u)
        for name in res:
            res[name][b, :, sel] = got[name][0]
    return res
