"""Softmax differential attention, rotary positions of several axes and the 4-bit cache, from their
definitions in float64 (any device), with the bounds that the roundings of a computation in fewer bits
stay within.  Test-only."""
from __future__ import annotations

import math

import torch


def hidden(b, nq, nk, causal=True, q_offset=None, kv_lens=None, device="cpu"):
    """(b, nq, nk): True where row i does not see key j."""
    off = torch.full((b,), max(nk - nq, 0)) if q_offset is None else torch.as_tensor(q_offset).expand(b)
    lens = torch.full((b,), nk) if kv_lens is None else torch.as_tensor(kv_lens).clamp(0, nk)
    i = torch.arange(nq, device=device)[None, :, None] + off.to(device).long()[:, None, None]
    j = torch.arange(nk, device=device)[None, None, :]
    hide = j >= lens.to(device).long()[:, None, None]
    return (hide | (j > i)) if causal else hide.expand(b, nq, nk)


def lambda_rows(lam, b, h, n, device):
    lam = torch.as_tensor(lam, dtype=torch.float64, device=device)
    if lam.numel() == 1:
        lam = lam.reshape(1, 1, 1)
    elif lam.dim() == 1:
        lam = lam[None, :, None]
    return lam.expand(b, h, n)[..., None]


def weights(q, k, scale, hide):
    """Softmax map of one branch; a row that sees nothing is zero.  k's heads are repeated."""
    s = (q @ k.transpose(2, 3)) * scale
    s = s.masked_fill(hide[:, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
    t = e.sum(-1, keepdim=True)
    return e / torch.where(t > 0, t, 1.0)


def attention(q1, q2, k1, k2, v, lam, scale=None, causal=True, q_offset=None, kv_lens=None, dout=None, u=0.0):
    """Outputs (and with dout the gradients) by name, and under name + "_off" how far from them a
    computation may be whose inputs are these and that rounds weights, score gradients and outputs
    relatively by at most u and everything else to 24 bits.

    With f = 2^-24 and sums of n terms off by at most n f times the sum of magnitudes, to first order: a
    score is off by D = (d + 2) f s sum|q||k|; in base 2 its exponent rounds twice, at most 3 |score| f more, with
    the maximum's; so a weight P is off by P (2 max D + ...), twice because its sum is off too.  Row
    sums r = sum(dO O) come from outputs rounded by u, or by f where they are kept longer: u is counted."""
    x = [t.detach().double() for t in (q1, q2, k1, k2, v)]
    q, k, v = x[:2], x[2:4], x[4]
    b, h, n, d = q[0].shape
    hk, nk, dv = v.shape[1:]
    g = h // hk
    s = 1 / math.sqrt(d) if scale is None else scale
    hide = hidden(b, n, nk, causal, q_offset, kv_lens, v.device)
    up = lambda t: t.repeat_interleave(g, 1)  # noqa: E731
    down = lambda t: t.reshape(b, hk, g, *t.shape[2:]).sum(2)  # noqa: E731
    kk, vv = [up(t) for t in k], up(v)
    lam4 = lambda_rows(lam, b, h, n, v.device)
    f = 2.0 ** -24
    p, pe, o = [], [], []
    for y in range(2):
        w = weights(q[y], kk[y], s, hide)
        sc = ((q[y].abs() @ kk[y].abs().transpose(2, 3)) * s).masked_fill(hide[:, None], 0.0)
        p.append(w)
        pe.append(w * (2 * (d + 8) * f * sc.amax(-1, keepdim=True) + (nk + 8) * f))
        o.append(w @ vv)
    a = p[0] - lam4 * p[1]
    big = p[0] + lam4.abs() * p[1]
    a_off = u * big + pe[0] + lam4.abs() * pe[1] + nk * f * big
    res = {"out": a @ vv}
    res["out_off"] = u * res["out"].abs() + a_off @ vv.abs()
    if dout is None:
        return res
    do = dout.detach().double()
    dp = do @ vv.transpose(2, 3)
    dp_abs = do.abs() @ vv.abs().transpose(2, 3)
    r = [(do * t).sum(-1, keepdim=True) for t in o]
    # r_2 from O_2, r_1 = dO O + lambda r_2; each output off by its own bound
    o2_off = u * o[1].abs() + (u * p[1] + pe[1] + nk * f * p[1]) @ vv.abs()
    r2_off = (do.abs() * (o2_off + dv * f * o[1].abs())).sum(-1, keepdim=True)
    r1_off = (do.abs() * (res["out_off"] + dv * f * res["out"].abs())).sum(-1, keepdim=True) + lam4.abs() * r2_off
    names = ("dq1", "dk1"), ("dq2", "dk2")
    for y, r_off in ((0, r1_off), (1, r2_off)):
        c = 1.0 if y == 0 else -lam4
        ds = p[y] * (dp - r[y]) * c
        ds_off = (c.abs() if y else 1.0) * (p[y] * (r_off + (dv + 4) * f * dp_abs) + pe[y] * (dp - r[y]).abs()) + (u + 4 * f) * ds.abs()
        ds_off = ds_off + (n + nk) * f * ds.abs()
        dq, dk = s * (ds @ kk[y]), s * (ds.transpose(2, 3) @ q[y])
        res[names[y][0]] = dq
        res[names[y][0] + "_off"] = u * dq.abs() + s * (ds_off @ kk[y].abs())
        res[names[y][1]] = down(dk)
        res[names[y][1] + "_off"] = u * down(dk).abs() + s * down(ds_off.transpose(2, 3) @ q[y].abs()) + h * f * down(dk.abs())
    res["dv"] = down(a.transpose(2, 3) @ do)
    res["dv_off"] = u * res["dv"].abs() + down((a_off + n * f * big).transpose(2, 3) @ do.abs())
    lt = torch.as_tensor(lam, dtype=torch.float64)
    shape = (1, 1, 1) if lt.numel() == 1 else (1, h, 1) if lt.dim() == 1 else tuple(lt.shape)

    def to_lambda(t):
        t = t[..., 0]
        for y, m in enumerate(shape):
            if m == 1:
                t = t.sum(y, keepdim=True)
        return t.reshape(lt.shape)

    res["dlam"] = to_lambda(-r[1])
    rows = b * h * n
    res["dlam_off"] = to_lambda(r2_off + min(rows, 4096) * f * r[1].abs()) + u * res["dlam"].abs()
    return res


def rotary(x, positions, inv_freq, sections, interleaved=False):
    """x turned, in float64."""
    x = x.detach().double()
    pairs = inv_freq.shape[0]
    axis = [a for a, m in enumerate(sections) for _ in range(m)]
    ang = positions.double()[axis].permute(1, 2, 0)[:, None] * inv_freq.double()
    c, s = ang.cos(), ang.sin()
    y = x.clone()
    at = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    return y


def held4(x):
    """The values a 4-bit cache holds for rows x (..., width): groups of 64 with m = bf16(min), s =
    bf16((max - m) / 15) rounded as 32-bit arithmetic rounds (the division in float64 first: torch multiplies 32-bit
    values on a GPU by the rounded reciprocal of a number instead), codes decided in float64."""
    y = x.detach().float().unflatten(-1, (-1, 64))
    m = y.amin(-1, keepdim=True).bfloat16()
    s = ((y.amax(-1, keepdim=True) - m.float()).double() / 15.0).float().bfloat16()
    s = torch.where(s.float() >= 2.0 ** -100, s, 0.0).double()
    code = ((y.double() - m.double()) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15) * (s > 0)
    val = m.double() + s * code
    bad = ~torch.isfinite(y).all(-1, keepdim=True) | ~torch.isfinite(s) | ~torch.isfinite(m)
    return torch.where(bad, math.nan, val).flatten(-2)
