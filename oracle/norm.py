"""Layer norm from its definition in float64 (any device), with the bounds that the roundings of a computation in 32
bits stay within.  Test-only."""
from __future__ import annotations

import torch

F = 2.0 ** -24
CHAIN = 64  # additions one after the other in a sum over a row: at most 16 of a lane, 7 between lanes, 16 between waves


def layer_norm(x, weight=None, bias=None, eps=1e-5, center=True, dy=None, u=0.0, u_w=0.0):
    """y, and with dy: dx, dweight, dbias, by name, and under name + "_off" how far a computation in 32 bits may be whose
    results are rounded relatively by at most u (those of the weights by u_w).

    To first order: a sum of n terms is off by CHAIN F sum |terms| (rows: as many as there are); the mean by that over n;
    a difference from the mean by the mean's error and F; the variance by the squares' errors; rstd relatively by half
    of the variance's error over itself and 4 F (sum with eps, root and quotient)."""
    x = x.detach().double()
    one = torch.ones((), dtype=torch.float64, device=x.device)
    beside = lambda t: t.detach().double()[:, None] if t.dim() == 2 else t.detach().double()  # noqa: E731
    w = one if weight is None else beside(weight)
    b = 0 * one if bias is None else beside(bias)
    avg = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    mean = avg(x) if center else 0 * x[..., :1]
    mean_off = CHAIN * F * avg(x.abs()) if center else 0 * mean
    d = x - mean
    d_off = mean_off + F * d.abs()
    var = avg(d * d)
    var_off = (CHAIN + 4) * F * var + 2 * mean_off * avg(d.abs()) + mean_off ** 2 + 2 * F * var
    rstd = (var + eps) ** -0.5
    r_rel = 0.5 * var_off / (var + eps) + 4 * F
    z = d * rstd
    z_off = d_off * rstd + z.abs() * (r_rel + F)
    y = z * w + b
    res = {"y": y, "y_off": u * y.abs() + w.abs() * z_off + 2 * F * (z * w).abs() + F * y.abs()}
    if dy is None:
        return res
    dy = dy.detach().double()
    g = dy * w
    c1 = avg(g) if center else 0 * mean
    c2 = avg(g * z)
    c1_off = (CHAIN + 2) * F * avg(g.abs()) if center else 0 * mean
    c2_off = (CHAIN + 4) * F * avg((g * z).abs()) + avg(g.abs() * z_off)
    inner = g - c1 - z * c2
    inner_off = 2 * F * g.abs() + c1_off + z.abs() * c2_off + z_off * c2.abs() + 3 * F * (g.abs() + c1.abs() + (z * c2).abs())
    res["dx"] = rstd * inner
    res["dx_off"] = u * res["dx"].abs() + rstd * inner_off + res["dx"].abs() * (r_rel + F)
    for name, like, t, t_off in (("dweight", weight, dy * z, dy.abs() * z_off), ("dbias", bias, dy, 0 * dy)):
        if like is None:
            continue
        over = (0, 2) if like.dim() == 2 else tuple(range(t.dim() - 1))
        rows = t.numel() // max(like.numel(), 1)
        total = lambda t: t.sum(over) if over else t  # noqa: E731
        res[name] = total(t)
        res[name + "_off"] = u_w * res[name].abs() + total(t_off) + (rows + 16) * F * total(t.abs())
    return res
