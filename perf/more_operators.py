"""Serving over pages and the norm of the heads' outputs, as cases that can be timed and compared.

A case is one pass through one of the operators. With `own` false a pass computes it in elementary
torch operations; with `own` true it makes the framework's calls. The kinds:

  append  the rows of new tokens enter a paged cache, queries and keys turned by their positions on
          the way
  attend  softmax differential attention of new tokens over the pages that hold their sequences
  norm    layer norm (or, without the mean, RMS norm) over the last axis; with "grad" a training
          step: forward and every gradient

The paged cache: k1, k2 (pages, hk, page, d) and v (pages, hk, page, dv). Position p of sequence b is row
p % page of page table[b, p // page]. Sequence b held lengths[b] positions before its new rows, of
which row i stands at lengths[b] + i and sees the positions up to its own. New rows come as a batch
("even": as many of each sequence), as a padded batch with their counts ("padded"), or packed behind each
other ("packed": sequence b has the rows starts[b] .. starts[b + 1] - 1); rows of no sequence are zero.

Rotary: pair p, values p and p + rot/2 of a row or 2 p and 2 p + 1, turns by its position times inv_freq[p].
Attention: out = (softmax(s q1 k1^T + M) - lambda softmax(s q2 k2^T + M)) v with s = 1/sqrt(d).
Rows of attention lie in (B, N, H, d) memory order, as a projection writes them.
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5


def _paged(name, kind, dtype, b, h, hk, new, held, d, dv, page, form="even", mix="even", rot=0, interleaved=False):
    """b sequences of up to `new` new rows behind up to `held` rows. mix: "even" all alike, "ragged" from
    half of them up, "mixed" one sequence with `new` rows and one row for each of the others."""
    case = {"kind": kind, "dtype": dtype, "b": b, "h": h, "hk": hk, "new": new, "held": held, "d": d, "dv": dv, "page": page,
            "form": form, "mix": mix}
    if kind == "append":
        case.update(rot=rot, interleaved=interleaved)
    return dict(case, name=name) if name else case


def _norm(name, dtype, b, h, n, width, grad, weight="row", bias=False, center=True, wide_weight=False):
    """Rows (b, h, n, width), h = 0: (b, n, width). weight: "none", "row" (width,) or "heads" (h, width)."""
    case = {"kind": "norm", "dtype": dtype, "b": b, "h": h, "n": n, "width": width, "grad": grad, "weight": weight,
            "bias": bias, "center": center, "wide_weight": wide_weight}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one new token of each of a few conversations: the smallest call of a serving step
        _paged("append-token", "append", "bf16", 8, 16, 4, 1, 900, 128, 128, 64, mix="ragged", rot=128),
        # a step that packs prompts of unequal lengths
        _paged("append-prompts", "append", "bf16", 4, 32, 8, 2048, 0, 128, 128, 64, "packed", "ragged", rot=128),
        # float32 rows of a padded batch, three quarters of each rotated in interleaved pairs
        _paged("append-fp32-padded", "append", "fp32", 3, 12, 12, 500, 333, 64, 128, 16, "padded", "ragged", rot=48, interleaved=True),
        # the newest token of one short conversation: nothing but latency
        _paged("step-short", "attend", "bf16", 1, 8, 8, 1, 999, 64, 64, 64),
        # the newest tokens of a full batch of long conversations of unequal lengths
        _paged("step-long", "attend", "bf16", 32, 32, 8, 1, 8191, 128, 128, 64, mix="ragged"),
        # chunks of two prompts behind what the cache holds already, odd lengths
        _paged("chunk", "attend", "bf16", 2, 16, 4, 500, 3855, 128, 128, 64),
        # one chunk deep in a long document
        _paged("chunk-long", "attend", "bf16", 1, 16, 4, 2048, 30000, 128, 128, 256),
        # a serving step: a chunk of one prompt packed with the newest tokens of other conversations
        _paged("mixed", "attend", "fp16", 24, 16, 4, 700, 5000, 64, 128, 32, "packed", "mixed"),
        # the norm of every head's output in a training step of differential attention
        _norm("norm-heads-train", "bf16", 4, 16, 4096, 128, True, "heads", center=False),
        # the norm before a wide layer, a training step
        _norm("norm-wide-train", "bf16", 4, 0, 4096, 4096, True, "row", True),
        # float32 rows of an odd width, a training step
        _norm("norm-odd-train", "fp32", 3, 0, 1371, 1111, True, "row", True),
        # the norm of the newest tokens' heads
        _norm("norm-token", "bf16", 8, 16, 1, 128, False, "row", center=False, wide_weight=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32", "fp16"])
    if kind == "norm":
        heads = rng.random() < 0.5
        width = rng.choice([64, 128, 128, 256, 72, 100]) if heads else _log(rng, 33, 9000)
        if not heads and rng.random() < 0.6:
            width = max(width // 64, 1) * 64
        h = rng.randint(1, 16) if heads else 0
        b = rng.randint(1, 4)
        n = _log(rng, 1, max(min(4000, 30_000_000 // (b * max(h, 1) * width)), 2))
        return _norm(None, dtype, b, h, n, width, rng.random() < 0.6, rng.choice(["none", "row", "heads"] if heads else ["none", "row", "row"]),
                     rng.random() < 0.4, rng.random() < 0.5, rng.random() < 0.5)
    d, dv = rng.choice([(64, 64), (64, 128), (128, 128), (128, 128), (128, 256)])
    hk = rng.choice([1, 2, 3, 4, 8])
    h = hk * rng.choice([1, 2, 4, 5, 8])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    mix = rng.choice(["even", "ragged", "mixed"])
    form = rng.choice(["even", "packed"]) if mix == "even" else rng.choice(["packed", "packed", "padded"])
    if kind == "append":
        b = rng.randint(1, 12)
        rot = rng.choice([0, d, d, d // 2, d * 3 // 4])
        return _paged(None, kind, dtype, b, h, hk, _log(rng, 1, 1500 // b + 1), _log(rng, 1, 1500), d, dv, page, form, mix, rot,
                      rng.random() < 0.4)
    if rng.random() < 0.5:  # newest tokens, or a few drafted ones
        new = rng.choice([1, 1, 1, 2, 4, 7])
        return _paged(None, kind, dtype, rng.randint(1, 24), h, hk, new, _log(rng, 1, 8000), d, dv, page, form, mix)
    h = hk * min(h // hk, max(16 // hk, 1))
    long = 4000 if dtype != "fp32" else 1200
    return _paged(None, kind, dtype, rng.randint(1, 3) if mix != "mixed" else rng.randint(2, 20), h, hk, _log(rng, 8, long // 4),
                  _log(rng, 1, long), d, dv, page, form, mix)


# ------------------------------------------------------------------ inputs
def _counts(case):
    """(new rows, rows held before) of each sequence."""
    b, new, held, mix = case["b"], case["new"], case["held"], case["mix"]
    if mix == "even":
        return [new] * b, [held] * b
    if mix == "mixed":
        return [new] + [1] * (b - 1), [held - (i * held) // (2 * b) for i in range(b)]
    if case["form"] == "even":  # as many new rows of each
        return [new] * b, [held - (i * held) // (2 * b) for i in range(b)]
    return [new - (i * new) // (2 * b) for i in range(b)], [held - (i * held) // (2 * b) for i in range(b)]


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _rows(g, b, h, n, d, dtype, spread=1.0):
    return (torch.randn(b, n, h, d, generator=g, device=g.device) * spread).to(_DTYPE[dtype]).transpose(1, 2)


def _drawn(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = case["dtype"]
    if case["kind"] == "norm":
        b, h, n, width = case["b"], case["h"], case["n"], case["width"]
        like = (lambda: _rows(g, b, h, n, width, dt)) if h else lambda: torch.randn(b, n, width, generator=g, device=dev).to(_DTYPE[dt])
        level = 0.5 * torch.randn(width, generator=g, device=dev)
        st = {"case": case, "x": (1.5 * like() + level.to(_DTYPE[dt]))}
        shape = (h, width) if case["weight"] == "heads" else (width,)
        wdt = torch.float32 if case["wide_weight"] else _DTYPE[dt]
        if case["weight"] != "none":
            st["weight"] = (1 + 0.3 * torch.randn(shape, generator=g, device=dev)).to(wdt)
        if case["bias"]:
            st["bias"] = (0.3 * torch.randn(shape, generator=g, device=dev)).to(wdt)
        if case["grad"]:
            st["dy"] = like()
        return st
    b, h, hk, d, dv, page = (case[x] for x in ("b", "h", "hk", "d", "dv", "page"))
    new, held = _counts(case)
    need = [-(-(x + y) // page) for x, y in zip(new, held)]
    pages = sum(need) + 2  # some pages belong to nobody
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((b, max(need) + 1), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    st = {"case": case, "table": table, "lengths": torch.tensor(held, dtype=torch.int32, device=dev)}
    for name, w in (("k1", d), ("k2", d), ("v", dv)):
        st["pool_" + name] = torch.randn(pages, hk, page, w, generator=g, device=dev, dtype=torch.float32).to(_DTYPE[dt])
    lead, n = (1, sum(new)) if case["form"] == "packed" else (b, max(new))
    if case["form"] == "packed":
        st["starts"] = torch.tensor([sum(new[:i]) for i in range(b + 1)], dtype=torch.int32, device=dev)
    elif case["form"] == "padded":
        st["counts"] = torch.tensor(new, dtype=torch.int32, device=dev)
    spread = 1.5 if case["kind"] == "attend" else 1.0
    st["q1"], st["q2"] = _rows(g, lead, h, n, d, dt, spread), _rows(g, lead, h, n, d, dt, spread)
    if case["kind"] == "attend":
        st["lam"] = (0.2 + 0.6 * torch.rand(h, generator=g, device=dev)).to(_DTYPE[dt])
        return st
    st["k1"], st["k2"], st["v"] = _rows(g, lead, hk, n, d, dt), _rows(g, lead, hk, n, d, dt), _rows(g, lead, hk, n, dv, dt)
    pairs = case["rot"] // 2
    if pairs:
        st["inv_freq"] = torch.exp(-math.log(10000.0) / pairs * torch.arange(pairs, device=dev, dtype=torch.float64)).float()
    return st


def prepare(case, seed):
    st = _drawn(case, seed)
    if own and case["kind"] != "norm":
        import tda_amd
        pools = [st.pop("pool_" + x) for x in ("k1", "k2", "v")]
        cache = st["cache"] = tda_amd.PagedKVCache(pools[0].shape[0], case["hk"], case["page"], case["d"], case["dv"],
                                                   dtype=_DTYPE[case["dtype"]], device=pools[0].device)
        for held, pool in zip((cache.k1, cache.k2, cache.v), pools):
            held.copy_(pool)
    return st


# ------------------------------------------------------------------ plain forms
def _row_index(st, case):
    """Of every new row: its batch entry and place along the sequence axis, its sequence, its position."""
    new, held = _counts(case)
    dev = st["table"].device
    lead, at, who, pos = [], [], [], []
    done = 0
    for s, (n, m) in enumerate(zip(new, held)):
        i = torch.arange(n, device=dev)
        lead.append(torch.full_like(i, 0 if case["form"] == "packed" else s))
        at.append(i + (done if case["form"] == "packed" else 0))
        who.append(torch.full_like(i, s))
        pos.append(i + m)
        done += n
    return [torch.cat(x) for x in (lead, at, who, pos)]


def _turn(x, cos, sin, rot, interleaved):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_append(st):
    case = st["case"]
    dt, rot, page = _DTYPE[case["dtype"]], case["rot"], case["page"]
    lead, at, who, pos = _row_index(st, case)

    def turned(x):
        rows = x[lead, :, at].float()  # (rows, heads, width)
        if not rot:
            return rows
        angle = (pos.double()[:, None] * st["inv_freq"].double())[:, None]  # in 64 bits: far positions
        return _turn(rows, angle.cos().float(), angle.sin().float(), rot, case["interleaved"])

    res = []
    for x in (st["q1"], st["q2"]):
        y = torch.zeros_like(x)
        y[lead, :, at] = turned(x).to(dt)
        res.append(y)
    place = st["table"][who, pos // page].long()
    for x in ("k1", "k2", "v"):
        rows = turned(st[x]) if x != "v" else st[x][lead, :, at].float()
        st["pool_" + x][place, :, pos % page] = rows.to(dt)
    return res + [st["pool_" + x] for x in ("k1", "k2", "v")]


def _held(pool, table, n):
    """The first n positions of one sequence: (hk, n, width)."""
    pages, hk, page, w = pool.shape
    return pool[table[: -(-n // page)].long()].transpose(0, 1).reshape(hk, -1, w)[:, :n]


def _softmax(s, hidden):
    s = s.masked_fill(hidden, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_attend(st):
    case = st["case"]
    dt, h, hk, d, dv = _DTYPE[case["dtype"]], case["h"], case["hk"], case["d"], case["dv"]
    new, held = _counts(case)
    q1, q2 = st["q1"], st["q2"]
    out = torch.zeros(*q1.shape[:2], q1.shape[2], dv, dtype=dt, device=q1.device)
    lam = st["lam"].float().view(hk, h // hk, 1, 1)
    done = 0
    for s, (n, m) in enumerate(zip(new, held)):
        lead, rows = (0, slice(done, done + n)) if case["form"] == "packed" else (s, slice(0, n))
        done += n
        k1, k2, v = (_held(st["pool_" + x], st["table"][s], n + m).float() for x in ("k1", "k2", "v"))
        hidden = torch.arange(n + m, device=v.device) > torch.arange(m, m + n, device=v.device)[:, None]

        def weights(q, k):  # the query heads of one key head stand below each other: one product for all of them
            x = q[lead, :, rows].float().reshape(hk, -1, d) @ k.transpose(1, 2)
            return _softmax(x.view(hk, h // hk, n, n + m) * (1 / math.sqrt(d)), hidden)

        a = weights(q1, k1) - lam * weights(q2, k2)
        out[lead, :, rows] = (a.view(hk, -1, n + m) @ v).view(h, n, dv).to(dt)
    return out


def _plain_norm(st):
    case = st["case"]
    dt = _DTYPE[case["dtype"]]
    x = st["x"].float()

    def per_row(w):  # beside the rows
        return w.float() if w.dim() == 1 else w.float()[:, None]

    if case["center"]:
        x = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
    xhat = x * rstd
    y = xhat
    if "weight" in st:
        y = y * per_row(st["weight"])
    if "bias" in st:
        y = y + per_row(st["bias"])
    res = [y.to(dt)]
    if not case["grad"]:
        return res
    dy = st["dy"].float()
    g = dy * per_row(st["weight"]) if "weight" in st else dy
    dx = g - xhat * (g * xhat).mean(-1, keepdim=True)
    if case["center"]:
        dx = dx - g.mean(-1, keepdim=True)
    res.append((dx * rstd).to(dt))
    for name, t in (("weight", dy * xhat), ("bias", dy)):
        if name in st:
            over = (0, 2) if st[name].dim() == 2 else tuple(range(t.dim() - 1))
            res.append(t.sum(over).to(st[name].dtype))
    return res


# ------------------------------------------------------------------ the framework's calls
def _calls(st):
    import tda_amd
    case = st["case"]
    if case["kind"] == "norm":
        args = (st["x"], st.get("weight"), st.get("bias"))
        if not case["grad"]:
            return [tda_amd.layer_norm(*args, eps=_EPS, center=case["center"])]
        leaves = [None if t is None else t.detach().requires_grad_(True) for t in args]
        y = tda_amd.layer_norm(*leaves, eps=_EPS, center=case["center"])
        return [y.detach()] + list(torch.autograd.grad(y, [t for t in leaves if t is not None], st["dy"]))
    cache = st["cache"]
    where = {"starts": st.get("starts"), "counts": st.get("counts")}
    if case["kind"] == "append":
        q1, q2 = cache.append(st["k1"], st["k2"], st["v"], st["table"], st["lengths"], st["q1"], st["q2"],
                              inv_freq=st.get("inv_freq"), interleaved=case["interleaved"], **where)
        return [q1, q2, cache.k1, cache.k2, cache.v]
    return cache.attend(st["q1"], st["q2"], st["lam"], st["table"], st["lengths"], **where)


def run(state):
    if own:
        return _calls(state)
    return {"append": _plain_append, "attend": _plain_attend, "norm": _plain_norm}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "norm":
        rows = case["b"] * max(case["h"], 1) * case["n"]
        values = rows * case["width"]
        # forward: x and y; a training step reads x and dy once and writes y and dx
        return {"bytes": (4 if case["grad"] else 2) * values * size, "flops": (17 if case["grad"] else 7) * values}
    h, hk, d, dv = case["h"], case["hk"], case["d"], case["dv"]
    new, held = _counts(case)
    if case["kind"] == "append":
        values = sum(new) * (2 * (h + hk) * d + hk * dv)
        return {"bytes": 2 * values * size, "flops": 3 * sum(new) * 2 * (h + hk) * case["rot"]}
    cache = sum(x + y for x, y in zip(new, held)) * hk * (2 * d + dv)
    seen = sum(n * m + n * (n + 1) // 2 for n, m in zip(new, held))
    return {"bytes": (cache + sum(new) * h * (2 * d + dv)) * size, "flops": h * seen * (4 * d + 2 * dv)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_attend(st):
    case = st["case"]
    new, held = _counts(case)
    page, group = case["page"], case["h"] // case["hk"]
    scale = case["d"] ** -0.5
    out = torch.zeros(*st["q1"].shape[:3], case["dv"], dtype=torch.float64, device=st["q1"].device)
    first = 0
    for s in range(case["b"]):
        p = torch.arange(held[s] + new[s], device=out.device)
        pg, row = st["table"][s].long()[p // page], p % page
        i = torch.arange(new[s], device=out.device)
        seq, at = (0, i + first) if case["form"] == "packed" else (s, i)
        first += new[s]
        unseen = p[None] > (i + held[s])[:, None]
        for x in range(case["h"]):
            y = x // group
            val = st["pool_v"][pg, y, row].double()
            maps = []
            for q, k in (("q1", "pool_k1"), ("q2", "pool_k2")):
                z = (st[q][seq, x].double()[at] @ st[k][pg, y, row].double().T).mul_(scale)
                z[unseen] = -math.inf
                z -= z.amax(1, keepdim=True)
                z.exp_()
                maps.append((z @ val) / z.sum(1, keepdim=True))
            out[seq, x, at] = maps[0] - st["lam"][x].double() * maps[1]
    return out


def _exact_append(st):
    case = st["case"]
    new, held = _counts(case)
    page, rot = case["page"], case["rot"]
    res = {x: st["pool_" + x].double() for x in ("k1", "k2", "v")}
    res.update({x: torch.zeros(st[x].shape, dtype=torch.float64, device=st[x].device) for x in ("q1", "q2")})
    first = 0
    for s in range(case["b"]):
        i = torch.arange(new[s], device=st["table"].device)
        seq, at = (0, i + first) if case["form"] == "packed" else (s, i)
        first += new[s]
        p = i + held[s]
        for x in ("q1", "q2", "k1", "k2", "v"):
            y = st[x][seq].double()[:, at].clone()
            if rot and x != "v":
                by = torch.polar(torch.ones((), dtype=torch.float64, device=p.device), p.double()[:, None] * st["inv_freq"].double())
                if case["interleaved"]:
                    y[..., :rot] = torch.view_as_real(torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * by).flatten(-2)
                else:
                    z = torch.complex(y[..., : rot // 2], y[..., rot // 2: rot]) * by
                    y[..., : rot // 2], y[..., rot // 2: rot] = z.real, z.imag
            if x in ("q1", "q2"):
                res[x][seq, :, at] = y
            else:
                res[x][st["table"][s].long()[p // page], :, p % page] = y.transpose(0, 1)
    return [res[x] for x in ("q1", "q2", "k1", "k2", "v")]


def _exact_norm(st):
    case = st["case"]
    x = st["x"].double()
    heads = lambda t: t.double().unsqueeze(1) if t.dim() == 2 else t.double()  # noqa: E731
    n = x.shape[-1]
    mu = x.sum(-1, keepdim=True) / n if case["center"] else torch.zeros_like(x[..., :1])
    var = ((x - mu) ** 2).sum(-1, keepdim=True) / n
    r = (var + _EPS) ** -0.5
    z = (x - mu) * r
    w = heads(st["weight"]) if "weight" in st else torch.ones((), dtype=torch.float64, device=x.device)
    res = [z * w + (heads(st["bias"]) if "bias" in st else 0.0)]
    if case["grad"]:
        dy = st["dy"].double()
        g = dy * w
        c2 = (g * z).sum(-1, keepdim=True) / n
        c1 = g.sum(-1, keepdim=True) / n if case["center"] else 0.0
        res.append(r * (g - c1 - z * c2))
        for name, t in (("weight", dy * z), ("bias", dy)):
            if name in st:
                res.append(t.sum(2).sum(0) if st[name].dim() == 2 else t.flatten(0, -2).sum(0))
    return res


def exact(case, seed):
    st = _drawn(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "norm": _exact_norm}[case["kind"]](st)
