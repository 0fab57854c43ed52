"""The operators around softmax differential attention, as cases that can be timed and compared.

A case is one pass through one of them. With `own` false a pass computes it in elementary torch
operations; with `own` true it makes the framework's calls. The kinds:

  train    a training step of the attention: forward and every gradient
  prefill  a forward of many query rows (a whole prompt, or a chunk behind a cache)
  decode   a forward of the newest token of each sequence over a cache in the queries' type
  kv4      a decoding step over a cache held in 4 bits: the newest token's rows enter the cache, then
           it attends
  store    a prompt's rows enter the 4-bit cache and are read back (as a chunk of many rows does)
  rotary   rotary positions of several axes on q1, q2, k1, k2; with "grad" the gradients too

Attention: out = (softmax(s q1 k1^T + M) - lambda softmax(s q2 k2^T + M)) v with s = 1/sqrt(d); M hides
the keys behind a row's own position and behind its sequence's length; a row that sees no key is zero.
h query heads share hk key/value heads. Rows lie in (B, N, H, d) memory order, as a projection
writes them.

The 4-bit cache: each row of each tensor in groups of 64 values x. m = bf16(min x),
s = bf16((max x - m) / 15) in 32 bits, code = min(max(rint((x - m) / s), 0), 15), value m + s code.
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_GROUP = 64
_SMALL = 2.0 ** -100  # a step below this is zero


def _att(name, kind, dtype, b, h, hk, nq, nk, d, dv, ragged=False):
    case = {"kind": kind, "dtype": dtype, "b": b, "h": h, "hk": hk, "nq": nq, "nk": nk, "d": d, "dv": dv, "ragged": ragged}
    return dict(case, name=name) if name else case


def _rot(name, dtype, b, h, hk, n, d, rot, axes, grad, interleaved=False, far=0):
    case = {"kind": "rotary", "dtype": dtype, "b": b, "h": h, "hk": hk, "n": n, "d": d, "rot": rot, "axes": axes,
            "grad": grad, "interleaved": interleaved, "far": far}
    return dict(case, name=name) if name else case


def listed():
    return [
        # training with heads of 64 whose values are twice as wide, as differential heads often are
        _att("train-values-wide", "train", "bf16", 4, 16, 16, 2048, 2048, 64, 128),
        # training a longer context whose query heads share keys and values
        _att("train-shared-heads", "train", "bf16", 2, 16, 4, 4096, 4096, 128, 128),
        # a float32 training step on a padded batch of an odd length
        _att("train-fp32-padded", "train", "fp32", 2, 12, 12, 1111, 1111, 64, 64, ragged=True),
        # scoring a long document
        _att("prefill-long", "prefill", "bf16", 1, 16, 4, 16384, 16384, 128, 128),
        # a chunk of a prompt behind what the cache holds already, both of odd lengths
        _att("prefill-chunk", "prefill", "bf16", 2, 16, 4, 500, 4355, 128, 128),
        # the newest token of one short conversation: the smallest serving call, nothing but latency
        _att("decode-short", "decode", "bf16", 1, 8, 8, 1, 1000, 64, 64),
        # the newest token of a batch of long conversations of unequal lengths
        _att("decode-long", "decode", "bf16", 32, 32, 8, 1, 8192, 128, 128, ragged=True),
        # the same two over a cache in 4 bits, the token's own rows entering it first
        _att("kv4-short", "kv4", "bf16", 1, 8, 8, 1, 1000, 64, 64),
        _att("kv4-long", "kv4", "bf16", 32, 32, 8, 1, 8192, 128, 128, ragged=True),
        # a prompt of a batch entering the 4-bit cache
        _att("kv4-store", "store", "bf16", 4, 32, 8, 2048, 2048, 128, 128),
        # one new token of each of a few conversations about images, far into their contexts
        _rot("rotary-token", "bf16", 8, 16, 4, 1, 128, 128, 3, False, far=100000),
        # a training step on video: three axes on part of each head, forward and backward
        _rot("rotary-train", "bf16", 4, 16, 16, 4096, 128, 96, 3, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["train", "train", "prefill", "prefill", "decode", "kv4", "store", "rotary"])
    d, dv = rng.choice([(64, 64), (64, 128), (128, 128), (128, 128), (128, 256)])
    hk = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 4, 5, 8])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32", "fp16"])
    b = rng.randint(1, 4)
    ragged = rng.random() < 0.4
    if kind == "train":
        h = min(hk * group, 16) // hk * hk
        n = _log(rng, 17, 2200 if dtype == "bf16" else 1100)
        return _att(None, kind, dtype, b, h, hk, n, n, d, dv, ragged)
    if kind == "prefill":
        h = min(hk * group, 16) // hk * hk
        nk = _log(rng, 40, 6000 if dtype == "bf16" else 2000)
        nq = nk if rng.random() < 0.5 else _log(rng, 18, nk)
        return _att(None, kind, dtype, b, h, hk, nq, nk, d, dv, ragged and nq == nk)
    if kind == "rotary":
        axes = rng.randint(1, 4)
        rot = rng.choice([d, d, d // 2, d * 3 // 4])
        return _rot(None, dtype, b, hk * group, hk, _log(rng, 1, 4000), d, rot, axes, rng.random() < 0.5,
                    rng.random() < 0.4, rng.choice([0, 0, 5000, 1000000]))
    nk = _log(rng, 2, 9000)
    b = rng.randint(1, 24)
    if kind == "decode":
        return _att(None, kind, dtype, b, hk * group, hk, 1, nk, d, dv, ragged)
    if kind == "kv4":
        return _att(None, kind, rng.choice(["bf16", "bf16", "fp32"]), b, hk * group, hk, 1, nk, d, dv, ragged)
    n = _log(rng, 1, 2500)
    return _att(None, "store", rng.choice(["bf16", "bf16", "fp32"]), min(b, 4), hk * group, hk, n, n, d, dv)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Each sequence's keys: all of them, or from half of them up."""
    b, nk = case["b"], case["nk"]
    return [nk - (i * nk) // (2 * b) if case["ragged"] else nk for i in range(b)]


def _sections(case):
    """The pairs of a head dealt to the axes: the first axis gets what is left over."""
    pairs, axes = case["rot"] // 2, case["axes"]
    each = pairs // (axes + 1) if axes > 1 else pairs
    return [pairs - each * (axes - 1)] + [each] * (axes - 1)


def _rows(g, b, h, n, d, dtype, spread=1.0):
    dev = g.device
    return (torch.randn(b, n, h, d, generator=g, device=dev) * spread).to(_DTYPE[dtype]).transpose(1, 2)


def _context(g, case, n):
    """Keys and values of n positions: keys with channels of their own level, as caches hold them."""
    b, hk, d, dv, dt = case["b"], case["hk"], case["d"], case["dv"], case["dtype"]
    level = 1.5 * torch.randn(1, hk, 1, d, generator=g, device=g.device)
    k1, k2 = ((_rows(g, b, hk, n, d, "fp32") + level).to(_DTYPE[dt]) for _ in range(2))
    return k1, k2, _rows(g, b, hk, n, dv, dt)


def _drawn(case, seed):
    """The inputs. Of "kv4": the queries, and the rows of every position, the newest ones among them."""
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev).manual_seed(seed)
    kind, dt, b, h, hk, d = case["kind"], case["dtype"], case["b"], case["h"], case["hk"], case["d"]
    if kind == "rotary":
        n = case["n"]
        st = {"case": case, "xs": [_rows(g, b, x, n, d, dt) for x in (h, h, hk, hk)]}
        pos = torch.arange(n, device=dev).expand(case["axes"], b, n)
        step = torch.randint(1, 40, (case["axes"], b, 1), generator=g, device=dev)
        st["positions"] = pos // step + torch.randint(0, case["far"] + 1, (case["axes"], b, 1), generator=g, device=dev)
        pairs = case["rot"] // 2
        st["inv_freq"] = torch.exp(-math.log(10000.0) / pairs * torch.arange(pairs, device=dev, dtype=torch.float64)).float()
        st["sections"] = _sections(case)
        if case["grad"]:
            st["douts"] = [_rows(g, b, x, n, d, dt) for x in (h, h, hk, hk)]
        return st
    nq, nk, dv = case["nq"], case["nk"], case["dv"]
    st = {"case": case, "q1": _rows(g, b, h, nq, d, dt, 1.5), "q2": _rows(g, b, h, nq, d, dt, 1.5)}
    st["lam"] = (0.2 + 0.6 * torch.rand(h, generator=g, device=dev)).to(_DTYPE[dt])
    st["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    if kind in ("train", "prefill", "decode"):
        st["k1"], st["k2"] = _rows(g, b, hk, nk, d, dt), _rows(g, b, hk, nk, d, dt)
        st["v"] = _rows(g, b, hk, nk, dv, dt)
        if kind == "train":
            st["dout"] = _rows(g, b, h, nq, dv, dt)
        return st
    st["k1"], st["k2"], st["v"] = _context(g, case, nk)
    st["start"] = torch.zeros(b, dtype=torch.int32, device=dev) if kind == "store" else st["lens"] - 1
    return st


def prepare(case, seed):
    st = _drawn(case, seed)
    if case["kind"] not in ("store", "kv4"):
        return st
    b, hk, nk, d, dv = case["b"], case["hk"], case["nk"], case["d"], case["dv"]
    context = [st[x] for x in ("k1", "k2", "v")]
    if case["kind"] == "kv4":  # the rows that a step brings; the cache holds the others
        at = st["start"].long().view(b, 1, 1, 1)
        st["k1"], st["k2"], st["v"] = (x.gather(2, at.expand(b, hk, 1, x.shape[3])) for x in context)
    if own:
        import tda_amd
        st["cache"] = tda_amd.Int4KVCache(b, hk, nk, d, dv, device=st["lens"].device)
        if case["kind"] == "kv4":
            st["cache"].append(*context, start=torch.zeros_like(st["lens"]))
    elif case["kind"] == "kv4":
        st["packed"] = [_pack(*_quantise(x)) for x in context]
    return st


# ------------------------------------------------------------------ plain forms
def _softmax(s, hidden):
    s = s.masked_fill(hidden, -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(s - m)
    return e / e.sum(-1, keepdim=True).clamp_min(1e-37)


def _attend(q1, q2, k1, k2, v, lam, lens, offset):
    """The formula on tensors of one type; offset: position of the first query row, one of each sequence."""
    b, h, nq, d = q1.shape
    hk, nk, dv = v.shape[1:]
    i = torch.arange(nq, device=v.device).view(1, nq, 1) + offset.view(b, 1, 1)
    j = torch.arange(nk, device=v.device).view(1, 1, nk)
    hidden = ((j > i) | (j >= lens.view(b, 1, 1))).view(b, 1, 1, nq, nk)

    def weights(q, k):  # the query heads of one key head stand below each other: one product for all of them
        s = q.reshape(b, hk, -1, d) @ k.transpose(2, 3)
        return _softmax(s.view(b, hk, h // hk, nq, nk) * (1 / math.sqrt(d)), hidden)

    a = weights(q1, k1) - lam.view(1, hk, h // hk, 1, 1) * weights(q2, k2)
    return (a.view(b, hk, -1, nk) @ v).view(b, h, nq, dv)


def _offset(st):
    case = st["case"]
    if case["kind"] in ("decode", "kv4"):
        return st["lens"].long() - case["nq"]
    return torch.full_like(st["lens"], case["nk"] - case["nq"]).long()


def _quantise(x):
    x = x.float()
    y = x.reshape(*x.shape[:-1], -1, _GROUP)
    m = y.amin(-1, keepdim=True).to(torch.bfloat16)
    s = ((y.amax(-1, keepdim=True) - m.float()) / 15.0).to(torch.bfloat16)
    s = torch.where(s < _SMALL, 0.0, s)
    t = (y.double() - m.double()) / s.double()  # in 64 bits: a value next to a border
    code = torch.where(s > 0, t.round().clamp(0, 15), 0.0).to(torch.uint8)
    return code, s, m


def _pack(code, s, m):
    return code[..., 0::2] | (code[..., 1::2] << 4), s, m


def _value(code, s, m):
    x = m.float() + s.float() * code.float()
    return x.flatten(-2)


def _unpack(byte, s, m):
    return torch.stack((byte & 15, byte >> 4), -1).flatten(-2), s, m


def _turn(x, cos, sin, rot, interleaved):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _angles(st):
    """(b, 1, n, pairs) in 64 bits: far positions."""
    at = st["positions"].double()
    axis = torch.repeat_interleave(torch.arange(len(st["sections"]), device=at.device),
                                   torch.tensor(st["sections"], device=at.device))
    return (at[axis].permute(1, 2, 0) * st["inv_freq"].double()).unsqueeze(1)


def _plain(st):
    case = st["case"]
    kind, dt = case["kind"], _DTYPE[case["dtype"]]
    if kind == "rotary":
        angle = _angles(st)
        cos, sin = angle.cos().float(), angle.sin().float()
        rot, inter = case["rot"], case["interleaved"]
        res = [_turn(x.float(), cos, sin, rot, inter).to(dt) for x in st["xs"]]
        if case["grad"]:
            res += [_turn(x.float(), cos, -sin, rot, inter).to(dt) for x in st["douts"]]
        return res
    if kind == "store":
        return [_value(*_unpack(*_pack(*_quantise(st[x])))).to(dt) for x in ("k1", "k2", "v")]
    lens, offset, lam = st["lens"].long(), _offset(st), st["lam"].float()
    q1, q2 = st["q1"].float(), st["q2"].float()
    if kind == "kv4":
        who, at = torch.arange(case["b"], device=lens.device), st["start"].long()
        for name, held in zip(("k1", "k2", "v"), st["packed"]):
            for store, new in zip(held, _pack(*_quantise(st[name]))):
                store[who, :, at] = new[:, :, 0]
        k1, k2, v = (_value(*_unpack(*x)) for x in st["packed"])
        return [_attend(q1, q2, k1, k2, v, lam, lens, offset).to(dt), st["start"] + 1]
    k1, k2, v = (st[x].float() for x in ("k1", "k2", "v"))
    if kind != "train":
        return _attend(q1, q2, k1, k2, v, lam, lens, offset).to(dt)
    xs = [x.detach().requires_grad_(True) for x in (q1, q2, k1, k2, v, lam)]
    out = _attend(*xs, lens, offset)
    return [out.detach().to(dt)] + [x.to(dt) for x in torch.autograd.grad(out, xs, st["dout"].float())]


# ------------------------------------------------------------------ the framework's calls
def _calls(st):
    import tda_amd
    case = st["case"]
    kind, dt = case["kind"], _DTYPE[case["dtype"]]
    if kind == "rotary":
        where = (st["positions"], st["inv_freq"], st["sections"])
        if not case["grad"]:
            return list(tda_amd.rotary_axes(st["xs"], *where, interleaved=case["interleaved"]))
        xs = [x.detach().requires_grad_(True) for x in st["xs"]]
        res = tda_amd.rotary_axes(xs, *where, interleaved=case["interleaved"])
        return [x.detach() for x in res] + list(torch.autograd.grad(res, xs, st["douts"]))
    if kind == "store":
        st["cache"].append(st["k1"], st["k2"], st["v"], start=st["start"])
        return list(st["cache"].read(dtype=dt))
    if kind == "kv4":
        st["cache"].append(st["k1"], st["k2"], st["v"], start=st["start"])
        return [st["cache"].attend(st["q1"], st["q2"], st["lam"]), st["cache"].lengths]
    lens = st["lens"] if case["ragged"] else None
    if kind == "decode":  # the newest token sees every key of its sequence
        return tda_amd.differential_attention(st["q1"], st["q2"], st["k1"], st["k2"], st["v"], st["lam"], causal=False,
                                              kv_lens=lens)
    xs = [st[x] for x in ("q1", "q2", "k1", "k2", "v", "lam")]
    if kind == "prefill":
        return tda_amd.differential_attention(*xs, kv_lens=lens)
    xs = [x.detach().requires_grad_(True) for x in xs]
    out = tda_amd.differential_attention(*xs, kv_lens=lens)
    return [out.detach()] + list(torch.autograd.grad(out, xs, st["dout"]))


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    b, h, hk, d = case["b"], case["h"], case["hk"], case["d"]
    if case["kind"] == "rotary":
        values = b * case["n"] * 2 * (h + hk) * d
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * 2 * values * size + 8 * case["axes"] * b * case["n"], "flops": passes * 3 * values}
    nq, nk, dv = case["nq"], case["nk"], case["dv"]
    keys = sum(_lengths(case))
    if case["kind"] == "store":
        values = keys * hk * (2 * d + dv)
        return {"bytes": 2 * values * size + 2 * values * 9 // 16, "flops": 6 * values}
    if case["kind"] in ("decode", "kv4"):
        seen = keys * nq
    else:  # row i of nq sees nk - nq + i + 1 keys, and no more than there are
        seen = sum(min(n, nk - nq + i + 1) for n in _lengths(case) for i in range(nq))
    cache = keys * hk * (2 * d + dv)
    rows = b * h * nq * (2 * d + dv)
    if case["kind"] == "kv4":
        return {"bytes": cache * 9 // 16 + (rows + b * hk * (2 * d + dv)) * size, "flops": h * seen * (4 * d + 2 * dv)}
    if case["kind"] == "train":  # inputs, the output's gradient and the output; the gradients
        return {"bytes": (2 * cache + 2 * rows + b * h * nq * dv) * size, "flops": h * seen * (16 * d + 6 * dv)}
    return {"bytes": (cache + rows) * size, "flops": h * seen * (4 * d + 2 * dv)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_head(q1, q2, k1, k2, v, lam, hidden, dout):
    """One query head in 64 bits: its output, and with dout the gradients, by the formulas."""
    scale = q1.shape[1] ** -0.5

    def weights(q, k):
        s = (q @ k.T).mul_(scale)
        s[hidden] = -math.inf
        s -= s.amax(1, keepdim=True).clamp_min(-1e300)
        s.exp_()
        total = s.sum(1, keepdim=True)
        return s.div_(torch.where(total > 0, total, 1.0))

    p1, p2 = weights(q1, k1), weights(q2, k2)
    o1, o2 = p1 @ v, p2 @ v
    if dout is None:
        return o1 - lam * o2
    dp = dout @ v.T
    row1, row2 = (dout * o1).sum(1, keepdim=True), (dout * o2).sum(1, keepdim=True)
    ds1 = p1 * (dp - row1) * scale
    ds2 = p2 * (dp - row2) * (-lam * scale)
    return o1 - lam * o2, ds1 @ k1, ds2 @ k2, ds1.T @ q1, ds2.T @ q2, (p1 - lam * p2).T @ dout, -row2.sum()


def _exact_attention(st, k1, k2, v):
    case = st["case"]
    b, h, hk, nq = case["b"], case["h"], case["hk"], case["nq"]
    nk, group = k1.shape[2], h // hk
    lens, offset = st["lens"].tolist(), _offset(st).tolist()
    train = case["kind"] == "train"
    out = torch.empty(b, h, nq, v.shape[3], dtype=torch.float64, device=v.device)
    if train:
        grads = [torch.zeros(x.shape, dtype=torch.float64, device=v.device) for x in (st["q1"], st["q2"], k1, k2, v, st["lam"])]
    j = torch.arange(nk, device=v.device)
    for n in range(b):
        i = torch.arange(nq, device=v.device) + offset[n]
        hidden = (j[None] > i[:, None]) | (j[None] >= lens[n])
        for x in range(h):
            y = x // group
            head = _exact_head(st["q1"][n, x].double(), st["q2"][n, x].double(), k1[n, y].double(), k2[n, y].double(),
                               v[n, y].double(), st["lam"][x].double(), hidden, st["dout"][n, x].double() if train else None)
            if not train:
                out[n, x] = head
                continue
            out[n, x] = head[0]
            grads[0][n, x], grads[1][n, x] = head[1], head[2]
            for to, part in zip(grads[2:5], head[3:6]):
                to[n, y] += part
            grads[5][x] += head[6]
    return [out, *grads] if train else out


def _exact_held(x):
    """The values that the 4-bit cache holds for x, in 64 bits from the definition on."""
    y = x.double().unflatten(-1, (-1, _GROUP))
    low = y.min(-1, keepdim=True).values.float().bfloat16().double()
    step = ((y.max(-1, keepdim=True).values - low) / 15).float().bfloat16().double()
    step = step * (step >= _SMALL)
    code = torch.round((y - low) / torch.where(step > 0, step, 1.0)).clamp(0, 15) * (step > 0)
    return (low + step * code).flatten(-2)


def exact(case, seed):
    st = _drawn(case, seed)
    kind = case["kind"]
    if kind == "store":
        return [_exact_held(st[x]) for x in ("k1", "k2", "v")]
    if kind == "rotary":
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=st["inv_freq"].device), _angles(st))
        rot, res = case["rot"], []
        for xs, by in ((st["xs"], turn), (st.get("douts") or [], turn.conj())):
            for x in xs:
                y = x.double().clone()
                if case["interleaved"]:
                    y[..., :rot] = torch.view_as_real(torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * by).flatten(-2)
                else:
                    z = torch.complex(y[..., : rot // 2], y[..., rot // 2: rot]) * by
                    y[..., : rot // 2], y[..., rot // 2: rot] = z.real, z.imag
                res.append(y)
        return res
    if kind == "kv4":
        return [_exact_attention(st, *(_exact_held(st[x]) for x in ("k1", "k2", "v"))), None]
    return _exact_attention(st, st["k1"], st["k2"], st["v"])
