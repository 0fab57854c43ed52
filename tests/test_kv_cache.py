"""The 4-bit cache (tda_amd.Int4KVCache): what it holds against the definition, exactly; the attention over
it against float64 on the values held, within the bounds of oracle/softmax.py."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

import tda_amd
from tda_amd.kv_cache import _from_codes
from oracle import softmax as oracle

BF, F32, F16 = torch.bfloat16, torch.float32, torch.float16
U = {BF: 2.0 ** -8, F32: 2.0 ** -24, F16: 2.0 ** -11}
DIMS = [(64, 64), (64, 128), (128, 128), (128, 256)]
gpu = pytest.mark.gpu


def rows(b, h, n, d, seed, dtype, level=0.0):
    g = torch.Generator("cpu").manual_seed(seed)
    x = torch.randn(b, n, h, d, generator=g) + level * torch.randn(1, 1, h, d, generator=g)
    return x.to(dtype).cuda().transpose(1, 2)


def context(b, hk, n, d, dv, dtype, seed=0):
    return rows(b, hk, n, d, seed, dtype, 1.5), rows(b, hk, n, d, seed + 1, dtype, 1.5), rows(b, hk, n, dv, seed + 2, dtype)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0)) and torch.equal(a.isnan(), b.isnan())


def held(x, dtype=F32):
    return oracle.held4(x).float().to(dtype)  # m + s code has at most 24 bits when their exponents are near


# ------------------------------------------------------------------ what it holds
@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
@pytest.mark.parametrize("d, dv", DIMS)
@pytest.mark.parametrize("n", [1, 7, 130])
def test_append_and_read(dtype, d, dv, n):
    c = tda_amd.Int4KVCache(2, 3, 131, d, dv)
    xs = context(2, 3, n, d, dv, dtype)
    c.append(*xs)
    assert c.lengths.tolist() == [n, n]
    for got, x in zip(c.read(n, F32), xs):
        want = oracle.held4(x)
        assert ((got.double() - want).abs() <= 2.0 ** -24 * want.abs()).all()  # one rounding of m + s code
    for got, x, w in zip(c.read(dtype=BF), xs, (d, d, dv)):
        assert got.shape == (2, 3, 131, w) and not got[:, :, n:].any()
        assert torch.equal(got[:, :, :n], held(x, BF))


@gpu
def test_values_next_to_borders():
    """Inputs laid on and one step beside every border between codes, with steps that are no power of two;
    constant groups, groups of zeros, a step below the smallest, subnormals."""
    m, s = torch.tensor(-1.0), torch.tensor(0.171875)
    q = torch.arange(15, dtype=torch.float64)
    border = (m.double() + (q + 0.5) * s.double()).float()
    up, down = (torch.nextafter(border, torch.tensor(w)) for w in (math.inf, -math.inf))
    row = torch.cat((m[None], border, up, down, (m + 15 * s)[None]))
    row = torch.cat((row, row[:1].expand(64 - row.numel())))
    lines = [row, torch.zeros(64), torch.full((64,), 3.7), torch.linspace(1, 1 + 1e-6, 64), 1e-33 * torch.arange(64.0),
             2.0 ** -140 * torch.arange(64.0), torch.cat((torch.full((63,), 1e-20), torch.ones(1))), -row * 1e30]
    x = torch.stack(lines)[None, None].cuda()  # (1, 1, 8, 64)
    c = tda_amd.Int4KVCache(1, 1, 8, 64, 64)
    c.append(x, x, x)
    for got in c.read(dtype=F32):
        want = oracle.held4(x)
        assert ((got.double() - want).abs() <= 2.0 ** -24 * want.abs()).all()


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_group_that_is_not_finite(bad):
    xs = [x.clone() for x in context(1, 2, 5, 128, 128, BF)]
    for x in xs:
        x[0, 1, 3, 70] = bad
    c = tda_amd.Int4KVCache(1, 2, 5, 128)
    c.append(*xs)
    for got, x in zip(c.read(dtype=F32), xs):
        nan = torch.zeros_like(got, dtype=torch.bool)
        nan[0, 1, 3, 64:] = True
        assert torch.equal(got.isnan(), nan) and same(got, held(x))


@gpu
def test_ragged_appends_leave_other_rows_alone():
    c = tda_amd.Int4KVCache(3, 2, 40, 64, 128)
    first = context(3, 2, 20, 64, 128, BF)
    c.append(*first, counts=torch.tensor([20, 3, 0]).cuda())
    assert c.lengths.tolist() == [20, 3, 0]
    second = context(3, 2, 25, 64, 128, BF, seed=9)
    c.append(*second, counts=torch.tensor([25, 7, 40], dtype=torch.int32).cuda())  # 45 > 40: dropped; 40 > 25: clamped
    assert c.lengths.tolist() == [40, 10, 25]
    for got, a, b in zip(c.read(dtype=F32), first, second):
        a, b = held(a), held(b)
        assert torch.equal(got[0], torch.cat((a[0], b[0, :, :20]), 1))
        assert torch.equal(got[1, :, :10], torch.cat((a[1, :, :3], b[1, :, :7]), 1)) and not got[1, :, 10:].any()
        assert torch.equal(got[2, :, :25], b[2])
    # one sequence rewritten from an earlier position; places outside the cache are dropped
    third = context(3, 2, 2, 64, 128, BF, seed=20)
    c.append(*third, start=torch.tensor([5, 39, -1]).cuda())
    assert c.lengths.tolist() == [7, 40, 1]
    c.lengths.fill_(40)
    for got, a, b, t in zip(c.read(dtype=F32), first, second, third):
        a, b, t = held(a), held(b), held(t)
        assert torch.equal(got[0, :, 5:7], t[0]) and torch.equal(got[0, :, 7:20], a[0, :, 7:])
        assert torch.equal(got[1, :, 39], t[1, :, 0])
        assert torch.equal(got[2, :, 0], t[2, :, 1]) and torch.equal(got[2, :, 1:25], b[2, :, 1:])


# ------------------------------------------------------------------ attention over it
def attend(c, q1, q2, lam, scale=None):
    """The oracle on the values that the cache holds."""
    n = q1.shape[2]
    ks = [x.double() for x in c.read(dtype=F32)]
    lens = c.lengths.clamp(0, c.capacity).cpu()
    return oracle.attention(q1, q2, *ks, lam, scale, u=U[BF] if q1.dtype == BF else 2.0 ** -16 if q1.dtype == F16 else U[F32],
                            q_offset=lens - n, kv_lens=lens), ks


def close(got, ref, c, ks, q1, q2, dtype):
    """The oracle's bound counts the sums' magnitudes with the held values; the kernel sums m and s code
    (bf16: s (128 + code), its 128 taken off) apart: up to 64 times the group's largest value for bf16 and
    5 times otherwise, in 24 bits.  That enters as a share of the largest magnitudes."""
    times = 64 if dtype == BF else 6
    f, d = 2.0 ** -24, c.head_dim
    big = max(x.abs().max().item() for x in ks[2:])
    score = max(q.double().abs().sum(-1).max().item() * k.abs().max().item() for q, k in ((q1, ks[0]), (q2, ks[1]))) / math.sqrt(d)
    extra = 4 * times * f * (score * big + (c.capacity ** 0.5 + 16) * big)
    off = ref["out_off"] + U[dtype] * ref["out"].abs() + extra
    if dtype == BF:  # weight times step is rounded, around a group's middle: up to 8 steps of 1/15 of its range
        off = off + U[BF] * ref["around"]
    assert ((got.double() - ref["out"]).abs() <= off).all()


def around(c, q1, q2, lam):
    """sum over keys of (P1 + |lambda| P2) times 8 steps of the value's group, per output."""
    v = c.read(dtype=F32)[2].double().nan_to_num()
    y = v.unflatten(-1, (-1, 64))
    reach = ((y.amax(-1, keepdim=True) - y.amin(-1, keepdim=True)).expand_as(y)).flatten(-2)
    lens = c.lengths.clamp(0, c.capacity).cpu()
    k1, k2 = (x.double() for x in c.read(dtype=F32)[:2])
    a = oracle.attention(q1, q2, k1, k2, reach, torch.tensor(0.0), q_offset=lens - q1.shape[2], kv_lens=lens)["out"]
    b = oracle.attention(q2, q1, k2, k1, reach, torch.tensor(0.0), q_offset=lens - q1.shape[2], kv_lens=lens)["out"]
    return a + oracle.lambda_rows(lam, *q1.shape[:3], q1.device).abs() * b


@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
@pytest.mark.parametrize("d, dv", DIMS)
@pytest.mark.parametrize("h, hk, n, cap", [(1, 1, 1, 1), (8, 8, 1, 1000), (8, 2, 1, 33), (40, 2, 1, 300), (4, 4, 4, 129),
                                           (6, 3, 7, 520), (4, 2, 16, 2000), (4, 1, 70, 300), (16, 1, 300, 300)])
def test_attend(dtype, d, dv, h, hk, n, cap):
    c = tda_amd.Int4KVCache(3, hk, cap, d, dv)
    c.append(*context(3, hk, cap, d, dv, dtype))
    c.lengths.copy_(torch.tensor([cap, (cap + 1) // 2, 0]))
    q1, q2 = rows(3, h, n, d, 50, dtype), rows(3, h, n, d, 51, dtype)
    lam = torch.linspace(-0.5, 0.9, h).cuda()
    got = c.attend(q1, q2, lam)
    assert got.dtype == dtype and not got[2].any()
    if not _from_codes(3, hk, h // hk * n, dtype):  # by way of read(): the values rounded to the queries' type
        ks = c.read(dtype=dtype)
        want = tda_amd.differential_attention(q1, q2, *ks, lam, q_offset=c.lengths - n, kv_lens=c.lengths)
        assert torch.equal(got, want)
        return
    ref, ks = attend(c, q1, q2, lam)
    ref["around"] = around(c, q1, q2, lam)
    close(got, ref, c, ks, q1, q2, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_decoding_steps(dtype):
    """A run of steps as a serving program makes them: a prompt, then token by token."""
    b, h, hk, d = 2, 8, 2, 64
    c = tda_amd.Int4KVCache(b, hk, 64, d)
    prompt = context(b, hk, 30, d, d, dtype)
    c.append(*prompt, counts=torch.tensor([30, 11]).cuda())
    for t in range(20):
        c.append(*context(b, hk, 1, d, d, dtype, seed=100 + 3 * t))
        q1, q2 = rows(b, h, 1, d, 300 + t, dtype), rows(b, h, 1, d, 400 + t, dtype)
        got = c.attend(q1, q2, 0.4)
        ref, ks = attend(c, q1, q2, 0.4)
        ref["around"] = around(c, q1, q2, 0.4)
        close(got, ref, c, ks, q1, q2, dtype)
    assert c.lengths.tolist() == [50, 31]


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_nothing_behind_the_length_is_read(dtype):
    c = tda_amd.Int4KVCache(2, 2, 200, 64, 128)
    bad = [x.clone() for x in context(2, 2, 200, 64, 128, dtype)]
    for x in bad:
        x[0, :, 77:] = math.nan
        x[1, :, 130:] = math.inf
    c.append(*bad)
    lens = torch.tensor([77, 130], dtype=torch.int32)
    c.lengths.copy_(lens)
    q1, q2 = rows(2, 4, 2, 64, 50, dtype), rows(2, 4, 2, 64, 51, dtype)
    got = c.attend(q1, q2, 0.5)
    ref, ks = attend(c, q1, q2, 0.5)
    ref["around"] = around(c, q1, q2, 0.5)
    close(got, ref, c, ks, q1, q2, dtype)
    # lengths out of range are clamped
    c.lengths.copy_(torch.tensor([-3, 1000]))
    got = c.attend(q1, q2, 0.5)
    assert not got[0].any() and got[1].isnan().any()


@gpu
def test_captured_steps():
    """Two graphs of append and attend on caches of their own, replayed between eager steps on a third."""
    b, h, hk, d = 2, 8, 2, 128
    new = [x.contiguous() for x in context(b, hk, 1, d, d, BF, seed=7)]
    q1, q2 = rows(b, h, 1, d, 50, BF).contiguous(), rows(b, h, 1, d, 51, BF).contiguous()
    caches = [tda_amd.Int4KVCache(b, hk, 3000, d) for _ in range(3)]
    for c in caches:
        c.append(*context(b, hk, 2500, d, d, BF), counts=torch.tensor([2500, 1200]).cuda())
        c.append(*new)
        c.attend(q1, q2, 0.3)
        c.lengths.sub_(1)

    def step(c):
        c.append(*new)
        return c.attend(q1, q2, 0.3)

    graphs, outs = [], []
    for c in caches[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    for k in range(3):
        for x in (*new, q1, q2):
            x.mul_(1.1 + 0.1 * k)
        want = step(caches[2])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c, got in zip(caches, outs):
            assert torch.equal(got, want) and torch.equal(c.lengths, caches[2].lengths)
    assert caches[0].lengths.tolist() == [2503, 1203]


@gpu
def test_other_stream_and_replaced_lengths():
    c = tda_amd.Int4KVCache(1, 2, 500, 64)
    c.append(*context(1, 2, 400, 64, 64, BF))
    q1, q2 = rows(1, 4, 1, 64, 50, BF), rows(1, 4, 1, 64, 51, BF)
    want = c.attend(q1, q2, 0.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.attend(q1, q2, 0.5)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    c.lengths = torch.full((1,), 300, dtype=torch.int32, device="cuda")
    short = c.attend(q1, q2, 0.5)
    d = tda_amd.Int4KVCache(1, 2, 300, 64)
    d.append(*(x[:, :, :300] for x in context(1, 2, 400, 64, 64, BF)))
    assert (short - d.attend(q1, q2, 0.5)).abs().max() <= 2.0 ** -6 * short.abs().max()  # another split of the keys
    for wrong in (torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int32), None):
        c.lengths = wrong
        with pytest.raises(ValueError):
            c.attend(q1, q2, 0.5)


# ------------------------------------------------------------------ refusals
def test_refusals_without_a_gpu():
    for args in ((0, 1, 4, 64), (1, 0, 4, 64), (1, 1, 0, 64), (1, 1, 4, 32), (1, 1, 4, 128, 64), (1, 1, 4, 64, 96)):
        with pytest.raises(ValueError):
            tda_amd.Int4KVCache(*args)
    with pytest.raises(ValueError, match="GPU only"):
        tda_amd.Int4KVCache(1, 1, 4, 64, device="cpu")


@gpu
def test_refusals():
    c = tda_amd.Int4KVCache(2, 2, 10, 64, 128)
    k, v = torch.zeros(2, 2, 3, 64, device="cuda"), torch.zeros(2, 2, 3, 128, device="cuda")
    many = torch.zeros(2, 2, 11, 64, device="cuda"), torch.zeros(2, 2, 11, 64, device="cuda"), torch.zeros(2, 2, 11, 128, device="cuda")
    for args in ((k, k, k), (k, k[:, :1], v), (k, k[:, :, :2], v), (k[:1], k[:1], v[:1]), (k.double(),) * 2 + (v.double(),),
                 (k.half(), k, v), (k.cpu(), k.cpu(), v.cpu()), many):
        with pytest.raises(ValueError):
            c.append(*args)
    for kw in (dict(counts=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(start=torch.zeros(2, device="cuda")),
               dict(counts=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            c.append(k, k, v, **kw)
    with pytest.raises(TypeError):
        c.append(None, k, v)
    for n in (0, 11, -1):
        with pytest.raises(ValueError):
            c.read(n)
    with pytest.raises(ValueError):
        c.read(dtype=torch.float64)
    q = torch.zeros(2, 4, 1, 64, device="cuda")
    for args in ((q, q[:, :2], 0.5), (q[:, :3], q[:, :3], 0.5), (q[:1], q[:1], 0.5), (q, q, torch.zeros(3)), (q.double(), q.double(), 0.5)):
        with pytest.raises(ValueError):
            c.attend(*args)
    with pytest.raises(ValueError):
        c.attend(q, q, 0.5, scale=-1.0)
    assert c.lengths.tolist() == [0, 0]
    c.append(k[:, :, :0], k[:, :, :0], v[:, :, :0])
    assert c.attend(q[:, :, :0], q[:, :, :0], 0.5).shape == (2, 4, 0, 128)


@gpu
def test_lengths_below_zero_count_from_the_start():
    c = tda_amd.Int4KVCache(2, 1, 8, 64, 64)
    c.lengths.copy_(torch.tensor([-3, 0]))
    xs = context(2, 1, 4, 64, 64, BF)
    c.append(*xs)
    assert c.lengths.tolist() == [4, 4]
    assert all(torch.equal(got[:, :, :4], held(x)) for got, x in zip(c.read(dtype=F32), xs))


@gpu
@pytest.mark.parametrize("n", [1, 40])
def test_lengths_beyond_the_capacity(n):
    c = tda_amd.Int4KVCache(1, 1, 50, 64, 64)
    c.append(*context(1, 1, 50, 64, 64, BF))
    q = rows(1, 1, n, 64, 3, BF)
    want = c.attend(q, q * 0.5, 0.5)
    c.lengths.fill_(1 << 30)
    assert torch.equal(c.attend(q, q * 0.5, 0.5), want)


@gpu
def test_capacity_and_starts_out_of_range():
    with pytest.raises(ValueError, match="capacity"):
        tda_amd.Int4KVCache(1, 1, (1 << 24) + 1, 64)
    c = tda_amd.Int4KVCache(2, 1, 8, 64, 64)
    xs = context(2, 1, 5, 64, 64, BF)
    c.append(*xs)
    want = c.read()
    c.append(*xs, start=torch.tensor([2 ** 31 - 1, -2 ** 31]).cuda())  # nothing to write, beyond either end
    assert c.lengths.tolist() == [8, 0]
    c.lengths.fill_(5)
    assert all(torch.equal(a, b) for a, b in zip(c.read(), want))


@gpu
def test_calls_of_one_signature_take_their_own_tensors():
    c, d = (tda_amd.Int4KVCache(2, 1, 64, 64, 64) for _ in range(2))
    for k in range(3):
        xs = context(2, 1, 3, 64, 64, BF, seed=10 * k)
        starts = torch.tensor([3 * k, 2 * k], dtype=torch.int32).cuda()  # no row is left unwritten
        c.append(*xs, start=starts)
        d.append(*xs, start=starts.long())  # another signature
        assert all(torch.equal(a, b) for a, b in zip(c.read(), d.read())) and torch.equal(c.lengths, d.lengths)
        q1, q2 = rows(2, 2, 1, 64, 40 + k, BF), rows(2, 2, 1, 64, 50 + k, BF)
        lam = torch.tensor([0.3, 0.1 * k]).cuda()
        assert torch.equal(c.attend(q1, q2, lam), d.attend(q1, q2, lam.double()))
    off = torch.empty(q1.numel() + 1, dtype=BF, device="cuda")[1:].view_as(q1).copy_(q1)
    assert torch.equal(c.attend(off, q2, lam), c.attend(q1, q2, lam))
    c.lengths = d.lengths.clone()
    c.lengths.fill_(4)
    d.lengths.fill_(4)
    assert torch.equal(c.attend(q1, q2, lam), d.attend(q1, q2, lam))
    for wrong in (c.lengths.long(), None, [4, 4]):
        c.lengths = wrong
        with pytest.raises(ValueError, match="lengths"):
            c.attend(q1, q2, lam)
    with pytest.raises(ValueError):
        d.attend(q1, q2, lam[:1].expand(3))
    with pytest.raises(ValueError):
        d.append(xs[0], xs[1].cpu(), xs[2])


@gpu
@pytest.mark.parametrize("fork", [copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))])
@pytest.mark.parametrize("n", [1, 40])
def test_a_copy_has_its_own_rows(fork, n):
    """A cache forked after calls of every kind: both go on by themselves, also with calls of signatures that the
    original has seen."""
    def step(c, seed):
        c.append(*context(2, 2, n, 64, 128, BF, seed))
        q = rows(2, 4, n, 64, seed + 5, BF)
        return [c.attend(q, q * 0.5, lam), *c.read(), c.lengths.clone()]

    lam = torch.tensor([0.1, 0.2, 0.3, 0.4]).cuda()
    first = tda_amd.Int4KVCache(2, 2, 200, 64, 128)
    step(first, 0)
    second = fork(first)
    got = [step(second, 10), step(first, 20), step(second, 30), step(first, 40)]
    for k, seeds in enumerate(((0, 10, 30), (0, 20, 40))):
        alone = tda_amd.Int4KVCache(2, 2, 200, 64, 128)
        want = [step(alone, s) for s in seeds][1:]
        assert all(torch.equal(a, b) for x, y in zip(got[k::2], want) for a, b in zip(x, y))


def test_a_copy_keeps_no_addresses():
    c = tda_amd.Int4KVCache.__new__(tda_amd.Int4KVCache)
    c._held, c._templates, c._plans = [torch.zeros(8)], {"a": b"1"}, {"b": b"2"}
    state = c.__getstate__()
    assert state["_templates"] == state["_plans"] == {} and c._templates and c._plans
    with pytest.raises(ValueError, match="GPU only"):
        copy.deepcopy(c)  # rows on the CPU, as a cache loaded there would have


@gpu
@pytest.mark.parametrize("n", [1, 300])
@pytest.mark.parametrize("given", [None, [0, 0, 0], [700, 5, 1], [900, 0, -4]])
def test_append_counts_that_are_the_lengths(n, given):
    """As with a copy of them, whichever workgroup comes last."""
    caches = [tda_amd.Int4KVCache(3, 16, 1000, 128, 256) for _ in range(2)]
    start = None if given is None else torch.tensor(given, dtype=torch.int32).cuda()
    xs = context(3, 16, n, 128, 256, BF, 1)
    for c in caches:
        c.append(*context(3, 16, 1000, 128, 256, BF, 4))
    for k in range(4):
        for c in caches:
            c.lengths.copy_(torch.tensor([n // 2, n, n // 3 + k]))
        caches[0].append(*xs, counts=caches[0].lengths, start=start)
        caches[1].append(*xs, counts=caches[1].lengths.clone(), start=start)
        assert torch.equal(caches[0].lengths, caches[1].lengths)
        if start is not None:
            assert caches[0].lengths.tolist() == [min(max(s + m, 0), 1000) for s, m in zip(given, (n // 2, n, min(n // 3 + k, n)))]
        for c in caches:
            c.lengths.fill_(1000)
        assert all(torch.equal(a, b) for a, b in zip(caches[0].read(), caches[1].read()))


@gpu
def test_append_lengths_as_part_of_another_tensor():
    c = tda_amd.Int4KVCache(2, 1, 8, 64)
    shared = torch.zeros(3, dtype=torch.int32).cuda()
    c.lengths = shared[:2]
    xs = context(2, 1, 1, 64, 64, BF)
    c.append(*xs, start=shared[:2])
    assert shared.tolist() == [1, 1, 0]
    for kw in (dict(start=shared[1:]), dict(counts=shared[1:])):
        with pytest.raises(ValueError, match="overlapping"):
            c.append(*xs, **kw)
    assert shared.tolist() == [1, 1, 0]


def test_the_step_is_a_quotient():
    """The oracle's step against numpy's division, which rounds once: of float16 groups about one in 700 has another
    with a product by the rounded 1 / 15."""
    x = torch.randn(200000, 64, generator=torch.Generator().manual_seed(3)).half()
    y = x.float()
    m = y.amin(-1, keepdim=True).bfloat16()
    quotient = (y.amax(-1, keepdim=True) - m.float()).numpy() / np.float32(15)
    s = torch.from_numpy(quotient).bfloat16().double()
    code = ((y.double() - m.double()) / s).round().clamp(0, 15)
    assert quotient.dtype == np.float32 and torch.equal(oracle.held4(x), m.double() + s * code)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
def test_many_groups(dtype):
    c = tda_amd.Int4KVCache(4, 8, 8192, 64, 128)
    xs = context(4, 8, 8192, 64, 128, dtype, 60)
    c.append(*xs)
    for got, x in zip(c.read(dtype=F32), xs):
        want = oracle.held4(x)
        assert ((got.double() - want).abs() <= 2.0 ** -24 * want.abs()).all()


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("part", ["keys", "values"])
@pytest.mark.parametrize("n", [1, 160])
def test_float16_queries_over_rows_beyond_float16(dtype, part, n):
    """Held values past 65504, whose scores and outputs float16 does hold, attended by a token and by many rows."""
    c = tda_amd.Int4KVCache(4, 8, 160, 64)
    k1, k2, v = context(4, 8, 160, 64, 64, dtype)
    q1, q2 = rows(4, 8, n, 64, 50, F16), rows(4, 8, n, 64, 51, F16)
    if part == "values":  # the two maps' averages of values around 90000
        v = 90000 + 1000 * v
    else:
        k1, k2, q1, q2 = k1 * 7e4, k2 * 7e4, q1 * 2.0 ** -10, q2 * 2.0 ** -10
    c.append(k1.to(dtype), k2.to(dtype), v.to(dtype))
    assert n == 1 or not _from_codes(4, 8, n, F16)
    got = c.attend(q1, q2, 1.0)
    ref, ks = attend(c, q1, q2, 1.0)
    assert max(x.abs().max().item() for x in ks) > 65520  # float16's infinity
    close(got, ref, c, ks, q1, q2, F16)


@gpu
def test_float16_rows_next_to_the_end_of_float16():
    """A group from -65504 to 65504 is held with a step that reaches beyond; read() and many rows stop at the end."""
    c = tda_amd.Int4KVCache(4, 8, 160, 64)
    x = torch.where(rows(4, 8, 160, 64, 1, F16) > 0, 65504.0, -65504.0).half()
    c.append(x * 2.0 ** -14, x * 2.0 ** -14, x)
    held = c.read(dtype=F32)[2]
    assert held.abs().max().item() > 65520
    ks = c.read(dtype=F16)
    assert torch.equal(ks[2], held.clamp(-65504, 65504).half())
    q = rows(4, 8, 160, 64, 2, F16)
    got = c.attend(q, q * 0.5, 0.5)
    want = tda_amd.differential_attention(q, q * 0.5, *ks, 0.5, q_offset=c.lengths - 160, kv_lens=c.lengths)
    assert torch.equal(got, want) and got.isfinite().all()
    x = x.float()
    x[1, 3, 5, 7] = math.nan  # a group that is not finite stays so
    c.append(x, x, x, start=torch.zeros(4, dtype=torch.int32).cuda())
    assert torch.equal(c.read(dtype=F16)[2].isnan(), c.read(dtype=F32)[2].isnan()) and c.read(dtype=F16)[2].isnan().sum() == 64
