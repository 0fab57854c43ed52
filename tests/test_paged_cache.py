"""The paged cache (tda_amd.PagedKVCache): what append() puts where against the definition in float64, and the attention
over the pages against float64 within the bounds of oracle/softmax.py."""
import copy
import math
import pickle

import pytest
import torch

import tda_amd
from oracle import paged as oracle
from oracle import softmax

BF, F32, F16 = torch.bfloat16, torch.float32, torch.float16
U = {BF: 2.0 ** -8, F32: 2.0 ** -24, F16: 2.0 ** -11}
TINY = {BF: 1e-30, F32: 1e-30, F16: 2.0 ** -25}
DIMS = [(64, 64), (64, 128), (128, 128), (128, 256)]
gpu = pytest.mark.gpu


def rows(b, h, n, d, seed, dtype, spread=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    return (torch.randn(b, n, h, d, generator=g) * spread).to(dtype).cuda().transpose(1, 2)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Setup:
    """A cache whose pages hold noise (NaN where nobody may look), a table of shuffled pages, and rows of a call in one of
    the three forms: new[s] rows behind held[s] positions."""

    def __init__(self, new, held, h, hk, d, dv, page, dtype, form="packed", seed=0, spare=2, behind=0):
        g = torch.Generator("cpu").manual_seed(seed)
        s = len(new)
        need = [-(-max(a + b, 0) // page) for a, b in zip(new, held)]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((s, max(max(need), 1) + 1), -1, dtype=torch.int32)
        at = 0
        for i, m in enumerate(need):
            self.table[i, :m] = order[at:at + m]
            at += m
        self.table = self.table.cuda()
        self.new, self.held_, self.page, self.dtype = new, held, page, dtype
        self.lengths = ints(*held)
        self.cache = c = tda_amd.PagedKVCache(pages, hk, page, d, dv, dtype=dtype)
        for i, t in enumerate((c.k1, c.k2, c.v)):
            t.copy_(torch.randn(t.shape, generator=g).to(dtype))
        self.where = {}
        lead, n = (1, sum(new) + behind) if form == "packed" else (s, max(max(new), 1) + (behind if form == "counts" else 0))
        if form == "packed":
            self.where["starts"] = ints(*[sum(new[:i]) for i in range(s + 1)])
        elif form == "counts":
            self.where["counts"] = ints(*new)
        else:
            assert len(set(new)) == 1
        self.lead, self.n = lead, n
        self.q1, self.q2 = rows(lead, h, n, d, seed + 1, dtype, 1.5), rows(lead, h, n, d, seed + 2, dtype, 1.5)
        self.k1, self.k2, self.v = rows(lead, hk, n, d, seed + 3, dtype), rows(lead, hk, n, d, seed + 4, dtype), rows(lead, hk, n, dv, seed + 5, dtype)

    def pools(self):
        return self.cache.k1, self.cache.k2, self.cache.v

    def spoil(self):
        """NaN in every place that no sequence's positions reach."""
        used = torch.zeros(self.cache.pages, self.page, dtype=torch.bool)
        for s, (a, b) in enumerate(zip(self.new, self.held_)):
            for p in range(max(a + b, 0)):
                at = oracle.place(self.table, self.page, self.cache.pages, s, p)
                if at:
                    used[at] = True
        free = ~used.cuda()
        for t in self.pools():
            t.transpose(1, 2)[free] = math.nan
        return self

    def attend(self, lam=0.4, **kw):
        got = self.cache.attend(self.q1, self.q2, lam, self.table, self.lengths, **{**self.where, **kw})
        kw.pop("most", None)
        host = {k: v.cpu() for k, v in {**self.where, **kw}.items() if isinstance(v, torch.Tensor)}
        ref = oracle.attend(self.q1, self.q2, self.pools(), lam, self.table, self.lengths.cpu(), kw.get("scale"), **host, u=U[self.dtype])
        tiny = TINY[self.dtype]
        if self.dtype == F16:  # weights below 2^-14 of a row's largest are off by up to 2^-25 each
            most = float(torch.as_tensor(lam).abs().max())
            tiny += ref["out"].shape[2] * 0 + (max(self.held_) + max(self.new)) * 2.0 ** -25 * (1 + most) * self.cache.v.nan_to_num().abs().max().item()
        far = (got.double() - ref["out"]).abs() - ref["out_off"] - U[self.dtype] * ref["out"].abs() - tiny
        assert got.shape == ref["out"].shape and got.dtype == self.dtype and torch.isfinite(got).all()
        assert far.max().item() <= 0, f"{far.max().item():.3g} past {ref['out_off'].flatten()[far.argmax()].item():.3g}"
        return got


# ------------------------------------------------------------------ attention
@gpu
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d, dv", DIMS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_newest_tokens(dtype, d, dv, page):
    for held, h, hk in (([0], 1, 1), ([5, 16, 15, 0, 300], 8, 2), ([1, 700], 10, 2), ([2000], 4, 4)):
        Setup([1] * len(held), held, h, hk, d, dv, page, dtype, "even").spoil().attend()


@gpu
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d, dv", DIMS)
@pytest.mark.parametrize("page", [16, 32, 128])
def test_chunks(dtype, d, dv, page):
    for new, held, h, hk in (([40, 40], [0, 37], 4, 2), ([130], [517], 5, 1), ([129], [0], 2, 2), ([33], [1100], 8, 1)):
        Setup(new, held, h, hk, d, dv, page, dtype, "even").spoil().attend()


@gpu
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("form", ["packed", "counts"])
def test_mixed_batches(dtype, form):
    """A chunk with newest tokens, sequences without rows, rows of no sequence, both forms' borders."""
    for d, dv in DIMS:
        for new, held, h, hk in (([70, 1, 0, 1, 9], [40, 900, 77, 0, 3], 4, 2), ([0, 0, 3], [5, 0, 50], 8, 2),
                                 ([16, 17, 15], [100, 0, 31], 1, 1), ([4, 5, 3, 1], [64, 63, 65, 2000], 8, 2)):
            s = Setup(new, held, h, hk, d, dv, 32, dtype, form, behind=5).spoil()
            got = s.attend(torch.linspace(0.1, 0.9, h).cuda())
            if form == "packed":
                assert not got[:, :, sum(new):].any()
            else:
                assert all(not got[i, :, n:].any() for i, n in enumerate(new))


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_sequences(dtype):
    """More sequences than a wave has lanes, few with rows, and more than that many rows each way."""
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 4, (150,), generator=g).tolist()
    new[70] = 41
    held = torch.randint(0, 90, (150,), generator=g).tolist()
    held[3] = 1500
    Setup(new, held, 4, 2, 64, 64, 16, dtype, "packed").spoil().attend()
    Setup([1] * 150, held, 4, 2, 64, 64, 16, dtype, "even").spoil().attend()
    Setup([7] * 150, held, 4, 1, 64, 64, 16, dtype, "even").spoil().attend()


@gpu
def test_long_sequences_are_cut_and_joined():
    for new, held, form in (([1], [9000], "even"), ([1, 1], [9000, 10], "even"), ([40], [7000], "even"), ([1, 60], [300, 6000], "packed"),
                            ([20, 60], [3000, 20], "packed"), ([3], [5000], "even"), ([4, 2, 0], [4000, 100, 9], "counts")):
        for dtype, (d, dv) in ((BF, (128, 128)), (F32, (64, 128)), (F16, (128, 256))):
            Setup(new, held, 4, 2, d, dv, 64, dtype, form).spoil().attend()


@gpu
@pytest.mark.parametrize("dtype, d, dv", [(BF, 64, 128), (F16, 128, 128), (F32, 128, 256)])
def test_tiles_with_every_row_are_cut(dtype, d, dv):
    """Tiles of 16 and of 128 rows without a spare one, whose parts end before any row's sight does."""
    for new, held, h, hk in (([8], [5000], 4, 2), ([1, 1], [4321, 77], 32, 2), ([4, 8], [2500, 900], 8, 2), ([32], [6011], 8, 2), ([16, 4], [3500, 4097], 8, 1)):
        Setup(new, held, h, hk, d, dv, 64, dtype, "packed").spoil().attend()


@gpu
@pytest.mark.parametrize("dtype, d, dv", [(BF, 128, 128), (F16, 64, 128), (F32, 64, 64)])
def test_a_few_tiles_more_than_fit_at_once(dtype, d, dv):
    """Stretches of more than one large tile, alone and among tokens; and prompts from the start, whose tiles stay whole."""
    for new, held, form in (([600], [1500], "even"), ([600], [1303], "packed"), ([600, 0], [1500, 7], "counts"), ([600, 1, 3], [1500, 300, 0], "packed"), ([600], [0], "even")):
        Setup(new, held, 64, 64, d, dv, 64, dtype, form).spoil().attend()


@gpu
@pytest.mark.parametrize("dtype, d, dv", [(BF, 128, 128), (F16, 64, 128)])
def test_tiles_that_stay_whole(dtype, d, dv):
    """A padded batch too large for its tiles to be cut, most of it padding; one long sequence among as many short ones as
    are taken whole."""
    s = Setup([700] + [1] * 23, [3000 - 60 * i for i in range(24)], 8, 2, d, dv, 32, dtype, "counts").spoil()
    got = s.attend()
    assert not got[1:, :, 1:].any()
    Setup([1] * 64, [20 + i for i in range(63)] + [20000], 16, 8, d, dv, 64, dtype, "even").spoil().attend()
    Setup([1] * 64, [20000] + [20 + i for i in range(63)], 16, 8, d, dv, 64, dtype, "packed").spoil().attend()


@gpu
def test_the_rows_bound_costs_no_results():
    s = Setup([1, 50, 1], [40, 300, 1000], 8, 2, 64, 64, 16, BF, "packed").spoil()
    want = s.attend()
    for most in (1, 2, 50, 1000):
        got = s.attend(most=most)
        assert (got.float() - want.float()).abs().max() < 0.1
    s = Setup([1, 50, 1], [40, 300, 1000], 8, 2, 64, 64, 16, BF, "counts").spoil()
    s.attend(most=1)


@gpu
def test_lambda_scale_and_layouts():
    h = 6
    for lam in (0.0, -1.5, torch.tensor(0.3).cuda(), torch.linspace(-1, 1, h).cuda().half(), torch.rand(1, h, 1).cuda(),
                torch.rand(1, h, 75).cuda().bfloat16(), torch.rand(1, 1, 75).cuda()):
        Setup([70, 1, 4], [33, 200, 0], h, 2, 64, 128, 16, BF, "packed").spoil().attend(lam)
    for lam in (torch.rand(3, h, 1).cuda(), torch.rand(3, 1, 70).cuda()):
        Setup([70, 1, 4], [33, 200, 0], h, 2, 64, 128, 16, BF, "counts").spoil().attend(lam)
    s = Setup([70, 1, 4], [33, 200, 0], h, 2, 64, 128, 16, F32, "packed").spoil()
    s.attend(scale=0.5)
    want = s.attend()
    s.q1, s.q2 = s.q1.contiguous(), s.q2.contiguous()
    assert torch.equal(s.attend(), want)
    odd = torch.zeros(1, h, 75, 65, device="cuda")
    odd[..., 1:] = s.q1
    s.q1 = odd[..., 1:]
    assert torch.equal(s.attend(), want)
    s.q1 = s.q1[:, :1].expand(1, h, 75, 64)  # every head the same rows
    s.attend()
    wide = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, : s.table.shape[1]] = s.table
    s.table = wide[:, : s.table.shape[1]]
    s.attend()
    s.table = s.table.t().contiguous().t()
    s.attend()


@gpu
@pytest.mark.parametrize("dtype, d, dv", [(BF, 64, 64), (F16, 128, 128), (F32, 128, 256)])
def test_room_for_more_than_is_held(dtype, d, dv):
    """Tables of 2048 positions, of which a few are held: small tiles are cut, and joined, or have one unit of keys."""
    for new, held, form in (([1] * 5, [5, 16, 15, 0, 300], "even"), ([3, 0, 2], [129, 700, 126], "counts"), ([2, 1, 3], [900, 0, 128], "packed")):
        s = Setup(new, held, 8, 2, d, dv, 16, dtype, form).spoil()
        wide = torch.full((s.table.shape[0], 128), -1, dtype=torch.int32, device="cuda")
        wide[:, : s.table.shape[1]] = s.table
        s.table = wide
        s.attend()
        s.attend(most=3)


@gpu
def test_shared_pages_and_pages_that_are_none():
    """Two sequences read one prefix; table entries out of range stand for rows of zeros."""
    s = Setup([1, 1, 20], [70, 75, 90], 4, 2, 64, 64, 16, BF, "packed")
    s.table[1, :4] = s.table[0, :4]
    s.attend()
    s.table[0, 2], s.table[2, 0], s.table[2, 4] = -1, s.cache.pages, 2 ** 31 - 1
    s.table[1, 1] = -(2 ** 31)
    s.attend()


@gpu
def test_lengths_out_of_range():
    """Positions below zero see nothing, positions past the table see all that it has."""
    s = Setup([3, 20, 1, 5], [10, 10, 40, 0], 4, 2, 64, 64, 16, BF, "packed")
    for lengths in ((-2, -7, -1, -30), (2 ** 31 - 1, 100, 2 ** 30, -(2 ** 31)), (63, 62, 64, 1)):
        s.lengths = ints(*lengths)
        s.held_ = list(lengths)
        got = s.cache.attend(s.q1, s.q2, 0.4, s.table, s.lengths, **s.where)
        ref = oracle.attend(s.q1, s.q2, s.pools(), 0.4, s.table, s.lengths.cpu().clamp(-2 ** 30, 2 ** 30), u=U[BF], starts=s.where["starts"].cpu())
        assert ((got.double() - ref["out"]).abs() <= ref["out_off"] + U[BF] * ref["out"].abs() + 1e-30).all()
    long = s.cache.attend(s.q1, s.q2, 0.4, s.table, torch.tensor([2 ** 40, 100, 2 ** 35, -2 ** 40]).cuda(), **s.where)
    assert torch.equal(long, s.cache.attend(s.q1, s.q2, 0.4, s.table, ints(2 ** 31 - 1, 100, 2 ** 30, -(2 ** 31)), **s.where))


@gpu
def test_values_that_are_not_finite_stay_with_their_sequence():
    for bad in (math.nan, math.inf, -math.inf):
        s = Setup([30, 1, 1], [50, 70, 20], 4, 2, 64, 64, 16, BF, "packed").spoil()
        clean = s.attend()
        s.cache.v[s.table[1, 2].item(), 1, 3, 5] = bad
        got = s.cache.attend(s.q1, s.q2, 0.4, s.table, s.lengths, **s.where)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[0, 2:, 30, 5] = True
        assert torch.equal(~got.isfinite(), hit) and torch.equal(got[~hit], clean[~hit])


# ------------------------------------------------------------------ append
def turned(x, pos, freq, inter, dtype):
    """x (lead, heads, n, d) in float64 and its bound, positions (axes, lead, n) of sections' pairs given as freq's axis."""
    sections, f = freq
    want = softmax.rotary(x, pos, f, sections, inter)
    pairs = f.shape[0]
    mag = x.double().abs()
    a, b = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if inter else (slice(0, pairs), slice(pairs, 2 * pairs)))
    size = mag.clone()
    size[..., a] = size[..., b] = mag[..., a] + mag[..., b]
    off = U[dtype] * want.abs() + 6 * 2.0 ** -24 * size + TINY[dtype]
    off[..., 2 * pairs:] = 0
    return want, off


def check_append(s, rot=0, sections=None, inter=False, positions=None, far=None):
    c = s.cache
    before = [t.clone() for t in s.pools()]
    kw = {}
    host = {k: v.cpu() for k, v in s.where.items()}
    default = torch.zeros((1, s.lead, s.n), dtype=torch.int64)
    own = torch.zeros((s.lead, s.n), dtype=torch.bool)
    places = []
    for i in range(s.table.shape[0]):
        b, r0, n, at = oracle.rows_of(i, s.lengths.cpu(), s.n, **host)
        default[0, b, r0:r0 + n] = at + torch.arange(n)
        own[b, r0:r0 + n] = True
        places += [(b, r0 + j, oracle.place(s.table.cpu(), s.page, c.pages, i, at + j)) for j in range(n)]
    if rot:
        pairs = rot // 2
        sec = sections or (pairs,)
        freq = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().cuda()
        kw = {"inv_freq": freq, "sections": sections, "positions": positions, "interleaved": inter}
        pos = (default.expand(len(sec), -1, -1) if positions is None else positions.long()).cuda()
        want = [turned(x, pos, (sec, freq), inter, s.dtype) for x in (s.q1, s.q2, s.k1, s.k2)]
    else:
        want = [(x.double(), torch.zeros_like(x, dtype=torch.float64)) for x in (s.q1, s.q2, s.k1, s.k2)]
    want.append((s.v.double(), torch.zeros_like(s.v, dtype=torch.float64)))
    out = c.append(s.k1, s.k2, s.v, s.table, s.lengths, s.q1, s.q2, **s.where, **kw)
    for x, got, (w, off) in zip((s.q1, s.q2), out, want):
        assert got.shape == x.shape and got.dtype == x.dtype and (s.n == 1 or got.stride() == x.stride())
        o = own.cuda()[:, None, :, None]
        assert ((got.double() - w).abs() <= off).logical_or(~o).all() and not got.masked_fill(o, 0).any()
    for pool, old, (w, off) in zip(s.pools(), before, want[2:]):
        for b, i, at in places:
            if at:
                assert ((pool[at[0], :, at[1]].double() - w[b, :, i]).abs() <= off[b, :, i]).all()
                old[at[0], :, at[1]] = pool[at[0], :, at[1]]
        assert torch.equal(pool, old)  # nothing else moved
    return out


@gpu
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d, dv", DIMS)
@pytest.mark.parametrize("inter", [False, True])
def test_append(dtype, d, dv, inter):
    for form, new, held, h, hk in (("even", [1, 1, 1], [0, 15, 700], 8, 2), ("packed", [33, 0, 1, 5], [3, 4, 16, 250], 3, 3),
                                   ("counts", [7, 20, 0], [9, 0, 40], 2, 1)):
        for rot, sections in ((0, None), (d, None), (d // 2, (d // 8, d // 16, d // 16)), (6, (1, 0, 2)), (d - 16, None)):
            check_append(Setup(new, held, h, hk, d, dv, 16, dtype, form, behind=3), rot, sections, inter)


@gpu
def test_append_of_many_rows():
    """Enough tokens for four a workgroup, the last one partly filled."""
    check_append(Setup([4001], [30], 2, 1, 64, 64, 64, BF, "packed", behind=2), 64)
    check_append(Setup([1400, 1399, 1398], [5, 0, 99], 2, 1, 64, 128, 128, F32, "counts"), 64, inter=True)


@gpu
def test_append_positions():
    g = torch.Generator().manual_seed(5)
    for far in (0, 10 ** 8):
        for dt in (torch.int32, torch.int64):
            pos = (far + torch.randint(0, 5000, (3, 1, 40), generator=g)).to(dt).cuda()
            check_append(Setup([30, 10], [3, 40], 2, 1, 64, 64, 32, F32, "packed"), 64, (8, 12, 12), False, pos)
            check_append(Setup([30, 10], [3, 40], 2, 1, 64, 64, 32, F32, "packed"), 64, (8, 12, 12), False, -pos)
    wide = torch.randint(0, 500, (40, 1, 3), generator=g).cuda().permute(2, 1, 0)
    check_append(Setup([30, 10], [3, 40], 2, 1, 64, 64, 32, BF, "packed"), 64, (8, 12, 12), True, wide)
    check_append(Setup([30, 10], [100000, 40], 2, 1, 64, 64, 256, F32, "packed"), 64)


@gpu
def test_append_sections_of_any_kind():
    """A list, a tensor, something that can be gone through once: the first call of a kind and a planned one alike."""
    kinds = [list, iter, lambda x: (n for n in x), torch.tensor, lambda x: map(int, x)]
    want = None
    for make in [tuple, *kinds, *kinds]:
        s = Setup([30, 10], [3, 40], 2, 1, 64, 64, 32, F32, "packed")
        for _ in range(2):
            out = s.cache.append(s.k1, s.k2, s.v, s.table, s.lengths, s.q1, s.q2, **s.where, inv_freq=torch.rand(32, generator=torch.Generator().manual_seed(1)).cuda(),
                                 sections=make((8, 12, 12)), positions=torch.arange(120).view(3, 1, 40).cuda())
            want = want or [*out, *s.pools()]
            assert all(torch.equal(a, b) for a, b in zip([*out, *s.pools()], want))
    with pytest.raises(ValueError, match="add up"):
        s.cache.append(s.k1, s.k2, s.v, s.table, s.lengths, **s.where, inv_freq=torch.rand(32).cuda(), sections=iter((8, 12)))


@gpu
def test_append_drops_what_has_no_place():
    s = Setup([9, 20, 6, 4], [10, 10, 40, 0], 4, 2, 64, 64, 16, BF, "packed")
    s.table[0, 0], s.table[1, 1], s.table[3, 0] = -1, s.cache.pages, 2 ** 31 - 1
    for lengths in ((-3, 30, 2 ** 30 - 5, -(2 ** 30)), (60, 63, 64, 1)):
        s.lengths = ints(*lengths)
        check_append(s, 64)


@gpu
def test_append_without_queries_and_layouts():
    s = Setup([30, 1, 5], [3, 40, 0], 4, 2, 64, 128, 16, BF, "packed")
    freq = torch.rand(32).cuda()
    s.cache.append(s.k1, s.k2, s.v, s.table, s.lengths, s.q1, s.q2, **s.where, inv_freq=freq)
    want = [t.clone() for t in s.pools()]
    for t in s.pools():
        t.zero_()
    again = Setup([30, 1, 5], [3, 40, 0], 4, 2, 64, 128, 16, BF, "packed")
    for t, w in zip(s.pools(), again.pools()):
        t.copy_(w)
    odd = torch.zeros(1, 2, 36, 72, dtype=BF, device="cuda")
    odd[..., 3:67] = s.k1
    assert s.cache.append(odd[..., 3:67], s.k2.contiguous(), s.v, s.table, s.lengths, **s.where, inv_freq=freq) is None
    assert all(torch.equal(a, b) for a, b in zip(s.pools(), want))


# ------------------------------------------------------------------ how they are called
def step(s, x, freq):
    q1, q2 = s.cache.append(x.k1, x.k2, x.v, s.table, s.lengths, x.q1, x.q2, **s.where, inv_freq=freq)
    return s.cache.attend(q1, q2, 0.4, s.table, s.lengths, **s.where)


@gpu
def test_prompts_and_steps_together():
    """Prompts, then steps in which one sequence brings a chunk and the others a token, against all rows at once; the
    lengths are the program's to add to."""
    h, hk, d, dv, page = 4, 2, 64, 128, 16
    total = [90, 41, 70]
    freq = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()
    whole = Setup(total, [0, 0, 0], h, hk, d, dv, page, F32, "packed", seed=3)
    want = step(whole, whole, freq)
    first = [sum(total[:i]) for i in range(3)]
    s = Setup(total, [0, 0, 0], h, hk, d, dv, page, F32, "packed", seed=4)
    done = [0, 0, 0]
    got = torch.empty_like(want)
    for new in ([50, 0, 20], [1, 30, 1], [1, 1, 0], [38, 10, 49]):
        idx = torch.cat([torch.arange(first[i] + done[i], first[i] + done[i] + n) for i, n in enumerate(new)]).cuda()

        class X:
            q1, q2, k1, k2, v = (getattr(whole, n)[:, :, idx] for n in ("q1", "q2", "k1", "k2", "v"))

        s.where = {"starts": ints(*[sum(new[:i]) for i in range(4)])}
        got[:, :, idx] = step(s, X, freq)
        s.lengths = s.lengths + ints(*new)
        done = [a + b for a, b in zip(done, new)]
    assert done == total
    for a, b in zip(s.pools(), whole.pools()):
        for i, n in enumerate(total):
            assert torch.equal(oracle.held(a, s.table, i, n), oracle.held(b, whole.table, i, n))
    # both are within 1e-4 of the formula: sums of at most 90 weighted values of a few units, 24 bits
    assert (got - want).abs().max() < 1e-4


@gpu
def test_graphs_and_streams():
    """A captured step advances by itself when the lengths are added to in it; two graphs with caches of their own."""
    freq = torch.rand(32).cuda()
    made = []
    for seed in (1, 2):
        s = Setup([1, 1, 1], [10, 30, 0], 8, 2, 64, 64, 16, BF, "even", seed=seed)
        s.table = torch.randperm(12).to(torch.int32).cuda().view(3, 4)
        s.cache = tda_amd.PagedKVCache(12, 2, 16, 64)
        for t in s.pools():
            t.normal_()
        made.append(s)
    side = torch.cuda.Stream()
    graphs = []
    for s in made:
        s.in_ = Setup([1, 1, 1], [10, 30, 0], 8, 2, 64, 64, 16, BF, "even", seed=9)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s, s.in_, freq)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.out = step(s, s.in_, freq)
            s.lengths += 1
        graphs.append(g)
    twins = [copy.deepcopy(s.cache) for s in made]
    lengths = [s.lengths.clone() for s in made]
    for i in range(4):
        for s, g, twin, n in zip(made, graphs, twins, lengths):
            new = Setup([1, 1, 1], [10, 30, 0], 8, 2, 64, 64, 16, BF, "even", seed=20 + i)
            for name in ("q1", "q2", "k1", "k2", "v"):
                getattr(s.in_, name).copy_(getattr(new, name))
            g.replay()
            torch.cuda.synchronize()
            q1, q2 = twin.append(new.k1, new.k2, new.v, s.table, n, new.q1, new.q2, inv_freq=freq)
            assert torch.equal(s.out, twin.attend(q1, q2, 0.4, s.table, n))
            n += 1
            assert torch.equal(s.lengths, n) and all(torch.equal(a, b) for a, b in zip(s.pools(), (twin.k1, twin.k2, twin.v)))
    s = made[0]
    want = step(s, s.in_, freq)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        got = step(s, s.in_, freq)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@gpu
def test_copies_and_pickles_have_pages_of_their_own():
    s = Setup([1, 1], [10, 30], 4, 2, 64, 64, 16, BF, "even")
    want = s.attend()
    for other in (copy.deepcopy(s.cache), pickle.loads(pickle.dumps(s.cache))):
        assert torch.equal(other.attend(s.q1, s.q2, 0.4, s.table, s.lengths), want)
        other.v.zero_()
        assert not other.attend(s.q1, s.q2, 0.4, s.table, s.lengths).any()
        assert torch.equal(s.cache.attend(s.q1, s.q2, 0.4, s.table, s.lengths), want)


@gpu
def test_pages_that_get_another_storage():
    """Calls of a signature that was seen before read and write where k1, k2 and v are now, not where they were; without
    a storage, or with one of another shape or type, they are refused."""
    s = Setup([1, 1], [10, 30], 4, 2, 64, 128, 16, BF, "even")
    c, freq = s.cache, torch.rand(32).cuda()
    run = lambda: step(s, s, freq)  # noqa: E731
    want = [run() for _ in range(3)][-1]
    filled = [t.clone() for t in s.pools()]
    old = [t.detach() for t in s.pools()]  # the storages that they had, still in use
    for t, x in zip(s.pools(), filled):
        t.data = x.clone()
    for t in old:
        t.fill_(math.nan)
    assert torch.equal(run(), want) and all(t.isnan().all() for t in old)
    assert all(torch.equal(t, x) for t, x in zip(s.pools(), filled))
    for t in s.pools():
        t.untyped_storage().resize_(0)  # given back ...
        with pytest.raises(ValueError, match="storage"):
            run()
        with pytest.raises(ValueError, match="storage"):
            c.attend(s.q1, s.q2, 0.4, s.table, s.lengths)
    for t, x in zip(s.pools(), filled):
        t.untyped_storage().resize_(x.nbytes)  # ... and taken again
        t.copy_(x)
    assert torch.equal(run(), want)
    for i, x in enumerate(filled):
        for bad in (x[:2], x.float(), x.transpose(1, 2).contiguous().transpose(1, 2), x.cpu()):
            c._held[i] = bad
            with pytest.raises(ValueError, match="must be a contiguous"):
                run()
            with pytest.raises(ValueError, match="must be a contiguous"):
                c.attend(s.q1, s.q2, 0.4, s.table, s.lengths)
        c._held[i] = x
    assert torch.equal(run(), want)


@gpu
@pytest.mark.parametrize("form", ["packed", "counts"])
def test_memory_of_a_call(form):
    """The first call of a kind takes as much as the next ones: its results, and the attention's workspace."""
    s = Setup([301, 1], [70, 600], 8, 2, 64, 128, 64, BF, form)
    size = s.lead * 8 * s.n * 2

    def peak(call):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = call()
        taken = torch.cuda.max_memory_allocated() - before
        assert len(got) in (1, 2)
        return taken

    rounded = lambda n: -(-n // 512) * 512  # noqa: E731
    append = [peak(lambda: s.cache.append(s.k1, s.k2, s.v, s.table, s.lengths, s.q1, s.q2, **s.where)) for _ in range(3)]
    assert append == [2 * rounded(64 * size)] * 3
    lam = torch.tensor(0.4).cuda()
    attend = [peak(lambda: [s.cache.attend(s.q1, s.q2, lam, s.table, s.lengths, **s.where)]) for _ in range(3)]
    assert attend == [attend[-1]] * 3 and attend[0] >= rounded(128 * size)


@gpu
def test_forward_mode_derivatives_are_refused():
    """Not dropped: the calls would return their results without a tangent."""
    s = Setup([1, 1], [10, 30], 4, 2, 64, 64, 16, BF, "even")
    names, lam, freq = ("k1", "k2", "v", "q1", "q2"), torch.tensor(0.4).cuda(), torch.rand(32).cuda()

    def append(rows, freq):
        return s.cache.append(rows["k1"], rows["k2"], rows["v"], s.table, s.lengths, rows["q1"], rows["q2"], inv_freq=freq)

    def attend(rows, lam):
        return s.cache.attend(rows["q1"], rows["q2"], lam, s.table, s.lengths)

    plain = {n: getattr(s, n) for n in names}
    append(plain, freq), attend(plain, lam)
    want = [*s.pools(), attend(plain, lam)]
    want = [t.clone() for t in want]
    dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
    with torch.autograd.forward_ad.dual_level():
        for n in names:
            with pytest.raises(NotImplementedError, match="append"):
                append({**plain, n: dual(plain[n])}, freq)
        with pytest.raises(NotImplementedError, match="append"):
            append(plain, dual(freq))
        for n in ("q1", "q2"):
            with pytest.raises(NotImplementedError, match="attend"):
                attend({**plain, n: dual(plain[n])}, lam)
        with pytest.raises(NotImplementedError, match="attend"):
            attend(plain, dual(lam))
        assert torch.equal(attend(plain, lam), want[3])  # tensors without one
    assert all(torch.equal(a, b) for a, b in zip(s.pools(), want))


@gpu
@pytest.mark.parametrize("dtype, hk, page, d, dv", [(BF, 8, 256, 128, 128), (F32, 1, 16, 64, 128)])
def test_pools_past_31_bits(dtype, hk, page, d, dv):
    """Pages behind 2^31 values (and 2^32 bytes) of the pools, next to the first ones: rows land there and are read from
    there, as in a small cache whose pages hold the same."""
    far = 2 ** 31 // (hk * page * d) + 9
    at = [0, far - 1, 1, far - 2, *range(far - 3, far - 9, -1)]  # where the pages of the small one stand
    s = Setup([90, 1, 1], [40, 130, 7], 8, hk, d, dv, page, dtype, "packed", spare=3)
    small, n = s.cache, s.cache.pages
    at += range(far - 9, far - 9 - n, -1)
    big = tda_amd.PagedKVCache(far, hk, page, d, dv, dtype=dtype)
    assert all(t.numel() > 2 ** 31 and t[far - 8:].data_ptr() - t.data_ptr() > 2 ** 32 - 1 for t in (big.k1, big.k2, big.v))
    idx = torch.tensor(at[:n]).cuda()
    for a, b in zip((small.k1, small.k2, small.v), (big.k1, big.k2, big.v)):
        for i in range(n):
            b[at[i]] = a[i]
    table = torch.where(s.table >= 0, idx.to(torch.int32)[s.table.clamp_min(0).long()], -1)
    freq = torch.rand(d // 2).cuda()
    for new in ([90, 1, 1], [1, 1, 1]):
        where = {"starts": ints(*[sum(new[:i]) for i in range(4)])}
        x = [t[:, :, :sum(new)] for t in (s.k1, s.k2, s.v, s.q1, s.q2)]
        got = [c.append(*x[:3], t, s.lengths, *x[3:], **where, inv_freq=freq) for c, t in ((small, s.table), (big, table))]
        assert all(torch.equal(a, b) for a, b in zip(*got))
        for a, b in zip((small.k1, small.k2, small.v), (big.k1, big.k2, big.v)):
            assert all(torch.equal(a[i], b[at[i]]) for i in range(n))
        want = small.attend(*got[0], 0.4, s.table, s.lengths, **where)
        assert want.any() and torch.equal(big.attend(*got[1], 0.4, table, s.lengths, **where), want)
    del big, a, b
    torch.cuda.empty_cache()


@gpu
def test_results_repeat():
    s = Setup([300, 1, 1, 40], [900, 5000, 3, 2000], 8, 2, 128, 128, 64, BF, "packed").spoil()
    want = s.attend()
    for _ in range(3):
        assert torch.equal(s.cache.attend(s.q1, s.q2, 0.4, s.table, s.lengths, **s.where), want)


@gpu
def test_nothing_to_do():
    c = tda_amd.PagedKVCache(4, 2, 16, 64)
    none = torch.zeros(0, 2, 1, 64, dtype=BF, device="cuda")
    table, lengths = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), ints()
    assert c.append(none, none, none, table, lengths) is None
    assert c.attend(none, none, 0.5, table, lengths).shape == (0, 2, 1, 64)
    none = torch.zeros(3, 2, 0, 64, dtype=BF, device="cuda")
    table, lengths = torch.zeros(3, 3, dtype=torch.int32, device="cuda"), ints(0, 0, 0)
    assert [t.shape for t in c.append(none, none, none, table, lengths, none, none)] == [none.shape] * 2
    assert c.attend(none, none, 0.5, table, lengths).shape == (3, 2, 0, 64)


# ------------------------------------------------------------------ refusals
def test_refusals_on_the_cpu():
    make = tda_amd.PagedKVCache
    with pytest.raises(ValueError, match="GPU only"):
        make(4, 2, 16, 64, device="cpu")
    for kw, match in (({"page_size": 24}, "page_size"), ({"page_size": 8}, "page_size"), ({"pages": 0}, "pages"), ({"kv_heads": 0}, "kv_heads"),
                      ({"head_dim": 96}, "head_dim"), ({"v_head_dim": 256}, "head_dim"), ({"dtype": torch.float64}, "dtype")):
        with pytest.raises(ValueError, match=match):
            make(**{"pages": 4, "kv_heads": 2, "page_size": 16, "head_dim": 64, "device": "cpu", **kw})


@gpu
def test_refusals():
    s = Setup([5, 1], [3, 40], 4, 2, 64, 128, 16, BF, "packed")
    c, good = s.cache, {"starts": s.where["starts"]}
    before = [t.clone() for t in s.pools()]

    def attend(match, q1=s.q1, q2=s.q2, lam=0.4, table=s.table, lengths=s.lengths, err=ValueError, **kw):
        with pytest.raises(err, match=match):
            c.attend(q1, q2, lam, table, lengths, **{**good, **kw})

    def append(match, k1=s.k1, k2=s.k2, v=s.v, table=s.table, lengths=s.lengths, q1=s.q1, q2=s.q2, err=ValueError, **kw):
        with pytest.raises(err, match=match):
            c.append(k1, k2, v, table, lengths, q1, q2, **{**good, **kw})

    for call in (attend, append):
        call("table must be", table=s.table.long())
        call("table must be", table=s.table[0])
        call("table must be on", table=s.table.cpu())
        call("an entry", table=s.table[:, :0])
        call("lengths", lengths=s.lengths[:1])
        call("lengths", lengths=s.lengths.float())
        call("lengths", lengths=s.lengths.cpu())
        call("starts", starts=ints(0, 5))
        call("exclude", counts=ints(5, 1))
        call("batch of 2", starts=None)
        call("counts", starts=None, counts=ints(1))
    attend("shape", q1=s.q1[..., :32])
    attend("shape", q2=s.q2[:, :2])
    attend("multiple", q1=s.q1[:, :3], q2=s.q2[:, :3])
    attend("holds", q1=s.q1.float(), q2=s.q2.float())
    attend("dtype mismatch", q2=s.q2.float())
    attend("GPU only", q1=s.q1.cpu(), q2=s.q2.cpu())
    attend("torch.Tensor", q1=None, err=TypeError)
    attend("lambda_param", lam=torch.rand(3).cuda())
    attend("scale", scale=0.0)
    attend("scale", scale=math.nan)
    attend("most", most=-1)
    append("together", q2=None)
    append("shape", k2=s.k2[:, :, :5])
    append("shape", v=s.v[..., :64])
    append("shape", q1=s.q1[:, :, :5], q2=s.q2[:, :, :5])
    append("holds", k1=s.k1.half(), k2=s.k2.half(), v=s.v.half(), q1=None, q2=None)
    freq = torch.rand(32).cuda()
    append("inv_freq", inv_freq=freq.double())
    append("add up", inv_freq=torch.rand(33).cuda())
    append("add up", inv_freq=freq, sections=(16, 8))
    append("sections", inv_freq=freq, sections=(8, 8, 8, 4, 4))
    append("need inv_freq", sections=(32,))
    append("need inv_freq", positions=torch.zeros(1, 1, 6, dtype=torch.int64).cuda())
    append("positions must have shape", inv_freq=freq, positions=torch.zeros(1, 1, 5, dtype=torch.int64).cuda())
    append("positions must be", inv_freq=freq, positions=torch.zeros(1, 1, 6).cuda())
    append("must be on", inv_freq=freq.cpu())
    assert all(torch.equal(a, b) for a, b in zip(s.pools(), before))
