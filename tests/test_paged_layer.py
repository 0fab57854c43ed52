"""The paged cache, the norm of the heads' outputs and the attention run together, as tda_amd.DifferentialAttention runs
them: training steps with every gradient against float64, and prompts, chunks and decoding steps of several sequences
against the layer's own forward over whole sequences."""
import copy
import math

import pytest
import torch

import tda_amd
from oracle import norm as norm_oracle
from test_differential_layer import Plain, layer, off

gpu = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16
U = 2.0 ** -24


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class PlainNorm(Plain):
    """Plain with the norm of the heads' outputs."""

    def out(self, o):
        r = (o.square().mean(-1, keepdim=True) + self.m.norm_eps).rsqrt()
        return super().out(o * r * self.w["norm_weight"])


def spread_of(v, o):
    return (v.square().mean() / o.square().mean(-1)).mean().sqrt().item()


def test_parameters():
    m = layer("cpu", head_norm=True, v_head_dim=128, lambda_init=0.75, dtype=BF)
    assert m.norm_weight.shape == (128,) and m.norm_weight.dtype == BF and m.norm_weight.tolist() == [0.25] * 128
    assert "norm_weight" in m.state_dict() and "head_norm=True" in repr(m)
    plain = layer("cpu")
    assert plain.norm_weight is None and "norm_weight" not in plain.state_dict() and "head_norm" not in repr(plain)


@gpu
@pytest.mark.parametrize("kw", [{}, {"v_head_dim": 128, "bias": True}])
@pytest.mark.parametrize("n", [1, 37, 150])
def test_training_step_with_the_norm(kw, n):
    """Every sum of the layer is off by its length times 2^-24 of its magnitudes, as in the layer without the norm, whose
    tolerance this is.  An output is a weighted mean of values and off as they are large; the norm divides a row by its
    root mean square, so its error counts relative to that: the values' root mean square over the row's, squares
    averaged over the rows, as the norm of all differences adds them up."""
    m = layer(head_norm=True, **kw)
    x = torch.randn(2, n, 96, generator=torch.Generator().manual_seed(5))
    up = torch.randn(2, n, 96, generator=torch.Generator().manual_seed(7))
    plain, xd = PlainNorm(m), x.double().requires_grad_()
    want = plain(xd, torch.arange(n).expand(1, 2, n))
    want.backward(up.double())
    xg = x.cuda().requires_grad_()
    got = m(xg)
    got.backward(up.cuda())
    with torch.no_grad():
        q1, q2, k1, k2, v = plain.project(xd)
        q1, q2, k1, k2 = (plain.turn(t, torch.arange(n).expand(1, 2, n)) for t in (q1, q2, k1, k2))
        score = (q1.norm(dim=-1).max() * k1.norm(dim=-1).max() / 8).item()
        spread = spread_of(v, plain.attend(q1, q2, k1, k2, v))
    tol = 4 * 3 * (96 + 4 * m.v_head_dim + 64 + 2 * n + norm_oracle.CHAIN) * U * (1 + score) * (1 + spread)
    assert tol < 0.1
    assert off(got, want.detach()) < tol and off(xg.grad, xd.grad) < tol
    for name, p in m.named_parameters():
        assert p.grad is not None and off(p.grad, plain.w[name].grad) < tol, name


@gpu
def test_training_step_bf16_runs():
    m = layer(dtype=BF, head_norm=True)
    x = torch.randn(2, 200, 96, device="cuda", dtype=BF, requires_grad=True)
    m(x).square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in (x, *m.parameters()))


def serve(m, x, total, schedule, form, pages=40, page_size=16):
    """Runs the sequences x[i, :total[i]] through m over a paged cache, new[i] rows a step: (outputs, cache, table)."""
    cache = m.new_paged_cache(pages, page_size)
    for t in (cache.k1, cache.k2, cache.v):
        t.fill_(math.nan)  # what nobody wrote
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(2))[: 3 * (pages // 3)].to(torch.int32).view(3, -1).cuda()
    lengths, done, out = ints(0, 0, 0), [0, 0, 0], torch.zeros_like(x)
    for new in schedule:
        if form == "packed":
            now = torch.cat([x[i, a:a + n] for i, (a, n) in enumerate(zip(done, new))])[None]
            got = m(now, cache=cache, table=table, lengths=lengths, starts=ints(*[sum(new[:i]) for i in range(4)]))[0]
            parts = got.split(list(new))
        else:
            now = x.new_full((3, max(new), x.shape[2]), 7.0)
            for i, (a, n) in enumerate(zip(done, new)):
                now[i, :n] = x[i, a:a + n]
            got = m(now, cache=cache, table=table, lengths=lengths, counts=ints(*new))
            parts = [got[i, :n] for i, n in enumerate(new)]
        assert not got.requires_grad
        for i, (a, n) in enumerate(zip(done, new)):
            out[i, a:a + n] = parts[i]
        lengths = lengths + ints(*new)
        done = [a + n for a, n in zip(done, new)]
    assert done == list(total)
    return out, cache, table


@gpu
@pytest.mark.parametrize("kw", [{}, {"v_head_dim": 128, "head_norm": True}, {"num_heads": 20, "kv_heads": 1, "head_dim": 128, "v_head_dim": 256},
                                {"rotary_sections": (16, 8), "head_norm": True, "bias": True}])
@pytest.mark.parametrize("form", ["packed", "counts"])
def test_serving_gives_what_the_whole_sequences_give(kw, form):
    """fp32.  Both sides compute the same formula in 24 bits; products of other row counts add up in other orders.  Each is
    within the training step's tolerance of the formula, so they are within twice it of each other."""
    m = layer(**kw)
    total = (90, 41, 70)
    x = torch.randn(3, 90, 96, generator=torch.Generator().manual_seed(8)).cuda()
    got, cache, table = serve(m, x, total, ((50, 3, 20), (1, 30, 1), (1, 1, 0), (38, 7, 49)), form)
    with torch.no_grad():
        for i, n in enumerate(total):
            want = m(x[i:i + 1, :n])
            q1, q2, k1, k2, v = m.project(x[i:i + 1, :n])
            score = (q1.norm(dim=-1).max() * k1.norm(dim=-1).max() / math.sqrt(m.head_dim)).item()
            spread = 1.0
            if m.norm_weight is not None:
                freq, pos = m._frequencies(), torch.arange(n, device="cuda").expand(len(m.rotary_sections), 1, n)
                o = tda_amd.differential_attention(*tda_amd.rotary_axes((q1, q2, k1, k2), pos, freq, m.rotary_sections), v, m.lambda_param)
                spread += spread_of(v, o)
            tol = 2 * 4 * 3 * (96 + m.num_heads * m.v_head_dim + m.head_dim + 2 * n + norm_oracle.CHAIN) * U * (1 + score) * spread
            assert tol < 0.1 and off(got[i:i + 1, :n], want.double().cpu()) < tol


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_serving_under_autocast(dtype):
    """A float32 layer whose projections come out in 16 bits, over pages of that type: the operators one by one give the
    same.  Pages of the weights' type are refused."""
    m = layer(head_norm=True, v_head_dim=128, rotary_sections=(16, 8))
    x = torch.randn(1, 45, 96, generator=torch.Generator().manual_seed(8)).cuda()
    where = {"table": ints(3, 1, 0, 4).view(2, 2), "lengths": ints(0, 9), "starts": ints(0, 30, 45)}
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        caches = [m.new_paged_cache(6, 16, dtype=dtype) for _ in range(2)]
        assert caches[0].dtype == dtype and m.new_paged_cache(6, 16).dtype == F32
        for c in caches:
            for t in (c.k1, c.k2, c.v):
                t.fill_(0.25)
        got = m(x, cache=caches[0], **where)
        q1, q2, k1, k2, v = m.project(x)
        assert q1.dtype == dtype and got.dtype == dtype
        q1, q2 = caches[1].append(k1, k2, v, q1=q1, q2=q2, **where, inv_freq=m._frequencies(), sections=(16, 8))
        o = caches[1].attend(q1, q2, m.lambda_param, **where)
        o = tda_amd.layer_norm(o, m.norm_weight, eps=m.norm_eps, center=False)
        assert torch.equal(got, m.out_proj(o.transpose(1, 2).flatten(2)))
        assert all(torch.equal(a, b) for a, b in zip(caches[0]._held, caches[1]._held))
        with pytest.raises(ValueError, match="holds"):
            m(x, cache=m.new_paged_cache(6, 16), **where)


@gpu
def test_padding_gives_the_bias():
    m = layer(bias=True, head_norm=True)
    x = torch.randn(1, 12, 96, device="cuda")
    cache = m.new_paged_cache(6, 16)
    y = m(x, cache=cache, table=ints(3, 1, 0, 4).view(2, 2), lengths=ints(0, 0), starts=ints(0, 4, 9))
    assert torch.equal(y[0, 9:], m.out_proj.bias.detach().expand(3, 96))


@gpu
def test_captured_serving_step():
    """A graph of one step that adds to the lengths in it, replayed with other work between; another layer's pages share
    table and lengths."""
    layers = [layer(dtype=BF, head_norm=True), layer(dtype=BF)]
    table = torch.randperm(12).to(torch.int32).cuda().view(2, 6)
    with torch.no_grad():
        x = torch.randn(2, 30, 96, device="cuda", dtype=BF)
        own = [m.new_paged_cache(12, 16) for m in layers]
        for c in own:
            for t in (c.k1, c.k2, c.v):
                t.zero_()

        def run(caches, rows, lengths):
            for m, c in zip(layers, caches):
                rows = rows + m(rows, cache=c, table=table, lengths=lengths)
            return rows

        lengths = ints(0, 0)
        run(own, x[:, :20], lengths)
        lengths += 20
        eager, n = copy.deepcopy(own), lengths.clone()
        now = x[:, 20:21].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(own, now, lengths)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(own, now, lengths)
            lengths += 1
        for i in range(20, 30):
            now.copy_(x[:, i:i + 1])
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, run(eager, x[:, i:i + 1].clone(), n))
            n += 1
    assert lengths.tolist() == [30, 30]
    for a, b in zip(own, eager):
        assert torch.equal(a.k1, b.k1) and torch.equal(a.k2, b.k2) and torch.equal(a.v, b.v)


@gpu
def test_refusals():
    m = layer()
    x = torch.zeros(2, 1, 96, device="cuda")
    cache, table, lengths = m.new_paged_cache(4, 16), ints(0, 1).view(2, 1), ints(0, 0)
    with pytest.raises(ValueError, match="needs table and lengths"):
        m(x, cache=cache)
    with pytest.raises(ValueError, match="needs table and lengths"):
        m(x, cache=cache, table=table)
    with pytest.raises(ValueError, match="go with a paged cache"):
        m(x, table=table, lengths=lengths)
    with pytest.raises(ValueError, match="go with a paged cache"):
        m(x, cache=m.new_cache(2, 8), lengths=lengths)
    with pytest.raises(ValueError, match="exclude"):
        m(x, kv_lens=lengths, cache=cache, table=table, lengths=lengths)
    with pytest.raises(ValueError, match="batch of 2"):
        m(x[:1], cache=cache, table=table, lengths=lengths)
    with pytest.raises(ValueError, match="holds"):
        m(x, cache=layer(dtype=BF).new_paged_cache(4, 16), table=table, lengths=lengths)


# ------------------------------------------------------------------ what layers without these could do
def test_layers_pickled_without_a_norm():
    m = tda_amd.DifferentialAttention(128, 2, bias=True)
    state = copy.deepcopy(m.__dict__)
    del state["norm_eps"], state["_parameters"]["norm_weight"]
    old = tda_amd.DifferentialAttention.__new__(tda_amd.DifferentialAttention)
    old.__setstate__(state)
    assert old.norm_weight is None and old.norm_eps == 1e-5 and repr(old) == repr(m)
    assert list(old.state_dict()) == list(m.state_dict()) and "norm_weight" not in old.state_dict()
    assert old.load_state_dict(m.state_dict()).missing_keys == []


def test_subclasses_with_the_arguments_of_a_4_bit_cache():
    """A forward of four arguments is called again without gradients as it was called."""
    calls = []

    class Mine(tda_amd.DifferentialAttention):
        def forward(self, x, positions=None, kv_lens=None, cache=None):
            calls.append((positions, kv_lens, cache, torch.is_grad_enabled()))
            return x if len(calls) == 2 else super().forward(x, positions, kv_lens, cache)

    class Cache:
        batch = 3

    cache, x = Cache(), torch.zeros(3, 1, 128)
    assert Mine(128, 2)(x, cache=cache) is x
    assert calls == [(None, None, cache, True), (None, None, cache, False)]
