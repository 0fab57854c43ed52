"""Softmax differential attention (tda_amd.differential_attention): refusals on the CPU, and on the GPU
every output and gradient against the definition in float64, within the bounds of oracle/softmax.py,
which count half a step of the type for each rounding."""
import math

import pytest
import torch

import tda_amd
from oracle import softmax as oracle

BF, F32, F16 = torch.bfloat16, torch.float32, torch.float16
U = {BF: 2.0 ** -8, F32: 2.0 ** -24, F16: 2.0 ** -11}
gpu = pytest.mark.gpu


def rows(shape, seed, dtype=BF, spread=1.0, seq_major=False, device="cuda"):
    g = torch.Generator("cpu").manual_seed(seed)
    b, h, n, d = shape
    x = (torch.randn(b, n, h, d, generator=g) * spread).transpose(1, 2)
    return (x if seq_major else x.contiguous()).to(dtype).to(device)


def inputs(b, h, hk, n, nk, d, dv, dtype, seq_major=False, spread=1.5):
    return [rows((b, h, n, d), 1, dtype, spread, seq_major), rows((b, h, n, d), 2, dtype, spread, seq_major),
            rows((b, hk, nk, d), 3, dtype, 1.0, seq_major), rows((b, hk, nk, d), 4, dtype, 1.0, seq_major),
            rows((b, hk, nk, dv), 5, dtype, 1.0, seq_major)]


def within(got, ref, name, u, extra=1e-30):
    """Every element within its bound; a type with fewer than 32 bits rounds the result once more."""
    want, off = ref[name], ref[name + "_off"]
    assert got.shape == want.shape, name
    far = (got.double() - want).abs() - off - u * want.abs() - extra
    assert torch.isfinite(got).all(), name
    assert far.max().item() <= 0, f"{name}: {far.max().item():.3g} past its bound of {off.flatten()[far.argmax()].item():.3g}"


def tiny(xs, lam, dout=None):
    """How far float16's smallest values may take a result, by name: below 2^-14 they are off by up to 2^-25.
    Forward weights are shares of a row's largest; the backward's are scaled by 2^8 (|lambda| <= 1 here), its score
    gradients by at least 2^12 / a, where a bounds them by half; the results themselves round last."""
    q, k, v = (max(x.abs().max().item() for x in y) for y in (xs[:2], xs[2:4], xs[4:]))
    most, last = float(torch.as_tensor(lam).abs().max()), 2.0 ** -25
    b, h, n, d = xs[0].shape
    nk, rows_of = xs[4].shape[2], n * h // xs[4].shape[1]
    res = {"out": last + nk * 2.0 ** -25 * (1 + most) * v}
    if dout is not None:
        norm = lambda x: x.double().norm(dim=-1).max().item()  # noqa: E731
        a = norm(dout) * norm(xs[4]) * max(1.0, most)
        dq, dk = (last + m * a * 2.0 ** -37 * x / math.sqrt(d) for m, x in ((nk, k), (rows_of, q)))
        res |= {"dq1": dq, "dq2": dq, "dk1": dk, "dk2": dk, "dv": last + rows_of * 2.0 ** -33 * dout.abs().max().item()}
    return res


def check(b, h, hk, n, nk, d, dv, dtype, lam, train=True, seq_major=False, **kw):
    xs = inputs(b, h, hk, n, nk, d, dv, dtype, seq_major)
    u = U[dtype]
    lam = lam if not isinstance(lam, torch.Tensor) else lam.cuda()
    ref_kw = {k: (v.cpu() if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}
    dout = rows((b, h, n, dv), 6, dtype) if train else None
    more = tiny(xs, lam, dout) if dtype == F16 else {}
    if not train:
        ref = oracle.attention(*xs, lam, u=u, **ref_kw)
        within(tda_amd.differential_attention(*xs, lam, **kw), ref, "out", u, 1e-30 + more.get("out", 0.0))
        return
    leaves = [x.requires_grad_(True) for x in xs]
    lam_leaf = lam.clone().requires_grad_(True) if isinstance(lam, torch.Tensor) else lam
    out = tda_amd.differential_attention(*leaves, lam_leaf, **kw)
    out.backward(dout)
    ref = oracle.attention(*xs, lam, u=u, dout=dout, **ref_kw)
    within(out, ref, "out", u, 1e-30 + more.get("out", 0.0))
    for x, name in zip(leaves, ("dq1", "dq2", "dk1", "dk2", "dv")):
        within(x.grad, ref, name, u, 1e-30 + more.get(name, 0.0))
    if isinstance(lam, torch.Tensor):
        assert lam_leaf.grad.dtype == lam.dtype
        within(lam_leaf.grad, ref, "dlam", U[lam.dtype])


# ------------------------------------------------------------------ refusals (CPU)
def cpu(shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


def test_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="GPU only"):
        q, k = cpu((1, 2, 3, 64)), cpu((1, 2, 3, 64))
        tda_amd.differential_attention(q, q, k, k, k, 0.5)


@pytest.mark.parametrize("change, error", [
    (dict(q1=None), TypeError), (dict(q1=cpu((2, 3, 64))), ValueError), (dict(k1=cpu((1, 2, 3, 64), F16)), ValueError),
    (dict(v=torch.zeros(1, 2, 3, 64, dtype=torch.int32)), ValueError)])
def test_refuses_bad_rows(change, error):
    a = {"q1": cpu((1, 2, 3, 64)), "q2": cpu((1, 2, 3, 64)), "k1": cpu((1, 2, 3, 64)), "k2": cpu((1, 2, 3, 64)),
         "v": cpu((1, 2, 3, 64))}
    a.update(change)
    with pytest.raises(error):
        tda_amd.differential_attention(*a.values(), 0.5)


@gpu
@pytest.mark.parametrize("change", [
    dict(q2=(1, 4, 4, 64)), dict(k1=(1, 2, 4, 64)), dict(k2=(1, 2, 5, 32)), dict(v=(2, 2, 5, 64)), dict(v=(1, 3, 5, 64)),
    dict(lam=torch.zeros(3)), dict(lam=torch.zeros(2, 2)), dict(lam=torch.zeros(4, dtype=torch.int32)),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(q_offset=-1),
    dict(q_offset=torch.zeros(3, dtype=torch.int32)), dict(kv_lens=torch.zeros(1)), dict(kv_lens=torch.zeros(2, dtype=torch.int64)),
    dict(kv_lens=torch.zeros(1, dtype=torch.int32)), dict(v=(1, 2, 5, 264)), dict(q1=(1, 4, 3, 136))])
def test_refusals(change):
    a = dict(q1=(1, 4, 3, 64), q2=(1, 4, 3, 64), k1=(1, 2, 5, 64), k2=(1, 2, 5, 64), v=(1, 2, 5, 64))
    kw = {k: change[k] for k in ("scale", "q_offset", "kv_lens") if k in change}
    if "kv_lens" in kw and kw["kv_lens"].dtype != torch.int32:
        kw["kv_lens"] = kw["kv_lens"].cuda()  # the int32 one stays on the CPU: the wrong device
    if isinstance(kw.get("q_offset"), torch.Tensor):
        kw["q_offset"] = kw["q_offset"].cuda()
    a.update({k: v for k, v in change.items() if k in a})
    if change.get("q1", (0,))[-1] == 136:
        a.update(q2=a["q1"], k1=(1, 2, 5, 136), k2=(1, 2, 5, 136))
    xs = [torch.zeros(s, device="cuda") for s in a.values()]
    with pytest.raises(ValueError):
        tda_amd.differential_attention(*xs, change.get("lam", 0.5), **kw)


# ------------------------------------------------------------------ results (GPU)
DIMS = [(64, 64), (64, 128), (128, 128), (128, 256)]


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d, dv", DIMS)
@pytest.mark.parametrize("n", [1, 31, 64, 129, 300])
def test_training_step(dtype, d, dv, n):
    check(2, 2, 2, n, n, d, dv, dtype, torch.tensor([0.8, -0.3]))


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h, hk, n, nk, off", [(6, 2, 70, 200, None), (4, 1, 129, 129, None), (3, 3, 40, 300, 17),
                                               (8, 2, 200, 64, 0), (5, 5, 130, 131, 1), (10, 2, 33, 400, 390)])
def test_shared_heads_and_offsets(dtype, h, hk, n, nk, off):
    check(2, h, hk, n, nk, 64, 128, dtype, torch.tensor(0.6), q_offset=off)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [[0, 1, 150], [64, 65, 63], [150, 300, -5]])
def test_padded_batch(dtype, causal, lens):
    check(3, 4, 2, 150, 150, 64, 64, dtype, torch.tensor([0.1, 0.9, 0.5, -2.0]), causal=causal,
          kv_lens=torch.tensor(lens, dtype=torch.int32).cuda())


@gpu
@pytest.mark.parametrize("n", [1, 3, 40, 140])
@pytest.mark.parametrize("train", [True, False])
def test_offsets_of_each_sequence(n, train):
    """Rows before the first position (negative ones) see nothing."""
    check(4, 4, 2, n, 200, 128, 128, BF, torch.tensor(0.7), train=train,
          q_offset=torch.tensor([-20, 0, 77, 199], dtype=torch.int64).cuda(),
          kv_lens=torch.tensor([200, 1, 100, 200], dtype=torch.int64).cuda())


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", ["scalar", "one", "heads", "rows", "batch", "per_batch_head", "expanded"])
@pytest.mark.parametrize("lam_dtype", [BF, F32, F16])
def test_lambda_of_every_shape(dtype, shape, lam_dtype):
    b, h, n = 2, 3, 45
    g = torch.Generator("cpu").manual_seed(9)
    size = {"scalar": (), "one": (1,), "heads": (h,), "rows": (b, h, n), "batch": (b, 1, 1), "per_batch_head": (b, h, 1),
            "expanded": (1, 1, n)}[shape]
    lam = torch.rand(size, generator=g).to(lam_dtype)
    if shape == "expanded":
        lam = lam.expand(b, h, n)
    check(b, h, h, n, n, 64, 64, dtype, lam)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
@pytest.mark.parametrize("d, dv", DIMS + [(16, 16), (32, 64), (80, 72), (64, 200)])
@pytest.mark.parametrize("h, hk, n, nk", [(1, 1, 1, 1), (8, 8, 1, 1000), (8, 2, 1, 33), (20, 1, 1, 700), (4, 4, 4, 129),
                                          (6, 3, 7, 520), (2, 1, 16, 3000)])
def test_few_rows(dtype, d, dv, h, hk, n, nk):
    """The kernels that split the key axis: decoding steps and short chunks."""
    check(3, h, hk, n, nk, d, dv, dtype, torch.linspace(0.2, 0.9, h), train=False,
          kv_lens=torch.tensor([nk, nk // 2, 0], dtype=torch.int32).cuda(), causal=n > 1)


@gpu
@pytest.mark.parametrize("d, dv, dtype", [(16, 16, BF), (32, 80, F32), (96, 96, BF), (64, 200, F32), (64, 64, F16)])
def test_padded_widths_and_float16(d, dv, dtype):
    check(1, 2, 2, 100, 100, d, dv, dtype, torch.tensor(0.5))


@gpu
@pytest.mark.parametrize("n", [1, 200])
def test_strided_rows(n):
    """Views of one projection output, every second head, an odd offset into a buffer."""
    check(2, 4, 4, n, 200, 64, 64, BF, torch.tensor(0.5), seq_major=True)
    xs = inputs(2, 8, 8, n, 200, 64, 128, BF)
    want = tda_amd.differential_attention(*(x[:, ::2].contiguous() for x in xs), 0.5)
    assert torch.equal(tda_amd.differential_attention(*(x[:, ::2] for x in xs), 0.5), want)
    off = [torch.empty(x.numel() + 1, dtype=BF, device="cuda")[1:].view(x.shape).copy_(x) for x in xs]
    assert torch.equal(tda_amd.differential_attention(*(x[:, ::2] for x in off), 0.5), want)
    wide = [torch.cat((x, x), -1)[..., ::2] for x in xs]  # a last stride of two
    a = tda_amd.differential_attention(*wide, 0.5)
    assert torch.equal(a, tda_amd.differential_attention(*(x.contiguous() for x in wide), 0.5))


@gpu
@pytest.mark.parametrize("n", [1, 40, 260])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_keys_may_hold_anything(n, bad):
    lens = torch.tensor([150, 37], dtype=torch.int32).cuda()
    xs = inputs(2, 2, 2, n, 300, 64, 64, BF)
    for x in xs[2:]:
        x[0, :, 150:] = 0
        x[1, :, 37:] = 0
    off = torch.tensor([150 - n, 37 - n]).cuda()
    want = tda_amd.differential_attention(*xs, 0.5, q_offset=off, kv_lens=lens)
    for x in xs[2:]:
        x[0, :, 150:] = bad
        x[1, :, 37:] = bad
    assert torch.equal(tda_amd.differential_attention(*xs, 0.5, q_offset=off, kv_lens=lens), want)
    if n == 260:
        return
    # a cache with room: rows behind the last query's position
    a = tda_amd.differential_attention(*(x[1:] for x in xs), 0.5, q_offset=36 - n + 1 if n < 37 else 0)
    assert n >= 37 or torch.isfinite(a).all()


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_hidden_keys_in_the_backward(bad):
    lens = torch.tensor([100, 37], dtype=torch.int32).cuda()
    xs = inputs(2, 4, 2, 150, 150, 64, 64, BF)
    dout = rows((2, 4, 150, 64), 6)
    grads = []
    for fill in (0.0, bad):
        for x in xs[2:]:
            x[0, :, 100:] = fill
            x[1, :, 37:] = fill
        leaves = [x.detach().clone().requires_grad_(True) for x in xs]
        tda_amd.differential_attention(*leaves, 0.5, kv_lens=lens).backward(dout)
        grads.append([x.grad for x in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@gpu
def test_visible_nan_reaches_its_rows():
    xs = inputs(1, 1, 1, 300, 300, 64, 64, BF)
    xs[2][0, 0, 250] = math.nan
    out = tda_amd.differential_attention(*xs, 0.5)
    assert torch.isnan(out[0, 0, 250:]).all() and torch.isfinite(out[0, 0, :250]).all()


@gpu
@pytest.mark.parametrize("scale", [1e-4, 3.0, 40.0])
def test_scales_and_large_scores(scale):
    """Scores of several hundreds: one key takes all the weight; running maxima move late and far."""
    xs = [x * 3 for x in inputs(1, 2, 2, 200, 200, 64, 64, F32)]
    out = tda_amd.differential_attention(*xs, 0.9, scale)
    ref = oracle.attention(*xs, 0.9, scale, u=U[F32])
    within(out, ref, "out", U[F32])


@gpu
def test_growing_scores_move_the_maximum():
    q1, q2, k1, k2, v = inputs(1, 1, 1, 256, 256, 64, 64, F32)
    ramp = torch.linspace(0, 40, 256, device="cuda")[None, None, :, None]
    k1, k2 = k1 + ramp * q1.mean(2, keepdim=True).sign(), k2 - ramp
    out = tda_amd.differential_attention(q1, q2, k1, k2, v, 0.5, causal=False)
    within(out, oracle.attention(q1, q2, k1, k2, v, 0.5, causal=False, u=U[F32]), "out", U[F32])


@gpu
@pytest.mark.parametrize("shape", [(0, 2, 3, 5), (2, 2, 0, 5), (2, 2, 3, 0)])
def test_empty(shape):
    b, h, n, nk = shape
    xs = [torch.randn(b, h, m, 64, device="cuda", requires_grad=True) for m in (n, n, nk, nk, nk)]
    lam = torch.tensor(0.5, device="cuda", requires_grad=True)
    out = tda_amd.differential_attention(*xs, lam)
    assert out.shape == (b, h, n, 64) and not out.any()
    out.sum().backward()
    assert all(x.grad is not None and not x.grad.any() for x in (*xs, lam))


@gpu
def test_gradient_against_differences():
    """Directional differences of the operator itself, in float32: h = 2^-7 balances h^2 / 6 of the third
    derivative (scores of order one) against 2^-24 / h of the rounding of a sum of 2 x 33 x 64 terms."""
    xs = inputs(1, 2, 1, 33, 33, 64, 64, F32, spread=1.0)
    lam = torch.tensor([0.3, 0.7], device="cuda")
    dout = rows((1, 2, 33, 64), 6, F32)
    leaves = [x.clone().requires_grad_(True) for x in (*xs, lam)]
    tda_amd.differential_attention(*leaves).backward(dout)
    f = lambda *a: (tda_amd.differential_attention(*a).double() * dout.double()).sum().item()  # noqa: E731
    for i, x in enumerate(leaves):
        g = torch.Generator("cpu").manual_seed(i)
        way = torch.randn(x.shape, generator=g).cuda()
        way /= way.norm()
        h = 2.0 ** -7
        at = lambda t: [y.detach() + (t * way if j == i else 0) for j, y in enumerate(leaves)]  # noqa: E731
        diff = (f(*at(h)) - f(*at(-h))) / (2 * h)
        want = (x.grad.double() * way.double()).sum().item()
        size = dout.norm().item()  # |f| changes by at most about |dout| |v| per unit way
        assert abs(diff - want) <= (h * h + 64 * 2.0 ** -24 / h) * size


@gpu
def test_partial_gradients_and_second_backward():
    xs = inputs(1, 2, 2, 70, 70, 64, 64, BF)
    dout = rows((1, 2, 70, 64), 6)
    full = [x.clone().requires_grad_(True) for x in xs]
    tda_amd.differential_attention(*full, 0.5).backward(dout)
    for i in range(5):
        some = [x.clone().requires_grad_(j == i) for j, x in enumerate(xs)]
        out = tda_amd.differential_attention(*some, 0.5)
        out.backward(dout, retain_graph=True)
        first = some[i].grad.clone()
        out.backward(dout)
        assert torch.equal(first, full[i].grad) and torch.equal(some[i].grad, first + first)
    # one leaf in two places
    q = xs[0].clone().requires_grad_(True)
    tda_amd.differential_attention(q, q, *xs[2:], 0.5).backward(dout)
    a, b = (xs[0].clone().requires_grad_(True) for _ in range(2))
    tda_amd.differential_attention(a, b, *xs[2:], 0.5).backward(dout)
    assert torch.equal(q.grad, a.grad + b.grad)


@gpu
def test_expanded_upstream_gradient():
    xs = [x.requires_grad_(True) for x in inputs(2, 2, 2, 50, 50, 64, 64, F32)]
    tda_amd.differential_attention(*xs, 0.5).sum().backward()
    got = [x.grad.clone() for x in xs]
    for x in xs:
        x.grad = None
    tda_amd.differential_attention(*xs, 0.5).backward(torch.ones(2, 2, 50, 64, device="cuda"))
    assert all(torch.equal(a, x.grad) for a, x in zip(got, xs))


@gpu
def test_same_bits_every_time():
    xs = inputs(2, 8, 2, 500, 500, 128, 128, BF)
    dout = rows((2, 8, 500, 128), 6)
    runs = []
    for _ in range(3):
        leaves = [x.detach().clone().requires_grad_(True) for x in xs]
        lam = torch.full((8,), 0.4, device="cuda", requires_grad=True)
        out = tda_amd.differential_attention(*leaves, lam)
        out.backward(dout)
        runs.append([out.detach(), lam.grad, *(x.grad for x in leaves)])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


@gpu
@pytest.mark.parametrize("n, nk, dtype", [(1, 3000, BF), (260, 260, BF), (260, 260, F16)])
def test_captured(n, nk, dtype):
    """Graphs of the forward and of a training step, replayed between eager work and compared with it."""
    xs = [x.requires_grad_(n > 1) for x in inputs(2, 4, 2, n, nk, 64, 64, dtype)]
    lens = torch.tensor([nk, nk - 7], dtype=torch.int32).cuda()
    lam = torch.full((4,), 0.5, device="cuda", requires_grad=n > 1)
    dout = rows((2, 4, n, 64), 6, dtype)

    def step():
        out = tda_amd.differential_attention(*xs, lam, kv_lens=lens)
        return [out.detach(), *torch.autograd.grad(out, [*xs, lam], dout)] if n > 1 else [out]  # no graph outlives a step

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for k in range(3):
        with torch.no_grad():
            for x in xs:
                x.mul_(0.9 - 0.1 * k)
        lens.fill_(nk - 30 * k)
        for g, got in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            want = [t.clone() for t in step()]
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_other_stream():
    xs = inputs(2, 4, 2, 300, 300, 64, 64, BF)
    want = tda_amd.differential_attention(*xs, 0.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [tda_amd.differential_attention(*xs, 0.5) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, want) for g in got)


@gpu
def test_rows_far_into_memory():
    """A cache whose rows lie beyond 2^32 bytes from its start: the last sequence of a large buffer."""
    b, hk, cap, d = 5, 4, 1 << 20, 128  # 5 GiB a tensor
    k = torch.zeros(b, hk, cap, d, dtype=BF, device="cuda")
    small = inputs(1, 8, hk, 1, 500, d, d, BF)
    k[-1, :, cap - 500:] = small[2][0]
    held = torch.tensor([0] * (b - 1) + [cap], dtype=torch.int32).cuda()
    q = [torch.cat([x] * b) for x in small[:2]]
    out = tda_amd.differential_attention(*q, k, k, k, 0.5, 0.5, causal=False, kv_lens=held)
    assert not out[:-1].any()
    kk = small[2].double().repeat_interleave(2, 1)
    o = []
    for x in small[:2]:  # the zero rows weigh exp(0) each and add nothing to the values
        s = (x.double() @ kk.transpose(2, 3)) * 0.5
        m = s.amax(-1, keepdim=True).clamp_min(0)
        e = torch.exp(s - m)
        o.append((e / (e.sum(-1, keepdim=True) + (cap - 500) * torch.exp(-m)), kk))
    want = o[0][0] @ kk - 0.5 * (o[1][0] @ kk)
    big = o[0][0] @ kk.abs() + 0.5 * (o[1][0] @ kk.abs())
    # weights and output rounded to bf16; the sum of 2^20 terms in 1024 parts of 32-bit adds, the
    # scores' 32-bit sums: under 2^-12 of the magnitudes together
    assert ((out[-1:].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * big).all()


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_no_keys_and_rows_that_are_not_finite(bad):
    q = rows((1, 2, 3, 64), 1, F32).fill_(bad).requires_grad_()
    none = torch.empty(1, 2, 0, 64, device="cuda", requires_grad=True)
    out = tda_amd.differential_attention(q, q, none, none, none, 0.5)
    assert out.shape == (1, 2, 3, 64) and not out.any()
    out.sum().backward()
    assert not q.grad.any() and none.grad.shape == none.shape


@gpu
def test_two_threads_on_two_streams():
    """Training steps of two threads at once, each on a stream of its own, give what they give alone."""
    import threading
    sets = [inputs(2, 4, 2, 300, 300, 64, 128, BF), inputs(1, 8, 8, 500, 500, 128, 128, BF)]
    sets = [[x.detach().clone().requires_grad_() for x in xs] for xs in sets]

    def step(xs):
        out = tda_amd.differential_attention(*xs, 0.5)
        return [out.detach(), *torch.autograd.grad(out, xs, out.detach())]

    want = [step(xs) for xs in sets]
    got, failed = [None, None], []
    torch.cuda.synchronize()

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[k] = [step(sets[k]) for _ in range(5)]
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for k in range(2):
        assert all(torch.equal(a, b) for res in got[k] for a, b in zip(res, want[k]))


@gpu
def test_the_same_tensors_twice():
    """q1 = q2, k1 = k2 and lambda 1: nothing is left, and each gradient is the two branches' together."""
    q, k, v = inputs(1, 2, 2, 200, 200, 64, 64, F32)[::2]
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = tda_amd.differential_attention(q, q, k, k, v, 1.0)
    # each branch is off by its own bound: 200 terms in 24 bits
    assert out.abs().max().item() <= 4 * 200 * 2.0 ** -24 * v.abs().max().item()
    out.sum().backward()
    lim = 4 * 200 * 64 * 2.0 ** -24 * v.abs().max().item() * 3
    assert q.grad.abs().max().item() <= lim * k.abs().max().item() and k.grad.abs().max().item() <= lim * 200 * q.abs().max().item()


@gpu
@pytest.mark.parametrize("scale", [0.0, -1.0, math.nan, math.inf, 1e-31, 1e31])
def test_scale_out_of_range(scale):
    xs = inputs(1, 2, 2, 5, 5, 64, 64, BF)
    with pytest.raises(ValueError, match="scale"):
        tda_amd.differential_attention(*xs, 0.5, scale=scale)


@gpu
def test_calls_of_one_signature_take_their_own_tensors():
    """A repeated call is the first one's with other addresses, lambdas and lengths; what differs is checked."""
    for n, nk in ((1, 700), (40, 300)):
        lam = torch.tensor([0.2, 0.5, 0.7, 0.9]).cuda()
        want = []
        for fresh in (False, True):
            for k in range(3):
                xs = [rows((2, h, m, 64), 10 * k + j, BF) for j, (h, m) in enumerate(((4, n), (4, n), (2, nk), (2, nk), (2, nk)))]
                lens = torch.tensor([nk - k, nk // (k + 2)], dtype=torch.int32).cuda()
                if fresh:  # another signature: the lengths in 64 bits
                    assert torch.equal(tda_amd.differential_attention(*xs, lam * k, kv_lens=lens.long()), want[k])
                else:
                    want.append(tda_amd.differential_attention(*xs, lam * k, kv_lens=lens))
        xs = [rows((2, h, m, 64), 70 + j, BF) for j, (h, m) in enumerate(((4, n), (4, n), (2, nk), (2, nk), (2, nk)))]
        ref = tda_amd.differential_attention(*xs, lam)
        assert torch.equal(tda_amd.differential_attention(*xs, lam), ref)
        off = torch.empty(xs[0].numel() + 1, dtype=BF, device="cuda")[1:].view_as(xs[0]).copy_(xs[0])  # 2 bytes past a line
        assert torch.equal(tda_amd.differential_attention(off, *xs[1:], lam), ref)
        xs[4].requires_grad_()
        assert tda_amd.differential_attention(*xs, lam).requires_grad  # and under no_grad it has none
        with torch.no_grad():
            assert not tda_amd.differential_attention(*xs, lam).requires_grad
        with pytest.raises(ValueError):
            tda_amd.differential_attention(xs[0], xs[1].cpu(), *xs[2:], lam)
        with pytest.raises(ValueError):
            tda_amd.differential_attention(xs[0], xs[1].float(), *xs[2:], lam)
        with pytest.raises(ValueError):
            tda_amd.differential_attention(*xs, lam[:3])


@gpu
@pytest.mark.parametrize("d, dv", DIMS + [(80, 72)])
@pytest.mark.parametrize("h, hk, n, nk, off", [(6, 2, 70, 200, None), (4, 1, 129, 129, None), (3, 3, 300, 1300, 17), (16, 16, 700, 700, None)])
def test_float16_without_gradients(d, dv, h, hk, n, nk, off):
    check(3, h, hk, n, nk, d, dv, F16, torch.linspace(-0.3, 0.9, h), train=False, q_offset=off,
          kv_lens=torch.tensor([nk, nk // 2, 0], dtype=torch.int32).cuda())


@gpu
@pytest.mark.parametrize("d, dv", DIMS)
@pytest.mark.parametrize("h, hk, n, lam", [(2, 2, 1, 0.5), (4, 2, 129, torch.linspace(-0.9, 0.9, 4)), (6, 6, 300, torch.tensor(0.7))])
def test_float16_training_step(d, dv, h, hk, n, lam):
    check(3, h, hk, n, n, d, dv, F16, lam, kv_lens=torch.tensor([n, (n + 1) // 2, 0], dtype=torch.int32).cuda())


@gpu
@pytest.mark.parametrize("by", [2.0 ** -12, 2.0 ** 10])
@pytest.mark.parametrize("lam", [0.5, 300.0])
def test_float16_gradients_keep_their_bits_at_any_scale(by, lam):
    """The same step with upstream gradients scaled by a power of two: the same gradients, scaled, to the bit where
    float16 holds both (the passes' own scales take the power out again); below 2^-14 each is off by up to 2^-25."""
    xs = [x * 0.25 for x in inputs(1, 4, 2, 200, 200, 64, 64, F16)]
    dout = rows((1, 4, 200, 64), 6, F16, 2.0 ** -2 if by > 1 else 1.0)
    dout = torch.where(dout.abs() < 2.0 ** -2, 0.0, dout)  # scaling stays exact
    res = []
    for y in (1.0, by):
        leaves = [x.clone().requires_grad_() for x in xs]
        tda_amd.differential_attention(*leaves, lam).backward(dout * y)
        res.append([x.grad.double() for x in leaves])
    for a, b in zip(*res):
        # (a value just below 2^-14 may round up to it from the coarser steps there)
        held = (b.abs() > 2.0 ** -14) & (a.abs() > 2.0 ** -14) & b.isfinite() & a.isfinite()
        assert torch.equal(a[held] * by, b[held])
        both = b.isfinite() & a.isfinite()
        assert both.any() and ((a * by - b).abs() <= 2.0 ** -25 * (1 + by) + 2.0 ** -11 * b.abs())[both].all()


@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
def test_rows_that_count_for_nothing(dtype):
    """Keys behind every row's sight and rows that see no key take no part in the gradients (nor in float16's
    scales), and get zeros."""
    xs = inputs(2, 2, 2, 40, 60, 64, 64, dtype)
    dout = rows((2, 2, 40, 64), 6, dtype)
    off = torch.tensor([-5, 10]).cuda()  # rows 0 .. 4 of the first sequence see nothing; its last key seen is 34
    res = []
    for bad in (0.0, math.inf):
        ys = [x.clone() for x in xs]
        for x in ys[2:]:
            x[0, :, 35:] = bad
            x[1, :, 50:] = bad
        d = dout.clone()
        d[0, :, :5] *= 1024.0 if bad else 0.0
        ys = [y.requires_grad_() for y in ys]
        tda_amd.differential_attention(*ys, 0.5, q_offset=off).backward(d)
        res.append([y.grad for y in ys])
    assert all(torch.equal(a, b) and b.isfinite().all() for a, b in zip(*res))
    assert not any(g[0, :, 35:].any() or g[1, :, 50:].any() for g in res[1][2:])


def overlapping(x, step):
    """Rows `step` values apart over x's first row (0: that row for every position)."""
    b, h, n, d = x.shape
    flat = torch.cat((x[:, :, 0], rows((b, h, n * step, 1), 77, x.dtype)[..., 0]), -1)
    return flat.as_strided(x.shape, (flat.stride(0), flat.stride(1), step, 1))


@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
@pytest.mark.parametrize("d, dv", DIMS)
@pytest.mark.parametrize("n", [1, 33, 50, 64, 129])
@pytest.mark.parametrize("causal", [True, False])
def test_upstream_gradient_broadcast_along_the_sequence(dtype, d, dv, n, causal):
    """As out.sum(2) or a mean over the sequence hands it down (rows with a stride of 0, or that overlap): the
    gradients of its contiguous copy, to the bit."""
    xs = inputs(2, 4, 2, n, n, d, dv, dtype)

    def step(dout):
        ys = [x.detach().requires_grad_() for x in xs]
        return torch.autograd.grad(tda_amd.differential_attention(*ys, 0.5, causal=causal), ys, dout)

    up = rows((2, 4, n, dv), 6, dtype)
    for dout in (up[:, :, :1].expand(-1, -1, n, -1), overlapping(up, 8)):
        assert all(torch.equal(a, b) for a, b in zip(step(dout), step(dout.contiguous())))


@gpu
def test_mean_over_the_sequence():
    xs = [x.requires_grad_() for x in inputs(2, 4, 2, 50, 50, 64, 64, F32)]
    up = rows((2, 4, 1, 64), 6, F32)
    tda_amd.differential_attention(*xs, 0.5).mean(2).backward(up[:, :, 0])
    ref = oracle.attention(*xs, 0.5, u=U[F32], dout=(up / 50).expand(-1, -1, 50, -1))
    for x, name in zip(xs, ("dq1", "dq2", "dk1", "dk2", "dv")):
        within(x.grad, ref, name, U[F32])


@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
@pytest.mark.parametrize("n, nk", [(1, 300), (50, 50), (129, 200)])
@pytest.mark.parametrize("by", [1.0, 12.0])
@pytest.mark.parametrize("step", [0, 8])
def test_rows_that_overlap(dtype, n, nk, by, step):
    """Every input with rows that are one row, or lie a few values apart; with scores of several hundreds too."""
    xs = inputs(2, 4, 2, n, nk, 64, 128, dtype)
    xs = [overlapping(x * by if k < 2 else x, step) for k, x in enumerate(xs)]
    lens = torch.tensor([nk, nk - 7], dtype=torch.int32).cuda()
    dout = rows((2, 4, n, 128), 6, dtype)

    def run(ys):
        ys = [y.detach().requires_grad_() for y in ys]
        with torch.no_grad():
            plain = tda_amd.differential_attention(*ys, 0.5, kv_lens=lens)
        out = tda_amd.differential_attention(*ys, 0.5, kv_lens=lens)
        return [plain, out.detach(), *torch.autograd.grad(out, ys, dout)]

    got, want = run(xs), run([x.contiguous() for x in xs])
    assert all(g.isfinite().all() and torch.equal(g, w) for g, w in zip(got, want))


def duals(device):
    """Calls of differential_attention in which one argument has a tangent."""
    from torch.autograd import forward_ad
    xs = [torch.randn(1, 2, 5, 64, device=device) for _ in range(5)] + [torch.full((2,), 0.5, device=device)]
    with torch.no_grad():
        if device == "cuda":
            tda_amd.differential_attention(*xs)  # later calls of this signature skip the checks
    for i in range(6):
        with forward_ad.dual_level():
            yield [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(xs)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(device, grad):
    with torch.set_grad_enabled(grad):
        for xs in duals(device):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                tda_amd.differential_attention(*xs)
        q, k, v = xs[0], xs[2], xs[4]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda t: tda_amd.differential_attention(t, q, k, k, v, 0.5), (q,), (q,))


@gpu
@pytest.mark.parametrize("by", [2.0 ** -8, 2.0 ** -12])
def test_float16_gradients_of_rows_of_unequal_size(by):
    """One power of two scales all of a call's score gradients: every other upstream row far smaller than the rest, one
    value row far larger; what float16's smallest values may take of the small rows is in tiny()."""
    xs = inputs(2, 4, 2, 150, 150, 64, 64, F16)
    dout = rows((2, 4, 150, 64), 6, F16)
    dout[:, :, 1::2] *= by
    xs[4][:, :, 5] *= 100
    leaves = [x.requires_grad_() for x in xs]
    tda_amd.differential_attention(*leaves, 0.5).backward(dout)
    ref, more = oracle.attention(*xs, 0.5, u=U[F16], dout=dout), tiny(xs, 0.5, dout)
    for x, name in zip(leaves, ("dq1", "dq2", "dk1", "dk2", "dv")):
        within(x.grad, ref, name, U[F16], 1e-30 + more[name])
