"""Rotary positions of several axes (tda_amd.rotary_axes) against float64, with gradients.

An output is x cos a - y sin a: with the angle's turn reduced in 64 bits, cosine and sine are off by at most
about 3 f (f = 2^-24: their own rounding, and that of the reduced angle, at most pi, to 24 bits, 2 pi
f / 2), the two products and the sum by f each: 6 f (|x| + |y|) and the output's own rounding: u relatively,
and in float16, whose values below 2^-14 stand 2^-24 apart, at least half of that, 2^-25."""
import pytest
import torch

import tda_amd
from oracle import softmax as oracle

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
gpu = pytest.mark.gpu


def setup(b, heads, n, d, rot, sections, dtype, far=0, seq_major=False, seed=0, pos_dtype=torch.int64):
    g = torch.Generator("cpu").manual_seed(seed)
    xs = []
    for h in heads:
        x = torch.randn(b, n, h, d, generator=g).transpose(1, 2)
        xs.append((x if seq_major else x.contiguous()).to(dtype).cuda())
    pos = torch.randint(far, far + 1000, (len(sections), b, n), generator=g).to(pos_dtype).cuda()
    freq = (10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))).float().cuda()
    return xs, pos, freq


def close(got, x, pos, freq, sections, inter, dtype, back=False):
    want = oracle.rotary(x, -pos if back else pos, freq, sections, inter)
    mag = oracle.rotary(x.abs(), pos, freq * 0, sections, inter)
    pairs = freq.shape[0]
    size = mag.clone()
    a, b = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if inter else (slice(0, pairs), slice(pairs, 2 * pairs)))
    size[..., a] = size[..., b] = mag[..., a] + mag[..., b]
    off = U[dtype] * want.abs() + 6 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert got.dtype == dtype and got.shape == x.shape
    assert ((got.double() - want).abs() <= off).all()
    assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])


@gpu
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("b, n, d, rot, sections", [
    (1, 1, 64, 64, (32,)), (2, 5, 128, 128, (16, 24, 24)), (3, 70, 128, 96, (20, 14, 14)), (2, 33, 80, 20, (3, 4, 3)),
    (1, 4100, 64, 64, (0, 32)), (2, 9, 7, 6, (1, 1, 1)), (1, 3, 256, 256, (100, 28, 0, 0)), (2, 2060, 16, 8, (2, 2))])
def test_turns_and_gradients(dtype, inter, b, n, d, rot, sections):
    xs, pos, freq = setup(b, (4, 4, 1, 1), n, d, rot, sections, dtype)
    douts = [x.clone() for x in setup(b, (4, 4, 1, 1), n, d, rot, sections, dtype, seed=1)[0]]
    leaves = [x.clone().requires_grad_(True) for x in xs]
    ys = tda_amd.rotary_axes(leaves, pos, freq, sections, interleaved=inter)
    grads = torch.autograd.grad(ys, leaves, douts)
    for x, y, dy, g in zip(xs, ys, douts, grads):
        close(y, x, pos, freq, sections, inter, dtype)
        close(g, dy, pos, freq, sections, inter, dtype, back=True)


@gpu
@pytest.mark.parametrize("far", [0, 100_000, 100_000_000])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_far_positions(far, pos_dtype):
    xs, pos, freq = setup(2, (3,), 20, 64, 64, (12, 20), torch.float32, far=far, pos_dtype=pos_dtype)
    close(tda_amd.rotary_axes(xs[0], pos, freq, (12, 20)), xs[0], pos, freq, (12, 20), False, torch.float32)
    back = tda_amd.rotary_axes(xs[0], -pos, freq, (12, 20))
    close(back, xs[0], -pos, freq, (12, 20), False, torch.float32)


@gpu
def test_strided_rows_and_positions():
    sections = (16, 8, 8)
    xs, pos, freq = setup(2, (8, 2), 50, 64, 64, sections, torch.bfloat16, seq_major=True)
    want = tda_amd.rotary_axes([x.contiguous() for x in xs], pos, freq, sections)
    got = tda_amd.rotary_axes(xs, pos, freq, sections)
    assert all(torch.equal(a, b) and a.stride() == x.stride() for a, b, x in zip(got, want, xs))
    wide = [torch.cat((x, x), 1)[:, : x.shape[1]] for x in xs]
    assert all(torch.equal(a, b) for a, b in zip(tda_amd.rotary_axes(wide, pos, freq, sections), want))
    odd = [torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x) for x in xs]  # 2-byte aligned
    assert all(torch.equal(a, b) for a, b in zip(tda_amd.rotary_axes(odd, pos, freq, sections), want))
    last = torch.cat((xs[0], xs[0]), -1).contiguous()[..., ::2]
    assert torch.equal(tda_amd.rotary_axes(last, pos, freq, sections),
                       tda_amd.rotary_axes(last.contiguous(), pos, freq, sections))
    one = pos[:1, :1].expand(3, 2, 50)  # every axis and sequence the same: stride 0
    assert torch.equal(tda_amd.rotary_axes(xs[0], one, freq, sections), tda_amd.rotary_axes(xs[0], one.contiguous(), freq, sections))
    assert torch.equal(tda_amd.rotary_axes(xs[0], pos.transpose(1, 2).contiguous().transpose(1, 2), freq, sections), want[0])


@gpu
def test_partial_gradients_empty_and_capture():
    xs, pos, freq = setup(2, (3, 2), 40, 64, 64, (32,), torch.bfloat16)
    leaf = xs[1].clone().requires_grad_(True)
    y = tda_amd.rotary_axes([xs[0], leaf], pos, freq, (32,))
    (y[0].float().sum() + y[1].float().sum()).backward()
    close(leaf.grad, torch.ones_like(leaf), pos, freq, (32,), False, torch.bfloat16, back=True)
    empty = torch.zeros(2, 3, 0, 64, device="cuda")
    assert tda_amd.rotary_axes(empty, pos[:, :, :0], freq, (32,)).shape == empty.shape
    with torch.no_grad():
        tda_amd.rotary_axes(xs, pos, freq, (32,))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = tda_amd.rotary_axes(xs, pos, freq, (32,))
        for k in range(3):
            pos.add_(17)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, tda_amd.rotary_axes(xs, pos, freq, (32,))))


def test_refusals_without_a_gpu():
    x, pos, freq = torch.zeros(1, 2, 3, 64), torch.zeros(1, 1, 3, dtype=torch.int64), torch.ones(32)
    with pytest.raises(ValueError, match="GPU only"):
        tda_amd.rotary_axes(x, pos, freq, (32,))
    with pytest.raises(TypeError):
        tda_amd.rotary_axes([None], pos, freq, (32,))
    with pytest.raises(ValueError):
        tda_amd.rotary_axes([x] * 5, pos, freq, (32,))
    with pytest.raises(ValueError):
        tda_amd.rotary_axes([], pos, freq, (32,))
    with pytest.raises(ValueError):
        tda_amd.rotary_axes([x, x[:, :, :2]], pos, freq, (32,))


@gpu
@pytest.mark.parametrize("change", [
    dict(sections=(31,)), dict(sections=(33, -1)), dict(sections=(8,) * 4 + (0,)), dict(sections=()), dict(freq=torch.ones(33)),
    dict(freq=torch.ones(32, dtype=torch.float64)), dict(freq=torch.ones(32, requires_grad=True)), dict(pos=torch.zeros(1, 1, 3)),
    dict(pos=torch.zeros(1, 1, 4, dtype=torch.int64)), dict(pos=torch.zeros(2, 1, 3, dtype=torch.int64)),
    dict(x=torch.zeros(1, 2, 3, 64, dtype=torch.float64)), dict(x=torch.zeros(2, 3, 64)), dict(cpu=True)])
def test_refusals(change):
    x = change.get("x", torch.zeros(1, 2, 3, 64)).cuda()
    pos = change.get("pos", torch.zeros(1, 1, 3, dtype=torch.int64))
    freq = change.get("freq", torch.ones(32)).cuda()
    if not change.get("cpu"):
        pos = pos.cuda()
    if change.get("freq") is not None and change["freq"].requires_grad:
        freq = freq.detach().requires_grad_(True)
    with pytest.raises(ValueError):
        tda_amd.rotary_axes(x, pos, freq, change.get("sections", (32,)))


@gpu
def test_calls_of_one_signature_take_their_own_tensors():
    for k in range(3):
        g = torch.Generator().manual_seed(k)
        xs = [torch.randn(2, h, 5, 64, generator=g).cuda() for h in (4, 2)]
        pos, freq = torch.randint(0, 99, (1, 2, 5), generator=g).cuda(), torch.rand(32, generator=g).cuda()
        got = tda_amd.rotary_axes(xs, pos, freq, (32,))
        want = tda_amd.rotary_axes(xs, pos.int(), freq, (32,))  # another signature
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(tda_amd.rotary_axes(xs[0], pos, freq, (32,)), got[0])
    xs[0].requires_grad_()
    assert tda_amd.rotary_axes(xs, pos, freq, (32,))[0].requires_grad
    with torch.no_grad():
        assert not tda_amd.rotary_axes(xs, pos, freq, (32,))[0].requires_grad
    with pytest.raises(ValueError):
        tda_amd.rotary_axes([xs[0], xs[1].half()], pos, freq, (32,))
    with pytest.raises(ValueError):
        tda_amd.rotary_axes(xs, pos, freq, (31,))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_is_refused(device):
    from torch.autograd import forward_ad
    x, pos, freq = torch.ones(1, 2, 3, 64, device=device), torch.ones(1, 1, 3, dtype=torch.int64, device=device), torch.ones(32, device=device)
    if device == "cuda":
        tda_amd.rotary_axes([x, x], pos, freq, (32,))  # later calls of this signature skip the checks
    with forward_ad.dual_level():
        y, f = forward_ad.make_dual(x, x), forward_ad.make_dual(freq, freq)
        for xs, by in (([x, y], freq), ([y, x], freq), ([x, x], f), (y, freq)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                tda_amd.rotary_axes(xs, pos, by, (32,))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: tda_amd.rotary_axes(t, pos, freq, (32,)), (x,), (x,))


@gpu
def test_sections_of_any_iterable():
    xs, pos, freq = setup(2, (3,), 5, 64, 64, (16, 8, 8), torch.float32)
    want = tda_amd.rotary_axes(xs[0], pos, freq, (16, 8, 8))
    for sections in ([16, 8, 8], iter((16, 8, 8)), (n for n in (16, 8, 8)), torch.tensor([16, 8, 8])):
        assert torch.equal(tda_amd.rotary_axes(xs[0], pos, freq, sections), want)
