"""Layer norm and RMS norm (tda_amd.layer_norm): refusals on the CPU, and on the GPU every output and gradient against
the definition in float64, within the bounds of oracle/norm.py, which count half a step of the type for each rounding."""
import contextlib
import ctypes
import math

import pytest
import torch

import tda_amd
from oracle import norm as oracle
from tda_amd import _abi, _sln_abi, norm

BF, F32, F16 = torch.bfloat16, torch.float32, torch.float16
U = {BF: 2.0 ** -8, F32: 2.0 ** -24, F16: 2.0 ** -11, torch.float64: 2.0 ** -24}
TINY = {F16: 2.0 ** -25}  # half a step of float16 below 2^-14
gpu = pytest.mark.gpu


def rows(shape, seed, dtype, device="cuda", level=0.7, spread=1.5):
    g = torch.Generator("cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread + level).to(dtype).to(device)


def within(got, ref, name, dtype):
    want, off = ref[name], ref[name + "_off"]
    assert got.shape == want.shape and got.dtype == dtype, name
    assert torch.isfinite(got).all(), name
    far = (got.double() - want).abs() - off - TINY.get(dtype, 1e-38)
    assert far.max().item() <= 0, f"{name}: {far.max().item():.3g} past {off.flatten()[far.argmax()].item():.3g}"


def check(x, weight, bias, dy=None, **kw):
    leaves = [None if t is None else t.detach().requires_grad_(dy is not None) for t in (x, weight, bias)]
    y = tda_amd.layer_norm(*leaves, **kw)
    wdt = next((t.dtype for t in (weight, bias) if t is not None), x.dtype)
    ref = oracle.layer_norm(x, weight, bias, dy=dy, u=U[x.dtype], u_w=U[wdt], **kw)
    within(y, ref, "y", x.dtype)
    if dy is not None:
        y.backward(dy)
        for t, leaf, name in zip((x, weight, bias), leaves, ("dx", "dweight", "dbias")):
            if t is not None:
                within(leaf.grad, ref, name, t.dtype)
    return y


# ------------------------------------------------------------------ widths, types, forms
@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("n, width", [(1, 1), (3, 7), (5, 8), (37, 64), (700, 65), (2, 127), (33, 128), (9, 250), (65, 256), (4, 511),
                                      (19, 513), (7, 1024), (5, 1100), (3, 2047), (6, 2048), (3, 2056), (2, 4096), (5, 4104),
                                      (3, 8191), (2, 8200), (3, 16383), (2, 16384)])
def test_widths(dtype, center, n, width):
    x, dy = rows((n, width), 1, dtype), rows((n, width), 2, dtype, level=0.1)
    check(x, rows((width,), 3, dtype, level=1.0, spread=0.3), rows((width,), 4, dtype), dy, center=center)


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("shape", [(2, 3, 50, 128), (1, 5, 1, 64), (3, 2, 7, 100), (2, 4, 129, 256)])
@pytest.mark.parametrize("heads", [True, False])
@pytest.mark.parametrize("wide", [True, False])
def test_weights_of_heads_and_wide_ones(dtype, shape, heads, wide):
    wshape = (shape[1], shape[3]) if heads else (shape[3],)
    wdt = F32 if wide else dtype
    for seq_major in (False, True):
        x, dy = rows(shape, 1, dtype), rows(shape, 2, dtype)
        if seq_major:
            x, dy = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x, dy))
        y = check(x, rows(wshape, 3, wdt), rows(wshape, 4, wdt), dy)
        assert y.stride() == x.stride()
        check(x, rows(wshape, 3, wdt), None, dy, center=False)
        check(x, None, rows(wshape, 4, wdt), dy)
    check(rows(shape, 1, dtype), None, None, rows(shape, 2, dtype))


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_rows(dtype):
    """More rows than the launch has places for: every loop runs more than once, the last one partly."""
    for shape in ((40011, 64), (20007, 520), (3001, 2500), (1501, 5000), (700, 9000)):
        check(rows(shape, 1, dtype), rows(shape[1:], 2, dtype), rows(shape[1:], 3, dtype), rows(shape, 4, dtype, level=0.1))
    x = rows((3, 5, 4001, 64), 1, dtype)
    check(x, rows((5, 64), 2, dtype), rows((5, 64), 3, dtype), rows(x.shape, 4, dtype))


@gpu
def test_strides():
    """Slices at odd elements, every second row, broadcast gradients, one column, a transposed last axis: results do not
    depend on where rows lie."""
    base = rows((4, 6, 30, 80), 1, BF)
    w, b = rows((6, 37), 2, BF), rows((6, 37), 3, BF)
    x = base[:, :, ::2, 3:40]
    dy = rows((4, 6, 15, 37), 4, BF)
    for view in (x, x.transpose(1, 2).contiguous().transpose(1, 2), base[:, :, ::2].transpose(2, 3).contiguous().transpose(2, 3)[..., 3:40]):
        leaf = view.detach().requires_grad_(True)
        y = tda_amd.layer_norm(leaf, w, b)
        assert torch.equal(y, tda_amd.layer_norm(x.contiguous(), w, b))
        y.backward(dy)
        want = x.contiguous().detach().requires_grad_(True)
        tda_amd.layer_norm(want, w, b).backward(dy)
        assert torch.equal(leaf.grad, want.grad)
    check(x, w, b, rows((4, 6, 1, 1), 5, BF).expand(4, 6, 15, 37))
    check(x, w, b, torch.ones((), dtype=BF, device="cuda").expand(4, 6, 15, 37))
    check(base[..., 5:6], rows((1,), 2, BF), None, base[..., 7:8])
    check(rows((1, 1, 1, 64), 6, BF).expand(3, 5, 7, 64), rows((64,), 7, BF), None, rows((3, 5, 7, 64), 8, BF))


@gpu
def test_shapes():
    w = rows((48,), 1, F32)
    for shape in ((48,), (5, 48), (2, 3, 48), (2, 3, 4, 48), (2, 1, 3, 2, 48)):
        check(rows(shape, 2, F32), w, w, rows(shape, 3, F32))
    x = rows((2, 3, 4, 5, 48), 4, F32).transpose(1, 3)
    assert torch.equal(tda_amd.layer_norm(x, w), tda_amd.layer_norm(x.contiguous(), w))
    for shape in ((0, 48), (2, 0, 48), (2, 3, 0, 48)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        leaf = w.clone().requires_grad_(True)
        y = tda_amd.layer_norm(x, leaf)
        y.sum().backward()
        assert y.shape == shape and x.grad.shape == shape and not leaf.grad.any()


def stepped(n, dtype=F32, device="cpu"):
    """n axes, the last of every second value; and n axes whose last is one value, expanded."""
    return (rows((2, 1, 3, 2, 4, 5)[6 - n + 1:] + (16,), 1, dtype, device)[..., ::2],
            rows((2, 1, 3, 2, 4, 5)[6 - n + 1:] + (1,), 2, dtype, device).expand(*(2, 1, 3, 2, 4, 5)[6 - n + 1:], 8))


@gpu
@pytest.mark.parametrize("dtype", [BF, F32, F16])
@pytest.mark.parametrize("n", [2, 4, 5, 6])
def test_a_last_axis_that_is_no_row(dtype, n):
    """Every second value, and one value for all columns: whatever the number of axes, those are the values that are read
    (axes beyond the fourth merge into a view, which keeps the last axis' stride)."""
    w, b = rows((8,), 3, dtype), rows((8,), 4, dtype)
    for x in stepped(n, dtype, "cuda"):
        assert x.dim() == n and x.stride(-1) != 1
        for dy in (rows(x.shape, 5, dtype), rows((*x.shape[:-1], 16), 6, dtype)[..., ::2], rows((), 7, dtype).expand(x.shape)):
            check(x, w, b, dy)
        check(x, None, None, dy, center=False)
        assert torch.equal(tda_amd.layer_norm(x, w, b), tda_amd.layer_norm(x.contiguous(), w, b))


@pytest.mark.parametrize("n", [2, 3, 4, 5, 6])
def test_rows_for_the_kernels(n):
    """The rows handed on have a unit last stride and hold x's values; a block of rows that do not is refused."""
    for x in (*stepped(n), rows((2, 1, 3, 2, 4, 5)[6 - n + 1:] + (8,), 1, F32, "cpu").transpose(0, 1)):
        r = norm._in_rows(x)
        assert r.dim() <= 4 and r.stride(-1) == 1 and torch.equal(r.reshape(x.shape), x)
    for x in stepped(n):
        flat = x.flatten(0, -2) if n > 4 else x
        a = _sln_abi.SlnFwdArgs.from_buffer_copy(norm._Plan(flat, None, None, 1e-5, True).block)
        a.x.data = a.y.data = 64
        assert a.x.stride[3] == flat.stride(-1) and _sln_abi.load().sln_validate_fwd(ctypes.byref(a)) == _abi.ERR_LAYOUT
    one = rows((2, 1, 3, 2, 4, 5)[6 - n + 1:] + (16,), 1, F32, "cpu")[..., 3:4]
    r = norm._in_rows(one)
    a = _sln_abi.SlnFwdArgs.from_buffer_copy(norm._Plan(r, None, None, 1e-5, True).block)
    assert list(a.x.stride)[-2:] == [16, 1] and r.data_ptr() == one.data_ptr()  # one value a row: read in place


@gpu
def test_values():
    """Rows far from zero keep their variance; constant rows are the bias; a row of one large value; zeros; NaN and
    infinities stay in their row and in the weights' gradients."""
    x = rows((40, 300), 1, F32, level=3000.0, spread=0.5)
    check(x, rows((300,), 2, F32), rows((300,), 3, F32), rows((40, 300), 4, F32))
    b = rows((300,), 3, F32)
    y = tda_amd.layer_norm(torch.full((3, 300), 4.0, device="cuda"), None, b)  # sums of 4 are exact
    assert torch.equal(y, b.expand(3, 300))
    assert not tda_amd.layer_norm(torch.zeros(2, 300, device="cuda"), center=False).any()
    x = torch.zeros(2, 300, device="cuda")
    x[:, 17] = 1e15
    check(x, None, None, rows((2, 300), 5, F32))
    check(x, None, None, rows((2, 300), 5, F32), center=False)
    for bad in (math.nan, math.inf):
        x = rows((9, 2100), 6, F32)
        clean = tda_amd.layer_norm(x)
        x[4, 2099] = bad
        y = tda_amd.layer_norm(x)
        assert y[4].isnan().any() and torch.equal(y[:4], clean[:4]) and torch.equal(y[5:], clean[5:])


@gpu
def test_eps_and_float64():
    x = rows((30, 130), 1, F32, level=0.0, spread=1e-3)
    for eps in (0.0, 1e-12, 1e-5, 1.0):
        check(x, None, None, rows((30, 130), 2, F32), eps=eps)
    x = rows((30, 130), 1, torch.float64)
    y = tda_amd.layer_norm(x, rows((130,), 2, torch.float64))
    assert y.dtype == torch.float64
    assert torch.equal(y, tda_amd.layer_norm(x.float(), rows((130,), 2, F32)).double())


@gpu
def test_gradient_against_differences():
    """The gradient of a sum of outputs times dy, against central differences of the definition in float64."""
    x, w, b, dy = (rows(s, i, F32, device="cpu").double() for i, s in enumerate(((2, 3, 4, 24), (3, 24), (3, 24), (2, 3, 4, 24))))
    leaves = [t.float().cuda().requires_grad_(True) for t in (x, w, b)]
    tda_amd.layer_norm(*leaves).backward(dy.float().cuda())
    loss = lambda *t: (oracle.layer_norm(*t)["y"] * dy).sum().item()  # noqa: E731
    args = [x, w, b]
    for k, leaf in enumerate(leaves):
        for at in range(0, args[k].numel(), 11):
            h = 1e-4
            up, down = (args[k].clone() for _ in range(2))
            up.view(-1)[at] += h
            down.view(-1)[at] -= h
            slope = (loss(*args[:k], up, *args[k + 1:]) - loss(*args[:k], down, *args[k + 1:])) / (2 * h)
            assert abs(leaf.grad.cpu().view(-1)[at].item() - slope) <= 1e-4 * (1 + abs(slope))


# ------------------------------------------------------------------ how it is called
@gpu
def test_partial_gradients_repeat_and_second_derivatives():
    x, w, b, dy = rows((3, 4, 200, 64), 1, BF), rows((4, 64), 2, BF), rows((4, 64), 3, BF), rows((3, 4, 200, 64), 4, BF)
    want = None
    for needs in ((True, True, True), (True, False, False), (False, True, False), (False, False, True), (True, False, True), (True, True, True)):
        leaves = [t.detach().clone().requires_grad_(n) for t, n in zip((x, w, b), needs)]
        tda_amd.layer_norm(*leaves).backward(dy)
        got = [t.grad for t in leaves]
        want = want or got
        for g, v, n in zip(got, want, needs):
            assert torch.equal(g, v) if n else g is None
    leaf = x.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(tda_amd.layer_norm(leaf).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            tda_amd.layer_norm(dual)


@gpu
def test_graphs_and_streams():
    """Captured training steps replayed between eager work, and calls on another stream."""
    x, w, b, dy = rows((2, 4, 300, 128), 1, BF), rows((4, 128), 2, BF), rows((4, 128), 3, BF), rows((2, 4, 300, 128), 4, BF)

    def step(t):
        leaves = [v.detach().requires_grad_(True) for v in (t, w, b)]
        y = tda_amd.layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in range(3):
        new = rows(x.shape, 10 + seed, BF)
        want = step(new)
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))
        torch.randn(1000, 1000, device="cuda").sum().item()
    want = step(x)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@gpu
def test_repeated_calls_look_at_their_arguments():
    """A call that was planned by its signature and one of another kind do not meet."""
    x = rows((4, 96), 1, F32)
    w = rows((96,), 2, F32)
    with torch.no_grad():
        for _ in range(2):
            assert torch.equal(tda_amd.layer_norm(x, w), tda_amd.layer_norm(x.clone(), w.clone()))
            assert not torch.equal(tda_amd.layer_norm(x, w), tda_amd.layer_norm(x, None, w))
            assert not torch.equal(tda_amd.layer_norm(x, w), tda_amd.layer_norm(x, w, center=False))
            assert not torch.equal(tda_amd.layer_norm(x, w), tda_amd.layer_norm(x, w, eps=0.1))
    leaf = w.clone().requires_grad_(True)
    assert tda_amd.layer_norm(x, leaf).requires_grad
    same = torch.nn.Parameter(w.clone())
    assert tda_amd.layer_norm(x, same).grad_fn is not None


def test_backward_block_of_saved_rows():
    """The argument block goes by the strides of the rows that the backward is given."""
    x = rows((4, 30, 6, 80), 1, F32, "cpu").transpose(1, 2)[..., 3:40]
    plan = norm._Plan(x, None, None, 1e-5, True)
    dy, want = torch.empty_strided(plan.shape, plan.strides), (True, False, False)
    for t in (x, x.contiguous(), x):
        key = t.stride(), t.dtype, dy.stride(), want
        block, _ = plan.bwd.get(key) or plan.backward_block(key, t, dy, want)
        assert list(_sln_abi.SlnBwdArgs.from_buffer_copy(block).x.stride) == list(t.stride())


@gpu
@pytest.mark.parametrize("first", ["plain", "moved"])
def test_saved_tensors_that_hooks_move(first):
    """Rows kept on the host (or anywhere) between the passes come back with other strides: the gradients are those of rows
    that stayed, for a call of either kind after the other."""
    w, b = rows((6, 37), 2, BF), rows((6, 37), 3, BF)
    base = rows((4, 30, 6, 80), 1, BF)
    for x in (base.transpose(1, 2)[..., 3:40], base.transpose(1, 2)[:, :, ::2, 5:42], base[0, 0, :, :37]):
        args = (x, w, b) if x.dim() == 4 else (x, w[0], b[0])
        dy = rows(x.shape, 4, BF)
        dy = dy.transpose(1, 2).contiguous().transpose(1, 2) if x.dim() == 4 else dy

        def grads(hooks):
            leaves = [t.detach().requires_grad_(True) for t in args]
            with hooks:
                y = tda_amd.layer_norm(*leaves)
            return torch.autograd.grad(y, leaves, dy)

        moved = lambda: torch.autograd.graph.save_on_cpu()  # noqa: E731
        wide = lambda: torch.autograd.graph.saved_tensors_hooks(  # noqa: E731
            lambda t: t, lambda t: torch.nn.functional.pad(t, (0, 11))[..., :-11] if t.shape == x.shape else t)
        apart = lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack((t, t), -1)[..., 0])  # noqa: E731
        stay = contextlib.nullcontext
        want = None
        for hooks in ([stay, moved, wide, apart, stay] if first == "plain" else [moved, apart, wide, stay, moved]):
            got = grads(hooks())
            want = want or got
            assert all(torch.equal(a, c) for a, c in zip(got, want))


@gpu
def test_memory_of_a_call():
    """A call takes its result and the copy of rows that it cannot read in place, and no more: neither the first of its kind
    nor one that is planned anew each time."""
    size = 2 * 8 * 1024 * 128 * 2

    def taken(x):
        total = lambda: torch.cuda.memory_stats()["allocated_bytes.all.allocated"]  # noqa: E731
        before = total()
        assert tda_amd.layer_norm(x).nbytes == size
        return total() - before

    x = rows((2, 8, 1024, 256), 1, BF)
    whole = x[..., :128].contiguous()
    for _ in range(2):
        assert taken(whole) == size and taken(whole.transpose(1, 2)) == size
        assert taken(x[..., :128]) == size and taken(x[..., ::2]) == 2 * size


@gpu
def test_eps_and_center_held_by_tensors():
    """A tensor whose value changes between two calls is read in each."""
    x = rows((4, 96), 1, F32)
    for device in ("cpu", "cuda"):
        eps, center = torch.tensor(1e-5, dtype=torch.float64, device=device), torch.tensor(True, device=device)
        for e, c in ((1e-5, True), (0.5, True), (0.5, False), (1e-5, False)):
            eps.fill_(e), center.fill_(c)
            for _ in range(2):
                assert torch.equal(tda_amd.layer_norm(x, eps=eps, center=center), tda_amd.layer_norm(x, eps=e, center=c))
        eps.fill_(-1.0)
        with pytest.raises(ValueError, match="eps"):
            tda_amd.layer_norm(x, eps=eps, center=center)


# ------------------------------------------------------------------ refusals
def test_refusals_on_the_cpu():
    x = torch.zeros(2, 3, 4, 8)
    with pytest.raises(ValueError, match="GPU only"):
        tda_amd.layer_norm(x)
    with pytest.raises(TypeError):
        tda_amd.layer_norm([1.0])
    with pytest.raises(ValueError, match="axis"):
        tda_amd.layer_norm(torch.tensor(1.0))


@gpu
def test_refusals():
    x = rows((2, 3, 4, 8), 1, BF)
    w = rows((8,), 2, BF)
    with pytest.raises(ValueError, match="float32, bfloat16"):
        tda_amd.layer_norm(torch.zeros(2, 8, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="last axis"):
        tda_amd.layer_norm(torch.zeros(2, 16385, device="cuda"))
    with pytest.raises(ValueError, match="last axis"):
        tda_amd.layer_norm(torch.zeros(2, 0, device="cuda"))
    for eps in (-1e-5, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            tda_amd.layer_norm(x, eps=eps)
    for bad in (w[:7], rows((4, 8), 3, BF), rows((3, 8, 1), 3, BF)):
        with pytest.raises(ValueError, match="weight must have shape"):
            tda_amd.layer_norm(x, bad)
    with pytest.raises(ValueError, match="weight must have shape"):
        tda_amd.layer_norm(x[0], rows((3, 8), 3, BF))
    with pytest.raises(ValueError, match="weight must be"):
        tda_amd.layer_norm(x, w.half())
    with pytest.raises(ValueError, match="alike"):
        tda_amd.layer_norm(x, w, w.float())
    with pytest.raises(ValueError, match="alike"):
        tda_amd.layer_norm(x, w, rows((3, 8), 3, BF))
    with pytest.raises(ValueError, match="device"):
        tda_amd.layer_norm(x, w.cpu())
    with pytest.raises(TypeError):
        tda_amd.layer_norm(x, 1.0)
