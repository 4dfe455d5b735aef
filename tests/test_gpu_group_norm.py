"""Group norm with an activation against its definition in 64 bits; every bound is the one
feature_reference derives from roundings, none was fitted."""
import ctypes as C

import pytest
import torch

import feature_reference as R
import triton_augment_b200 as ta
from triton_augment_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _features(shape, dtype, seed=0, mean=0.0, channels_last=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    last = shape[:-3] + shape[-2:] + shape[-3:-2]
    x = (torch.randn(last, generator=g, device=DEV) * (0.5 + torch.rand(shape[-3], generator=g, device=DEV))
         + mean + torch.randn(shape[-3], generator=g, device=DEV)).to(dtype).movedim(-1, -3)
    return x if channels_last else x.contiguous()


def _params(c, dtype, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return ((1 + 0.3 * torch.randn(c, generator=g, device=DEV)).to(dtype), (0.3 * torch.randn(c, generator=g, device=DEV)).to(dtype))


def _check(x, groups, weight, bias, act, eps=1e-5, same_on_frame=False, dy=None):
    want = R.group_norm(x.detach(), groups, None if weight is None else weight.detach(), None if bias is None else bias.detach(),
                        eps, act, same_on_frame, dy)
    got = ta.group_norm(x, groups, weight, bias, eps, act, same_on_frame=same_on_frame)
    assert got.dtype == x.dtype and got.movedim(-3, -1).is_contiguous()
    R.assert_within(got, want["y"], want["y_tol"], "y")
    if dy is not None:
        leaves = [("dx", x), ("dweight", weight), ("dbias", bias)]
        leaves = [(n, t) for n, t in leaves if t is not None and t.requires_grad]
        for (name, leaf), grad in zip(leaves, torch.autograd.grad(got, [t for _, t in leaves], dy)):
            assert grad.dtype == leaf.dtype
            R.assert_within(grad, want[name], want[name + "_tol"], name)
    return got


# one pixel to many, odd planes, groups of one channel to all, channel counts of every vector width
SHAPES = [((1, 8, 1, 1), 2), ((1, 64, 14, 14), 8), ((3, 320, 9, 7), 32), ((2, 30, 17, 5), 6), ((2, 33, 5, 6), 11), ((5, 7, 3, 3), 7),
          ((2, 36, 31, 2), 4), ((1, 16, 1, 257), 1), ((2, 1, 40, 40), 1), ((1, 2056, 3, 3), 8), ((4, 512, 1, 1), 32), ((2, 96, 65, 67), 12),
          ((1, 130, 64, 48), 10), ((70, 16, 5, 5), 4), ((2, 40, 128, 130), 4), ((3, 320, 14, 14), 32), ((2, 640, 14, 13), 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, groups", SHAPES)
def test_forward_and_gradients(shape, groups, dtype):
    act = ("none", "silu", "gelu", "relu")[(shape[1] + groups) % 3 if shape != (2, 30, 17, 5) else 0]
    x = _features(shape, dtype).requires_grad_()
    w, b = (t.requires_grad_() for t in _params(shape[1], torch.float32))
    _check(x, groups, w, b, act, dy=_features(shape, dtype, 7))


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("param", TYPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_activations_and_parameter_types(act, param, dtype):
    x = _features((2, 48, 13, 11), dtype, 3)
    w, b = _params(48, param)
    dy = _features((2, 48, 13, 11), dtype, 4)
    if act == "relu":
        # the slope jumps at zero: keep away from it by more than the arithmetic can err
        z = R.group_norm(x, 6, w, b, 1e-5, "none")
        dy = torch.where(z["y"].abs() > 4 * z["y_tol"], dy, torch.zeros_like(dy))
    _check(x.requires_grad_(), 6, w.requires_grad_(), b.requires_grad_(), act, dy=dy)


@pytest.mark.parametrize("weight, bias", [(True, False), (False, True), (False, False)])
def test_missing_parameters_and_partial_gradients(weight, bias):
    w, b = _params(24, torch.float32)
    x = _features((2, 24, 9, 9), torch.float32)
    dy = _features((2, 24, 9, 9), torch.float32, 5)
    _check(x.clone().requires_grad_(), 4, w if weight else None, b if bias else None, "silu", dy=dy)       # only x
    if weight or bias:
        _check(x, 4, w.requires_grad_() if weight else None, b.requires_grad_() if bias else None, "silu", dy=dy)   # only parameters


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shared", [False, True])
def test_clips(shared, dtype):
    x = _features((2, 5, 40, 7, 9), dtype).requires_grad_()
    w, b = (t.requires_grad_() for t in _params(40, dtype))
    _check(x, 4, w, b, "silu", same_on_frame=shared, dy=_features((2, 5, 40, 7, 9), dtype, 3))
    one = _check(x[0, 0], 4, w, b, "none")
    assert one.shape == (40, 7, 9)


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Row-major input, strided channels, a sliced plane, an expanded gradient, odd storage offsets."""
    w, b = _params(32, torch.float32)
    x = _features((2, 32, 6, 10), dtype)
    want = ta.group_norm(x, 4, w, b, activation="silu")
    assert torch.equal(ta.group_norm(x.contiguous(), 4, w, b, activation="silu"), want)
    assert want.is_contiguous(memory_format=torch.channels_last)
    wide = _features((2, 64, 8, 12), dtype, 2)
    cut = wide[:, 3:35, 1:7, 2:]
    _check(cut.detach().requires_grad_(), 4, w, b, "silu", dy=torch.ones((), dtype=dtype, device=DEV).expand(cut.shape))
    flat = torch.empty(x.numel() + 1, dtype=dtype, device=DEV)               # rows off every vector boundary
    odd = flat[1:].view(2, 6, 10, 32).permute(0, 3, 1, 2)
    odd.copy_(x)
    _check(odd.requires_grad_(), 4, w, b, "silu", dy=x)


def test_large_mean_keeps_its_digits():
    """A mean of 1000 spreads: the deviations, not the squares' difference, make the variance."""
    for shape in ((2, 32, 24, 24), (1, 8, 300, 300)):
        x = _features(shape, torch.float32, mean=1000.0).requires_grad_()
        w, b = _params(shape[1], torch.float32)
        _check(x, 8, w, b, "none", dy=_features(shape, torch.float32, 6))


def test_constant_groups_and_eps():
    x = torch.full((2, 8, 5, 5), 3.25, device=DEV)
    w, b = _params(8, torch.float32)
    assert torch.equal(ta.group_norm(x, 2, w, b), b.view(1, 8, 1, 1).expand_as(x))
    x = _features((2, 8, 5, 5), torch.float32)
    _check(x, 2, w, b, "none", eps=0.5)
    assert bool(torch.isnan(ta.group_norm(torch.full_like(x, 3.25), 2, w, b, eps=0.0)).all())            # 0 / 0


def test_nan_and_infinity_stay_in_their_group():
    x = _features((2, 8, 6, 6), torch.float32)
    clean = ta.group_norm(x, 2, activation="silu")
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[0, 1, 2, 3] = bad
        got = ta.group_norm(y, 2, activation="silu")
        assert bool(torch.isnan(got[0, :4]).all()) and torch.equal(got[1], clean[1]) and torch.equal(got[0, 4:], clean[0, 4:])


@pytest.mark.parametrize("shape", [(0, 8, 4, 4), (2, 8, 0, 4)])
def test_empty(shape):
    x = torch.empty(shape, device=DEV, requires_grad=True)
    w, b = (t.requires_grad_() for t in _params(8, torch.float32))
    y = ta.group_norm(x, 2, w, b)
    assert y.shape == shape
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert gx.shape == shape and not gw.any() and not gb.any()


def test_gradient_against_differences():
    """Directional central differences of the 64-bit definition: step 1e-4, error of order step^2 and
    of the float32 gradient, both far below the 1e-3 asked for."""
    x = _features((2, 24, 7, 5), torch.float32).requires_grad_()
    w, b = (t.requires_grad_() for t in _params(24, torch.float32))
    dy = _features((2, 24, 7, 5), torch.float32, 9)
    grads = torch.autograd.grad(ta.group_norm(x, 4, w, b, activation="gelu"), (x, w, b), dy)
    g = torch.Generator(device=DEV).manual_seed(11)
    f = lambda *t: float((R.group_norm(t[0], 4, t[1], t[2], 1e-5, "gelu")["y"] * dy.double()).sum())
    for i in range(3):
        base = [t.detach().double() for t in (x, w, b)]
        d = torch.randn(base[i].shape, generator=g, device=DEV, dtype=torch.float64)
        up, down = [list(base) for _ in range(2)]
        up[i], down[i] = base[i] + 1e-4 * d, base[i] - 1e-4 * d
        num, ana = (f(*up) - f(*down)) / 2e-4, float((grads[i].double() * d).sum())
        assert abs(num - ana) <= 1e-3 * (float((grads[i].double().abs() * d.abs()).sum()) + 1e-9), (i, num, ana)


def test_results_repeat_bit_for_bit_and_on_another_stream():
    x = _features((6, 64, 33, 31), torch.bfloat16).requires_grad_()
    w, b = (t.requires_grad_() for t in _params(64, torch.float32))
    dy = _features((6, 64, 33, 31), torch.bfloat16, 2)

    def once():
        y = ta.group_norm(x, 8, w, b, activation="silu")
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            again = once()
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_captured_and_replayed_with_new_data():
    """Forward and backward in one graph; two graphs replayed in turn do not share scratch."""
    def build(shape, groups):
        x = _features(shape, torch.float16).requires_grad_()
        w, b = (t.requires_grad_() for t in _params(shape[1], torch.float32))
        dy = _features(shape, torch.float16, 2)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(ta.group_norm(x, groups, w, b, activation="silu"), (x, w, b), dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ta.group_norm(x, groups, w, b, activation="silu")
            outs = (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))
        return graph, x, w, b, dy, outs
    built = [build((2, 64, 40, 40), 8), build((3, 33, 21, 20), 11), build((1, 128, 200, 200), 32)]     # clusters, odd channels, two launches
    for seed in (21, 22):
        for graph, x, w, b, dy, outs in built:
            with torch.no_grad():
                x.copy_(_features(x.shape, x.dtype, seed))
            graph.replay()
        torch.cuda.synchronize()
        for (graph, x, w, b, dy, outs), groups in zip(built, (8, 11, 32)):
            want = R.group_norm(x.detach(), groups, w.detach(), b.detach(), 1e-5, "silu", dy=dy)
            for got, name in zip(outs, ("y", "dx", "dweight", "dbias")):
                R.assert_within(got, want[name], want[name + "_tol"], name)


@pytest.mark.parametrize("shape, groups", [((2, 40, 9, 9), 5), ((1, 40, 300, 200), 5)])
def test_parameters_off_vector_boundaries(shape, groups):
    """float32 weights that start in the middle of a vector, gradients included; 16-bit ones at odd elements."""
    for dtype in TYPES:
        pool = torch.randn(2, 41, device=DEV).to(dtype)
        w, b = (pool[i, 1:].detach().requires_grad_() for i in (0, 1))
        assert w.data_ptr() % 16 != 0
        _check(_features(shape, torch.bfloat16).requires_grad_(), groups, w, b, "silu", dy=_features(shape, torch.bfloat16, 4))


@pytest.mark.parametrize("side, rows, chain", [(30, 300, 20), (260, 133, 15)])
def test_outliers_in_the_first_pixels(side, rows, chain):
    """The eight pixels that a block takes its pivot from are d = 1000 spreads off.  Its `rows` rows add up to
    rows d^2 where the deviations are 8 d^2, in chains of `chain` additions, each off by u: the squares' sum is off by
    (chain + 3) u, the square of the sum by twice that, together 3 (chain + 3) rows / 8 u of the variance and half of it in
    rstd; the mean by chain u d rows / side^2.  One cluster block of three, and one chunk of 512."""
    x = _features((2, 32, side, side), torch.float32)[:2 if side == 30 else 1].contiguous(memory_format=torch.channels_last)
    x[:, :, 0, :8] = 1000.0
    w, b = _params(32, torch.float32)
    y = ta.group_norm(x, 8, w, b)
    want = R.group_norm(x, 8, w, b, 1e-5, "none")
    total = side * side
    spread = 1000.0 * (8 / total) ** 0.5                              # of the whole sample, to a per cent
    xhat = ((want["y"] - b.double()[:, None, None]) / w.double()[:, None, None]).abs()
    extra = R.U * (1.02 * 1.5 * (chain + 3) * rows / 8 * xhat + 1.02 * chain * 1000.0 / spread * rows / total)
    R.assert_within(y, want["y"], want["y_tol"] + extra * w.double().abs()[:, None, None], "y")


def test_two_streams_at_once():
    """Calls that overlap on the GPU share nothing: each gives the bits it gives alone."""
    xs = [_features((4, 64, 64, 64), torch.bfloat16, s).requires_grad_() for s in (1, 2)]
    dy = _features((4, 64, 64, 64), torch.bfloat16, 5)
    alone = []
    for x in xs:
        y = ta.group_norm(x, 8, activation="silu")
        alone.append((y.detach(), torch.autograd.grad(y, x, dy)[0]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                y = ta.group_norm(x, 8, activation="silu")
                got.append((y.detach(), torch.autograd.grad(y, x, dy)[0]))
        torch.cuda.synchronize()
        for a, g in zip(alone, got):
            assert torch.equal(a[0], g[0]) and torch.equal(a[1], g[1])


def test_class_double_backward_and_scratch():
    gn = ta.TritonGroupNorm(4, 32, activation="silu").to(DEV)
    x = _features((2, 32, 8, 8), torch.bfloat16).requires_grad_()
    y = gn(x)
    y.float().sum().backward()
    assert gn.weight.grad.shape == (32,) and x.grad.shape == x.shape
    gx, = torch.autograd.grad(gn(x).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.float().sum().backward()
    # the C entry refuses scratch that is too small instead of writing behind it
    xs = torch.rand(1, 200 * 200, 33, device=DEV)
    stats, out = torch.empty(2, 3, device=DEV), torch.empty_like(xs)
    p = _lib.GroupNormParams()
    p.struct_size, p.n, p.rows, p.channels, p.groups, p.eps = C.sizeof(p), 1, 200 * 200, 33, 3, 1e-5
    p.x, p.y, p.mean, p.rstd = xs.data_ptr(), out.data_ptr(), stats.data_ptr(), stats.data_ptr() + 12
    need = _lib.load().ta_b200_group_norm_scratch_bytes(C.byref(p), 0)
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    p.scratch, p.scratch_bytes = scratch.data_ptr(), need - 1
    if need:
        assert _lib.load().ta_b200_group_norm(C.byref(p), None) == -6
    with pytest.raises(ValueError, match="must be on"):
        ta.group_norm(xs.view(1, 200, 200, 33).movedim(-1, 1), 3, torch.ones(33))
