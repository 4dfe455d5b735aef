"""Dropout against its definition: the mask is the published generator's, bit for bit; kept values
are off by their roundings at most."""
import math

import pytest
import torch

import feature_reference as R
import triton_augment_b200 as ta

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _randn(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _expect(x, keep, p, residual=None):
    """Result and bound: x times the rounded 1 / (1 - p) (two roundings) and the sum with the residual
    (one), all in float32, then the type's own rounding."""
    keep = keep.to(x.device)
    scaled = torch.where(keep, x.double() / (1 - p) if p < 1 else torch.zeros_like(x, dtype=torch.float64), torch.zeros((), dtype=torch.float64, device=x.device))
    y = scaled if residual is None else scaled + residual.double()
    tol = R.half_step(x.dtype) * y.abs() * (1 + 4 * R.U) + 3 * R.U * (scaled.abs() + y.abs()) + R.tiny(x.dtype)
    return y, torch.where(keep, tol, torch.zeros_like(tol))               # dropped: exact


def _shared(ndim, mode, same_on_batch, same_on_frame):
    s = {"element": set(), "channel": {ndim - 2, ndim - 1}, "pixel": {ndim - 3}, "sample": {ndim - 3, ndim - 2, ndim - 1}}[mode]
    if same_on_batch and ndim >= 4:
        s.add(0)
    if same_on_frame and ndim == 5:
        s.add(1)
    return s


def _check(x, p, seed, residual=None, order=None, shared=(), **kw):
    got = ta.dropout(x, p, seed, residual=residual, **kw)
    keep = R.dropout_keep(tuple(x.shape), p, seed, kw.get("offset", 0), shared, order)
    y, tol = _expect(x.detach(), keep, p, None if residual is None else residual.detach())
    R.assert_within(got, y, tol, "y")
    assert got.dtype == x.dtype
    return got, keep.to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.25, 0.5, 0.9, 1.0])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (1, 197, 768), (2, 3, 5, 7), (4097,)])
def test_element_masks(shape, p, dtype):
    _check(_randn(shape, dtype), p, 1234567890123456789)


@pytest.mark.parametrize("seed", [0, -1, 2 ** 63, 2 ** 64 - 1, 1 << 32])
def test_seeds_and_offsets(seed):
    x = _randn((999,), torch.float32)
    for offset in (0, 1, 2 ** 32 - 1):
        _check(x, 0.3, seed, offset=offset)


def test_threshold_refinement():
    """p of one, one and a half and two steps of 2^-16, and of 2^-32: the lower halves decide where the
    upper ones are equal - about 32 of these 2^21 entries sit there."""
    x = torch.ones(1 << 21, device=DEV)
    for p in (2.0 ** -16, 1.5 * 2.0 ** -16, 0.25 + 3 * 2.0 ** -20, 2.0 ** -32, 1 - 2.0 ** -32):
        _check(x, p, 77)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("same_on_batch, same_on_frame", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("mode", ["element", "channel", "pixel", "sample"])
@pytest.mark.parametrize("shape", [(6, 5, 7), (3, 16, 8, 8), (3, 5, 7, 9), (2, 3, 8, 4, 16), (2, 3, 5, 7, 3), (1, 2, 1, 1, 1), (9, 1, 24, 1, 8)])
def test_shared_masks(shape, mode, same_on_batch, same_on_frame, dtype):
    shared = _shared(len(shape), mode, same_on_batch, same_on_frame)
    x = _randn(shape, dtype)
    kw = dict(mode=mode, same_on_batch=same_on_batch, same_on_frame=same_on_frame)
    _check(x, 0.4, 5, shared=shared, **kw)
    nd = len(shape)
    order = list(range(nd - 3)) + [nd - 2, nd - 1, nd - 3]
    last = x.movedim(-3, -1).contiguous().movedim(-1, -3)
    if not last.is_contiguous():
        got, _ = _check(last, 0.4, 5, residual=x, shared=shared, order=order, **kw)
        assert got.movedim(-3, -1).is_contiguous()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("same_on_batch, same_on_frame", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("shape, mode, last", [
    ((2, 3, 64, 70), "channel", True), ((3, 33, 40, 41), "channel", True), ((2, 2, 63, 67), "channel", True), ((2, 256, 5, 7), "channel", True),
    ((2, 4096, 1, 2), "channel", True), ((2, 4097, 1, 2), "channel", True), ((3, 2047, 1, 5), "channel", True), ((2, 3, 5, 50, 60), "channel", True),
    ((2, 1, 1, 4096), "channel", True), ((3, 31, 17, 16), "pixel", False), ((2, 6, 3, 30, 31), "pixel", False), ((2, 9, 5, 11, 19), "element", False),
    ((3, 4, 9, 17, 15), "element", True)])
def test_masks_that_repeat(shape, mode, last, same_on_batch, same_on_frame, dtype):
    """A row of entries shared by the rows above it: short and long rows, planes that end inside a vector and inside a block."""
    shared = _shared(len(shape), mode, same_on_batch, same_on_frame)
    x, nd = _randn(shape, dtype), len(shape)
    r = _randn(shape, dtype, 1)
    order = list(range(nd - 3)) + [nd - 2, nd - 1, nd - 3] if last else None
    if last:
        x = x.movedim(-3, -1).contiguous().movedim(-1, -3)
        if x.is_contiguous():
            order = None
    for residual in (None, r):
        _check(x, 0.4, 5, residual=residual, shared=shared, order=order, mode=mode, same_on_batch=same_on_batch, same_on_frame=same_on_frame)
    assert not bool(ta.dropout(x, 1.0, 5, mode=mode, same_on_batch=same_on_batch, same_on_frame=same_on_frame).any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mode", ["element", "channel"])
def test_gradients(mode, dtype):
    """dx = keep dy / (1 - p), the residual's gradient is dy itself."""
    shape = (2, 6, 9, 5)
    x, r = (_randn(shape, dtype, s).requires_grad_() for s in (1, 2))
    y, keep = _check(x, 0.2, 42, residual=r, mode=mode, shared=_shared(4, mode, False, False))
    dy = _randn(shape, dtype, 3)
    dx, dr = torch.autograd.grad(y, (x, r), dy)
    want, tol = _expect(dy, keep, 0.2)
    R.assert_within(dx, want, tol, "dx")
    assert torch.equal(dr, dy)
    # linear in x and in the residual: a difference of two calls is the gradient's product
    if dtype == torch.float32:
        d = _randn(shape, dtype, 4)
        num = (ta.dropout((x + d).detach(), 0.2, 42, mode=mode).double() - ta.dropout(x.detach(), 0.2, 42, mode=mode).double()).mul(dy.double()).sum()
        ana = (dx.double() * d.double()).sum()
        assert abs(float(num - ana)) <= 8 * R.U * float((dy.abs() * (x.detach().abs() + d.abs())).double().sum()) / 0.8
    expanded = torch.autograd.grad(ta.dropout(x, 0.2, 42, mode=mode).sum(), x)[0]
    want, tol = _expect(torch.ones_like(x), keep, 0.2)
    R.assert_within(expanded, want, tol, "expanded dy")


def test_dropped_values_contribute_nothing():
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.full((4096,), bad, device=DEV)
        keep = R.dropout_keep((4096,), 0.5, 9).to(DEV)
        got = ta.dropout(x, 0.5, 9, residual=torch.ones_like(x))
        assert torch.equal(got[~keep], torch.ones_like(got[~keep])) and not bool(torch.isfinite(got[keep]).any())
        assert not bool(ta.dropout(x, 1.0, 9).any())


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Unaligned storage, strided and expanded input, residual in another layout, empty tensors."""
    flat = _randn((4100,), dtype)
    _check(flat[1:4098], 0.3, 8)
    _check(flat[3:4099], 0.3, 8, residual=flat[1:4097])
    _check(flat[:4096].view(64, 64).t(), 0.3, 8)
    _check(flat[:5].expand(7, 5), 0.3, 8)
    x = _randn((2, 6, 4, 4), dtype)
    last = x.contiguous(memory_format=torch.channels_last)
    a = ta.dropout(last, 0.3, 8, residual=x)
    assert torch.equal(a, ta.dropout(last, 0.3, 8, residual=last)) and a.is_contiguous(memory_format=torch.channels_last)
    assert ta.dropout(x[:0], 0.3, 8).shape == (0, 6, 4, 4)
    e = torch.empty(0, 3, device=DEV, requires_grad=True)
    assert torch.autograd.grad(ta.dropout(e, 0.3, 8).sum(), e)[0].shape == (0, 3)


def test_entries_beyond_32_bits():
    """A mask of more than 2^32 entries: the last values of a half-precision tensor of 2^32 + 16 elements."""
    n = 2 ** 32 + 16
    x = torch.ones(n, dtype=torch.float16, device=DEV)
    got = ta.dropout(x, 0.5, 3)
    for first in (0, 2 ** 31 - 8, 2 ** 32 - 8):
        keep = torch.from_numpy(R.mask_numbers(24, 3, first=first) >= 2 ** 31).to(DEV)
        assert torch.equal(got[first:first + 24] != 0, keep)
    del x, got
    torch.cuda.empty_cache()


def test_shared_masks_beyond_32_bits():
    """Two samples of 2^31 + 8 halves under one mask, and a mask entry per sample: the general index arithmetic in 64 bits."""
    plane = 2 ** 31 + 8
    x = torch.ones(2, 1, 1, plane, dtype=torch.float16, device=DEV)
    got = ta.dropout(x, 0.5, 3, same_on_batch=True)
    for first in (0, plane - 24):
        keep = torch.from_numpy(R.mask_numbers(24, 3, first=first) >= 2 ** 31).to(DEV)
        for n in (0, 1):
            assert torch.equal(got[n, 0, 0, first:first + 24] != 0, keep)
    del got
    got = ta.dropout(x, 0.5, 3, mode="sample")
    keep = R.mask_numbers(2, 3) >= 2 ** 31
    for n in (0, 1):
        assert bool((got[n, 0, 0, ::65537] != 0).all()) == bool(keep[n]) and bool((got[n, 0, 0, -9:] != 0).any()) == bool(keep[n])
    del x, got
    torch.cuda.empty_cache()


def test_rows_next_to_the_32_bit_limit():
    """The row kernel hands over to the general one before an index of its last block could wrap."""
    for numel in (2 ** 32 - 2 ** 15, 2 ** 32 - 8):
        x = torch.ones(1, 1, 2, numel // 2, dtype=torch.float16, device=DEV).permute(0, 2, 1, 3).contiguous()        # two channels
        got = ta.dropout(x, 0.5, 7, mode="channel")
        keep = R.mask_numbers(2, 7) >= 2 ** 31
        for c in (0, 1):
            assert bool((got[0, c, 0, ::65537] != 0).all()) == bool(keep[c]) and bool((got[0, c, 0, -4097:] != 0).any()) == bool(keep[c])
        del x, got
    torch.cuda.empty_cache()


def test_seed_tensor_and_generator():
    x = _randn((5000,), torch.float32)
    seed = torch.tensor([987654321987654321], device=DEV)
    assert torch.equal(ta.dropout(x, 0.3, seed), ta.dropout(x, 0.3, 987654321987654321))
    torch.manual_seed(5)
    a, b = ta.dropout(x, 0.3), ta.dropout(x, 0.3)
    torch.manual_seed(5)
    c = ta.dropout(x, 0.3)
    assert torch.equal(a, c) and not torch.equal(a, b)
    leaf = x.clone().requires_grad_()
    y = ta.dropout(leaf, 0.3)                       # the backward pass sees the seed of the forward pass
    g, = torch.autograd.grad(y.sum(), leaf)
    assert torch.equal(g != 0, y.detach() != 0)
    y = ta.dropout(leaf, 0.3, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_captured_replays_draw_anew_and_match_their_gradients():
    drop = ta.TritonDropout(0.4)
    x = _randn((64, 100), torch.float32).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(drop(x).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(x)
        g, = torch.autograd.grad(y, x, torch.ones_like(y))
    masks = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        masks.append(y.detach().clone() != 0)
        assert torch.equal(masks[-1], g != 0)
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])
    # a seed tensor the caller refills
    seed = torch.zeros(1, dtype=torch.int64, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = ta.dropout(x, 0.4, seed)
    for s in (3, 4):
        seed.fill_(s)
        graph.replay()
        assert torch.equal(out, ta.dropout(x.detach(), 0.4, s))
    same = ta.GraphedTransform(ta.TritonDropout(0.4, mode="channel"), _randn((4, 16, 8, 8), torch.float16))
    a = same().clone()
    assert not torch.equal(a, same())


def test_class_and_sharing():
    drop = ta.TritonDropout(0.5, mode="pixel")                  # same_on_frame by default, as in the transforms
    x = torch.ones(2, 4, 3, 16, 16, device=DEV)
    y = drop(x)
    assert torch.equal(y, y[:, :1, :1].expand_as(y)) and not torch.equal(y[0], y[1])
    r = torch.full_like(x, 2.0)
    assert torch.equal(drop.eval()(x, r), x + r) and drop(x) is x
    both = ta.TritonDropout(0.5, same_on_batch=True)(x)
    assert torch.equal(both[0], both[1]) and math.isclose(float((both != 0).float().mean()), 0.5, abs_tol=0.1)
    assert ta.TritonDropout(0.5)(torch.ones(8, 8, device=DEV)).shape == (8, 8)
