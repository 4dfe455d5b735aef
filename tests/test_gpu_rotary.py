"""Rotary positions with one to three axes against the definition in 64 bits."""
import pytest
import torch

import feature_reference as R
import triton_augment_b200 as ta

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _randn(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _check(q, k, angles, sections, pairing="interleaved", spectrum="axis", prefix=0, grads=True, **kw):
    q, k = q.detach(), None if k is None else k.detach()
    if grads:
        q.requires_grad_()
        k = None if k is None else k.requires_grad_()
    out = ta.rotary_embedding(q, k, sections=sections, pairing=pairing, spectrum=spectrum, prefix=prefix, **kw)
    outs = [out] if k is None else list(out)
    ins = [q] if k is None else [q, k]
    for got, x in zip(outs, ins):
        assert got.dtype == x.dtype
        R.assert_within(got, *R.rotary(x.detach(), angles, sections, pairing, prefix), "forward")
    if grads:
        dys = [_randn(t.shape, t.dtype, 50 + i) for i, t in enumerate(ins)]
        for g, dy in zip(torch.autograd.grad(outs, ins, dys), dys):
            R.assert_within(g, *R.rotary(dy, angles, sections, pairing, prefix, inverse=True), "gradient")
    return outs


# every vector width, sections that end inside a vector, lone elements, empty sections
CASES = [((14, 14), (32, 32), 64, 4, 4, 0), ((2, 3, 5), (16, 24, 24), 64, 3, 1, 0), ((7,), (128,), 128, 2, 2, 0), ((3, 4), (20, 16), 37, 2, 1, 2),
         ((2, 2, 2), (4, 6, 2), 14, 5, 0, 1), ((1, 1, 1), (32, 48, 48), 128, 16, 4, 0), ((5, 3), (0, 6), 6, 1, 1, 4), ((4,), (2,), 3, 1, 0, 0),
         ((9, 5), (32, 36), 72, 6, 2, 1), ((3, 3), (256, 256), 520, 2, 1, 0), ((2, 2), (0, 0), 8, 2, 2, 0), ((8, 6), (40, 40), 96, 32, 8, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("spectrum", ["axis", "joint"])
@pytest.mark.parametrize("grid, sections, dim, heads, kv, prefix", CASES)
def test_grids(grid, sections, dim, heads, kv, prefix, spectrum, pairing, dtype):
    n, length = 3, int(torch.Size(grid).numel()) + prefix
    q = _randn((n, length, heads, dim), dtype)
    k = _randn((n, length, kv, dim), dtype, 1) if kv else None
    angles = R.rotary_angles(R.grid_positions(grid, 1, device=DEV), sections, spectrum=spectrum)
    outs = _check(q, k, angles, sections, pairing, spectrum, prefix, grid=grid)
    assert torch.equal(outs[0][:, :prefix], q[:, :prefix]) and torch.equal(outs[0][..., sum(sections):], q[..., sum(sections):])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pos", [torch.int64, torch.int32, torch.float32])
@pytest.mark.parametrize("per_sample", [True, False])
def test_position_tensors(per_sample, pos, dtype):
    n, length, sections = 4, 11, (16, 24, 24)
    g = torch.Generator(device=DEV).manual_seed(2)
    shape = (n, length, 3) if per_sample else (length, 3)
    p = (torch.randint(-40000, 40000, shape, generator=g, device=DEV).to(pos) if pos != torch.float32
         else torch.rand(shape, generator=g, device=DEV) * 5000 - 1000)
    angles = R.rotary_angles((p if per_sample else p[None]).double(), sections)
    q, k = _randn((n, length, 8, 64), dtype), _randn((n, length, 2, 64), dtype, 1)
    _check(q, k, angles, sections, positions=p)
    strided = torch.stack((p, p), -1)[..., 0]                              # every second element
    _check(q, k, angles, sections, "halves", positions=strided)
    prefixed = R.rotary_angles((p if per_sample else p[None]).double()[:, 3:], sections)
    _check(q, k, prefixed, sections, prefix=3, positions=p)


def test_far_positions_lose_no_digits():
    """Up to 2^24, where a float32 product would be off by whole turns; beyond it two floats carry the position."""
    p = torch.tensor([[0], [1], [4095], [100003], [2 ** 24 - 1], [2 ** 24 + 1], [-(2 ** 24) + 3], [2 ** 27 + 12345]], device=DEV)
    q = _randn((1, 8, 2, 64), torch.float32)
    angles = R.rotary_angles(p.double()[None], (64,))
    # the last position: the frequency's 48 bits leave 2^27 / 2 pi 2^-48 turns, 6e-7 of an angle: 10 more u
    got = ta.rotary_embedding(q, sections=(64,), positions=p)
    want, tol = R.rotary(q, angles, (64,), "interleaved")
    tol[:, -1] *= 2
    R.assert_within(got, want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("grid, sections", [((5, 7), (16, 16)), ((3, 5, 7), (8, 12, 12)), ((6,), (32,))])
def test_windows(grid, sections, dtype):
    """Crop offsets and flips: tensors, numbers, fractional offsets, and the same patches of the whole image."""
    n, cells = 5, int(torch.Size(grid).numel())
    q, k = _randn((n, cells, 2, 32), dtype), _randn((n, cells, 1, 32), dtype, 1)
    g = torch.Generator(device=DEV).manual_seed(4)
    left = torch.rand(n, generator=g, device=DEV) * 700
    flip = torch.tensor([True, False, True, True, False], device=DEV)
    kw, ref = dict(left=left, flip_horizontal=flip), dict(left=left, flip=flip)
    if len(grid) > 1:
        kw["top"] = ref["top"] = torch.randint(0, 900, (n,), generator=g, device=DEV)
    angles = R.rotary_angles(R.grid_positions(grid, n, 14.0, device=DEV, **ref), sections)
    _check(q, k, angles, sections, grid=grid, patch=14, **kw)
    angles = R.rotary_angles(R.grid_positions(grid, n, 16.0, left=33, device=DEV, flip=True), sections)
    _check(q, None, angles, sections, "halves", grid=grid, patch=16, left=33, flip_horizontal=True)


def test_crop_keeps_its_places():
    """Patches of a crop at whole-patch offsets get exactly the rotation they have in the whole image."""
    whole = _randn((1, 64, 4, 32), torch.float32).expand(2, 64, 4, 32)
    full = ta.rotary_embedding(whole, sections=(16, 16), grid=(8, 8), patch=16).view(2, 8, 8, 4, 32)
    part = whole.reshape(2, 8, 8, 4, 32)[:, 2:5, 3:7]
    got = ta.rotary_embedding(part.reshape(2, 12, 4, 32), sections=(16, 16), grid=(3, 4), patch=16, top=32, left=48)
    assert torch.equal(got.view(2, 3, 4, 4, 32), full[:, 2:5, 3:7])
    mirrored = part.flip(2).reshape(2, 12, 4, 32)
    got = ta.rotary_embedding(mirrored, sections=(16, 16), grid=(3, 4), patch=16, top=32, left=48, flip_horizontal=True)
    assert torch.equal(got.view(2, 3, 4, 4, 32), full[:, 2:5, 3:7].flip(2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
def test_layouts(pairing, dtype):
    """Slices of a fused projection, transposed heads, odd storage, strided elements, expanded gradients."""
    n, grid, h, d, sections = 2, (4, 6), 3, 64, (32, 32)
    angles = R.rotary_angles(R.grid_positions(grid, 1, device=DEV), sections)
    qkv = _randn((n, 24, 3, h, d), dtype)
    _check(qkv[:, :, 0], qkv[:, :, 1], angles, sections, pairing, grid=grid)
    heads_first = _randn((n, h, 24, d), dtype).transpose(1, 2)
    out, = _check(heads_first, None, angles, sections, pairing, grid=grid)
    assert out.transpose(1, 2).is_contiguous()
    flat = _randn((n * 24 * h * d + 1,), dtype)[1:].view(n, 24, h, d)
    _check(flat, None, angles, sections, pairing, grid=grid)
    _check(_randn((n, 24, h, 2 * d), dtype)[..., ::2], None, angles, sections, pairing, grid=grid)
    _check(_randn((n, 24, h, d + 1), dtype)[..., 1:], None, angles, sections, pairing, grid=grid)
    _check(_randn((1, 1, h, d), dtype).expand(n, 24, h, d), None, angles, sections, pairing, grid=grid, grads=False)
    q = _randn((n, 24, h, d), dtype).requires_grad_()
    g, = torch.autograd.grad(ta.rotary_embedding(q, sections=sections, pairing=pairing, grid=grid).sum(), q)
    R.assert_within(g, *R.rotary(torch.ones_like(q), angles, sections, pairing, inverse=True))


def test_only_one_output_used_and_empty():
    q, k = (_randn((2, 6, 2, 8), torch.float32, s).requires_grad_() for s in (1, 2))
    a, b = ta.rotary_embedding(q, k, sections=(4, 4), grid=(2, 3))
    gk, gq = torch.autograd.grad(b.sum(), (k, q), allow_unused=True)
    assert gq is None
    R.assert_within(gk, *R.rotary(torch.ones_like(k), R.rotary_angles(R.grid_positions((2, 3), 1, device=DEV), (4, 4)), (4, 4), "interleaved", inverse=True))
    for shape in ((0, 6, 2, 8), (2, 6, 0, 8)):
        assert ta.rotary_embedding(torch.empty(shape, device=DEV), sections=(4, 4), grid=(2, 3)).shape == shape
    assert ta.rotary_embedding(torch.empty(2, 0, 2, 8, device=DEV), sections=(4, 4), grid=(0, 3)).shape == (2, 0, 2, 8)
    only = _randn((2, 3, 2, 8), torch.float32)
    assert torch.equal(ta.rotary_embedding(only, sections=(8,), grid=(0,), prefix=3), only)


def test_infinities_stay_in_their_pair():
    q = _randn((1, 4, 1, 8), torch.float32)
    clean = ta.rotary_embedding(q, sections=(4,), grid=(4,))
    q[0, 2, 0, 1], q[0, 3, 0, 6] = float("inf"), float("nan")
    got = ta.rotary_embedding(q, sections=(4,), grid=(4,))
    same = torch.ones_like(q, dtype=torch.bool)
    same[0, 2, 0, :2], same[0, 3, 0, 6] = False, False
    assert torch.equal(got[same], clean[same]) and bool(torch.isnan(got[0, 3, 0, 6])) and not bool(torch.isfinite(got[0, 2, 0, :2]).any())


def test_rotation_is_undone_by_its_gradient():
    """The turn is orthogonal: its transpose applied to the result gives the input back; and the
    gradient agrees with a difference of two calls (the operator is linear)."""
    q = _randn((2, 12, 4, 64), torch.float32).requires_grad_()
    y = ta.rotary_embedding(q, sections=(32, 32), grid=(3, 4))
    back, = torch.autograd.grad(y, q, y.detach())
    pair = q.detach().abs() + q.detach().view(2, 12, 4, 32, 2).flip(-1).reshape(q.shape).abs()
    assert bool(((back - q).abs() <= 40 * R.U * pair).all())
    d, dy = _randn(q.shape, torch.float32, 3), _randn(q.shape, torch.float32, 4)
    g, = torch.autograd.grad(ta.rotary_embedding(q, sections=(32, 32), grid=(3, 4)), q, dy)
    f = lambda t: ta.rotary_embedding(t.detach(), sections=(32, 32), grid=(3, 4)).double()
    num, ana = float(((f(q + d) - f(q)) * dy.double()).sum()), float((g.double() * d.double()).sum())
    assert abs(num - ana) <= 64 * R.U * float(((q.detach().abs() + d.abs()) * dy.abs()).double().sum()) * 2


def test_captured_single_tokens():
    """A decode step: positions and queries change between replays; other stream, same bits."""
    q, k = _randn((8, 1, 16, 128), torch.bfloat16), _randn((8, 1, 4, 128), torch.bfloat16, 1)
    pos = torch.zeros(8, 1, 3, dtype=torch.int64, device=DEV)
    kw = dict(sections=(32, 48, 48), pairing="halves", spectrum="joint", positions=pos)
    ta.rotary_embedding(q, k, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oq, ok = ta.rotary_embedding(q, k, **kw)
    for step in (5, 31000):
        pos.fill_(step)
        q.copy_(_randn(q.shape, q.dtype, step))
        graph.replay()
        angles = R.rotary_angles(pos.double(), (32, 48, 48), spectrum="joint")
        R.assert_within(oq, *R.rotary(q, angles, (32, 48, 48), "halves"))
        R.assert_within(ok, *R.rotary(k, angles, (32, 48, 48), "halves"))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = ta.rotary_embedding(q, k, **kw)
        side.synchronize()
        assert torch.equal(again[0], oq) and torch.equal(again[1], ok)


def test_tokens_beyond_32_bits():
    """A transposed view whose last head starts past 2^32 elements."""
    h, length, d = 2, 2 ** 25 + 8, 64
    base = torch.zeros(1, h, length, d, dtype=torch.float16, device=DEV)
    base[0, 1, -4:] = 1.0
    x = base.transpose(1, 2)[:, -4:]
    assert x.storage_offset() * 2 > 2 ** 32 and x.stride(2) > 2 ** 31
    got = ta.rotary_embedding(x, sections=(64,), grid=(4,))
    angles = R.rotary_angles(R.grid_positions((4,), 1, device=DEV), (64,))
    R.assert_within(got, *R.rotary(x, angles, (64,), "interleaved"))
    del base, x
    torch.cuda.empty_cache()


def test_class():
    rope = ta.TritonRotaryEmbedding((16, 24, 24), patch=16)
    q = _randn((2, 12, 3, 64), torch.bfloat16)
    a, b = rope(q, q, grid=(3, 2, 2), top=5)
    assert torch.equal(a, b) and torch.equal(a, ta.rotary_embedding(q, sections=(16, 24, 24), grid=(3, 2, 2), patch=16, top=5))
    pos = torch.arange(36, device=DEV).view(12, 3)
    assert torch.equal(rope(q, positions=pos), ta.rotary_embedding(q, sections=(16, 24, 24), positions=pos))
    with pytest.raises(ValueError, match="must be on"):
        rope(q, positions=pos.cpu())
    with pytest.raises(ValueError):
        rope(q, grid=(3, 2, 2), top=torch.zeros(3, device=DEV))
