"""The C entries' results in the place of their inputs: the bits of the calls with results of their own."""
import ctypes as C

import pytest
import torch

import triton_augment_b200 as ta
from triton_augment_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.float16, torch.bfloat16]
CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 4}          # TA_B200_F32, _F16, _BF16


def _call(entry, p):
    lib = _lib.load()
    p.struct_size = C.sizeof(p)
    _lib.check(getattr(lib, entry)(C.byref(p), _lib._stream(0)), entry)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, c, h, w, groups", [(2, 64, 20, 20, 8), (1, 128, 200, 200, 32), (2, 33, 9, 11, 11), (3, 130, 40, 31, 10), (1, 2056, 3, 3, 1)])
def test_group_norm(n, c, h, w, groups, dtype):
    x = torch.randn(n, h, w, c, device=DEV).to(dtype)
    dy = torch.randn(n, h, w, c, device=DEV).to(dtype)
    weight, bias = torch.randn(2, c, device=DEV)
    leaves = [t.clone().requires_grad_() for t in (x, weight, bias)]
    y = ta.group_norm(leaves[0].permute(0, 3, 1, 2), groups, leaves[1], leaves[2], activation="silu")
    want = torch.autograd.grad(y, leaves, dy.permute(0, 3, 1, 2))
    lib, stats = _lib.load(), torch.empty(2, n * groups, device=DEV)
    dw, db, held = torch.empty_like(weight), torch.empty_like(bias), x.clone()
    p = _lib.GroupNormParams()
    p.dtype, p.param_dtype, p.activation = CODE[dtype], CODE[torch.float32], _lib.ACTIVATIONS["silu"]
    p.n, p.rows, p.channels, p.groups, p.eps = n, h * w, c, groups, 1e-5
    p.weight, p.bias, p.mean, p.rstd = weight.data_ptr(), bias.data_ptr(), stats.data_ptr(), stats[1].data_ptr()
    p.struct_size = C.sizeof(p)

    def run(entry, backward):
        size = lib.ta_b200_group_norm_scratch_bytes(C.byref(p), backward)
        scratch = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
        p.scratch, p.scratch_bytes = scratch.data_ptr(), size
        _call(entry, p)
    p.x = p.y = held.data_ptr()
    run("ta_b200_group_norm", 0)
    assert torch.equal(held, y.detach().permute(0, 2, 3, 1))
    p.x, p.y, p.dy, p.dx, p.dweight, p.dbias = x.data_ptr(), None, dy.data_ptr(), dy.data_ptr(), dw.data_ptr(), db.data_ptr()
    run("ta_b200_group_norm_backward", 1)
    for got, grad in zip((dy, dw, db), want):
        assert torch.equal(got, grad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start", [0, 1])
@pytest.mark.parametrize("sizes, shared", [((1, 1, 1, 40001), 0), ((3, 1, 70, 257), 8), ((3, 1, 70, 257), 4), ((3, 2, 70, 129), 5), ((2, 3, 5, 7), 2)])
def test_dropout(sizes, shared, start, dtype):
    numel = sizes[0] * sizes[1] * sizes[2] * sizes[3]
    pool = torch.randn(3, (numel + 31) // 16 * 16, device=DEV).to(dtype)
    x, r, out = (t[start:start + numel] for t in pool)

    def run(source, residual, target):
        p = _lib.DropoutParams()
        p.dtype, p.p, p.seed, p.shared, p.offset = CODE[dtype], 0.3, 77, shared, 2
        p.sizes[:] = sizes
        p.x, p.y = source.data_ptr(), target.data_ptr()
        p.residual = None if residual is None else residual.data_ptr()
        _call("ta_b200_dropout", p)
        return target.clone()
    plain, added = run(x, None, out), run(x, r, out)
    assert torch.equal(run(x.clone() if start == 0 else x, r, r), added)
    held = pool[0].clone()
    assert torch.equal(run(held[start:start + numel], None, held[start:start + numel]), plain)
    assert torch.equal(held[:start], pool[0][:start]) and torch.equal(held[start + numel:], pool[0][start + numel:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("dim, sections, start", [(64, (32, 32), 0), (72, (32, 36), 0), (64, (32, 32), 1), (19, (6, 8), 0), (40, (16, 16), 3)])
def test_rotary(dim, sections, start, pairing, dtype):
    n, grid, heads, kv = 2, (5, 7), 3, 2
    tokens = grid[0] * grid[1]
    size = n * tokens * heads * dim
    pool = torch.randn(2, (size + 31) // 16 * 16, device=DEV).to(dtype)
    q = pool[0][start:start + size].view(n, tokens, heads, dim)
    k = pool[1][start:start + n * tokens * kv * dim].view(n, tokens, kv, dim)
    want = ta.rotary_embedding(q, k, sections=sections, grid=grid, pairing=pairing)
    p = _lib.RotaryParams()
    p.dtype, p.n, p.tokens, p.q_heads, p.k_heads, p.dim, p.axes = CODE[dtype], n, tokens, heads, kv, dim, 2
    p.sections[:], p.grid[:], p.base, p.patch = (*sections, 0), (*grid, 0), 1e4, 1.0
    p.pairing, p.spectrum = _lib.PAIRINGS[pairing], _lib.SPECTRA["axis"]
    p.q = p.q_out = q.data_ptr()
    p.k = p.k_out = k.data_ptr()
    p.q_strides[:] = p.q_out_strides[:] = q.stride()[:3]
    p.k_strides[:] = p.k_out_strides[:] = k.stride()[:3]
    tail = pool[:, start + size:].clone()
    _call("ta_b200_rotary", p)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(pool[:, start + size:], tail)
