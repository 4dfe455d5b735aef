"""Feature operators without a GPU: what they refuse (Python and C ABI), the reference formulas'
own sanity, mask and parameter layouts."""
import ctypes as C

import numpy as np
import pytest
import torch

import feature_reference as R
import triton_augment_b200 as ta
from triton_augment_b200 import _lib
from triton_augment_b200._functional_features import _mask_layout

X = torch.rand(2, 8, 3, 5)


@pytest.mark.parametrize("kw, err, text", [
    (dict(x=[1.0]), TypeError, "torch.Tensor"),
    (dict(x=X.double()), TypeError, "float32, float16 or bfloat16"),
    (dict(x=X[0, 0]), ValueError, "3D, 4D, or 5D"),
    (dict(num_groups=3), ValueError, "groups"),
    (dict(num_groups=0), ValueError, "num_groups"),
    (dict(num_groups=2.0), ValueError, "num_groups"),
    (dict(weight=torch.ones(7)), ValueError, "shape"),
    (dict(weight=torch.ones(8), bias=torch.ones(8).half()), TypeError, "one dtype"),
    (dict(weight=torch.ones(8).double()), TypeError, "float32"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    (dict(activation="tanh"), ValueError, "activation"),
    (dict(activation=None), ValueError, "activation"),
    (dict(), ValueError, "CUDA"),
])
def test_group_norm_refusals(kw, err, text):
    args = dict(x=X, num_groups=4)
    args.update(kw)
    with pytest.raises(err, match=text):
        ta.group_norm(**args)


@pytest.mark.parametrize("kw, err, text", [
    (dict(x="x"), TypeError, "torch.Tensor"),
    (dict(x=X.long()), TypeError, "float32, float16 or bfloat16"),
    (dict(p=1.5), ValueError, r"p \(1.5\)"),
    (dict(p=-0.1), ValueError, "p "),
    (dict(p=float("nan")), ValueError, "p "),
    (dict(mode="row"), ValueError, "mode"),
    (dict(x=torch.rand(4, 4), mode="channel"), ValueError, "3D, 4D, or 5D"),
    (dict(x=torch.rand(4, 4), same_on_batch=True), ValueError, "3D, 4D, or 5D"),
    (dict(offset=-1), ValueError, "offset"),
    (dict(offset=2 ** 32), ValueError, "offset"),
    (dict(offset=1.0), ValueError, "offset"),
    (dict(seed=1.5), TypeError, "seed"),
    (dict(seed=torch.zeros(2, dtype=torch.int64)), TypeError, "one int64"),
    (dict(seed=torch.zeros(1)), TypeError, "one int64"),
    (dict(residual=X[:1]), ValueError, "shape"),
    (dict(residual=X.half()), TypeError, "residual"),
    (dict(), ValueError, "CUDA"),
    (dict(seed=None), ValueError, "CUDA"),
])
def test_dropout_refusals(kw, err, text):
    args = dict(x=X, p=0.5, seed=1)
    args.update(kw)
    with pytest.raises(err, match=text):
        ta.dropout(**args)


Q = torch.rand(2, 6, 4, 16)
POS = torch.zeros(6, 2, dtype=torch.int64)


@pytest.mark.parametrize("kw, err, text", [
    (dict(q=None), TypeError, "torch.Tensor"),
    (dict(q=Q[0]), ValueError, "heads"),
    (dict(q=Q.int()), TypeError, "float32"),
    (dict(k=Q[:, :5]), ValueError, "shape"),
    (dict(k=Q.half()), TypeError, "like q"),
    (dict(sections=()), ValueError, "one to three axes"),
    (dict(sections=(4, 4, 4, 4)), ValueError, "one to three axes"),
    (dict(sections=(3, 5)), ValueError, "even"),
    (dict(sections=(8, 10)), ValueError, "add up"),
    (dict(base=0.0), ValueError, "base"),
    (dict(base=float("inf")), ValueError, "base"),
    (dict(pairing="both"), ValueError, "pairing"),
    (dict(spectrum="x"), ValueError, "spectrum"),
    (dict(prefix=7), ValueError, "prefix"),
    (dict(grid=None), ValueError, "exactly one"),
    (dict(positions=POS), ValueError, "exactly one"),
    (dict(grid=(2, 2)), ValueError, "patches"),
    (dict(grid=6), ValueError, "sizes"),
    (dict(grid=(-2, -3)), ValueError, "sizes"),
    (dict(patch=0), ValueError, "patch"),
    (dict(grid=None, positions=POS[:5]), ValueError, "shape"),
    (dict(grid=None, positions=POS.double()), TypeError, "positions"),
    (dict(grid=None, positions=[[0, 0]] * 6), TypeError, "positions"),
    (dict(grid=None, positions=POS.float().requires_grad_()), ValueError, "gradients"),
    (dict(grid=None, positions=POS, top=3), ValueError, "top belongs"),
    (dict(grid=None, positions=POS, patch=2), ValueError, "patch belongs"),
    (dict(sections=(8,), grid=(6,), top=3), ValueError, "height"),
    (dict(), ValueError, "CUDA"),
    (dict(top=torch.zeros(2)), ValueError, "CUDA"),
])
def test_rotary_refusals(kw, err, text):
    args = dict(q=Q, sections=(8, 8), grid=(2, 3))
    args.update(kw)
    with pytest.raises(err, match=text):
        ta.rotary_embedding(**args)


def test_class_arguments():
    with pytest.raises(ValueError):
        ta.TritonGroupNorm(3, 8)
    with pytest.raises(ValueError):
        ta.TritonGroupNorm(2, 8, activation="x")
    with pytest.raises(ValueError):
        ta.TritonDropout(1.5)
    with pytest.raises(ValueError):
        ta.TritonDropout(mode="x")
    with pytest.raises(ValueError):
        ta.TritonRotaryEmbedding((3,))
    with pytest.raises(ValueError, match="channels"):
        ta.TritonGroupNorm(2, 8)(torch.rand(1, 6, 2, 2))
    assert "silu" in repr(ta.TritonGroupNorm(2, 8, activation="silu"))
    assert "p=0.1" in repr(ta.TritonDropout(0.1)) and "halves" in repr(ta.TritonRotaryEmbedding((4, 4), pairing="halves"))
    gn = ta.TritonGroupNorm(2, 8, dtype=torch.bfloat16)
    assert [tuple(v.shape) for v in gn.state_dict().values()] == [(8,), (8,)] and gn.weight.dtype == torch.bfloat16
    assert ta.TritonGroupNorm(2, 8, affine=False).weight is None
    x = torch.rand(2, 3)
    assert ta.TritonDropout(0.0)(x) is x and ta.TritonDropout(0.5).eval()(x) is x


# ----------------------------------------------------------------------------- C ABI
def _gn(**kw):
    p = _lib.GroupNormParams()
    p.struct_size = C.sizeof(_lib.GroupNormParams)
    p.n, p.rows, p.channels, p.groups, p.eps = 1, 4, 8, 2, 1e-5
    p.x = p.y = p.mean = p.rstd = 4096
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw, code", [
    (dict(struct_size=8), -2), (dict(dtype=_lib.U8), -3), (dict(weight=4096, param_dtype=7), -3), (dict(activation=9), -4),
    (dict(groups=3), -2), (dict(groups=0), -2), (dict(n=-1), -2), (dict(eps=-1.0), -2), (dict(n=1 << 22), -8),
    (dict(rows=1 << 31), -8), (dict(x=None), -1), (dict(mean=None), -1), (dict(x=4097), -4), (dict(mean=4098), -4), (dict(weight=4098), -4),
    (dict(channels=1 << 21, groups=1), -8),
])
def test_group_norm_abi_refusals(kw, code):
    assert _lib.load().ta_b200_group_norm(C.byref(_gn(**kw)), None) == code
    assert _lib.load().ta_b200_group_norm(None, None) == -1
    if "n" not in kw:
        assert _lib.load().ta_b200_group_norm_backward(C.byref(_gn(**kw)), None) in (code, -1)     # dy is missing too


def _dr(**kw):
    p = _lib.DropoutParams()
    p.struct_size = C.sizeof(_lib.DropoutParams)
    p.sizes[:] = (1, 1, 1, 8)
    p.p, p.x, p.y = 0.5, 4096, 4096
    for k, v in kw.items():
        if k == "sizes":
            p.sizes[:] = v
        else:
            setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw, code", [
    (dict(struct_size=8), -2), (dict(dtype=_lib.U8_F16), -3), (dict(p=1.01), -4), (dict(p=float("nan")), -4),
    (dict(sizes=(1, 1, -1, 8)), -2), (dict(sizes=(1 << 14, 1 << 14, 1 << 14, 1)), -8), (dict(x=None), -1), (dict(y=None), -1),
    (dict(x=4097), -4), (dict(seed_ptr=4100), -4),
])
def test_dropout_abi_refusals(kw, code):
    assert _lib.load().ta_b200_dropout(C.byref(_dr(**kw)), None) == code
    assert _lib.load().ta_b200_dropout(None, None) == -1
    assert _lib.load().ta_b200_dropout(C.byref(_dr(sizes=(1, 0, 1, 8), x=None)), None) == 0       # empty: nothing to do


def _ro(**kw):
    p = _lib.RotaryParams()
    p.struct_size = C.sizeof(_lib.RotaryParams)
    p.n, p.tokens, p.q_heads, p.dim, p.axes, p.base, p.patch = 1, 6, 2, 16, 2, 1e4, 1.0
    p.sections[:] = (8, 8, 0)
    p.grid[:] = (2, 3, 0)
    p.q = p.q_out = 4096
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw, code", [
    (dict(struct_size=8), -2), (dict(dtype=_lib.U8), -3), (dict(prefix=7), -2), (dict(dim=0), -2), (dict(axes=4), -4), (dict(axes=0), -4),
    (dict(sections=(7, 9, 0)), -2), (dict(sections=(8, 10, 0)), -2), (dict(sections=(-8, 8, 0)), -2),
    (dict(dim=600, sections=(300, 300, 0)), -8), (dict(dim=1 << 17), -8), (dict(base=0.0), -4), (dict(pairing=2), -4),
    (dict(spectrum=2), -4), (dict(position_kind=4), -4), (dict(grid=(2, 2, 0)), -2), (dict(grid=(-2, -3, 0)), -2), (dict(patch=0.0), -4),
    (dict(axes=1, sections=(8, 0, 0), grid=(6, 0, 0), top=4096), -4), (dict(q=None), -1), (dict(k_heads=1), -1),
    (dict(position_kind=1), -1), (dict(position_kind=1, positions=4100), -4), (dict(q=4097), -4), (dict(top=4097), -4), (dict(tokens=1 << 31, position_kind=1), -8),
])
def test_rotary_abi_refusals(kw, code):
    assert _lib.load().ta_b200_rotary(C.byref(_ro(**kw)), None) == code
    assert _lib.load().ta_b200_rotary(None, None) == -1


def test_struct_sizes():
    """sizeof on LP64, as the C compiler lays the header's structs out."""
    assert [C.sizeof(s) for s in (_lib.GroupNormParams, _lib.DropoutParams, _lib.RotaryParams)] == [144, 96, 280]


# ----------------------------------------------------------------------------- layouts and references
def test_mask_layout():
    assert _mask_layout((2, 5, 3, 4), False, 0, True, False) == ((2, 1, 5, 12), 1)
    assert _mask_layout((2, 5, 3, 4), False, 1, False, False) == ((2, 1, 5, 12), 8)
    assert _mask_layout((2, 5, 3, 4), True, 1, False, False) == ((2, 1, 12, 5), 4)
    assert _mask_layout((2, 5, 3, 4), True, 2, True, False) == ((2, 1, 12, 5), 8 | 1)
    assert _mask_layout((2, 6, 5, 3, 4), False, 3, False, True) == ((2, 6, 5, 12), 4 | 8 | 2)
    assert _mask_layout((2, 6, 5, 3, 4), False, 0, False, True) == ((2, 6, 5, 12), 2)
    assert _mask_layout((5, 3, 4), False, 1, False, False) == ((1, 1, 5, 12), 8)


def test_reference_generator_known_answers():
    """The published vectors of Philox4x32-10: counter and key of zeros, and of all ones."""
    zero = [int(v[0]) for v in R.philox([np.zeros(1)] * 4, (0, 0))]
    assert zero == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = [int(v[0]) for v in R.philox([np.full(1, 0xFFFFFFFF)] * 4, (0xFFFFFFFF, 0xFFFFFFFF))]
    assert ones == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_reference_mask_statistics():
    """Kept share of p = 0.3 over 2^16 entries: within five standard deviations; neighbours independent."""
    keep = R.dropout_keep((1 << 16,), 0.3, 1234).double()
    sd = (0.3 * 0.7 / (1 << 16)) ** 0.5
    assert abs(float(keep.mean()) - 0.7) < 5 * sd
    assert abs(float((keep[1:] * keep[:-1]).mean()) - 0.49) < 5 * (0.49 * 0.51 * 3 / (1 << 16)) ** 0.5
    assert bool(R.dropout_keep((100,), 0.0, 1).all()) and not bool(R.dropout_keep((100,), 1.0, 1).any())


def test_reference_group_norm_against_torch_and_differences():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 6, 3, 4, generator=g, dtype=torch.float64)
    w, b = torch.randn(6, generator=g, dtype=torch.float64), torch.randn(6, generator=g, dtype=torch.float64)
    dy = torch.randn(2, 6, 3, 4, generator=g, dtype=torch.float64)
    for act, fn in (("none", lambda t: t), ("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu), ("relu", torch.relu)):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = fn(torch.nn.functional.group_norm(leaves[0], 3, leaves[1], leaves[2], 1e-5))
        grads = torch.autograd.grad(y, leaves, dy)
        r = R.group_norm(x, 3, w, b, 1e-5, act, dy=dy)
        for name, want in zip(("y", "dx", "dweight", "dbias"), (y.detach(), *grads)):
            assert float((r[name] - want).abs().max()) < 1e-12, (act, name)


def test_rotary_configuration_is_kept_by_value():
    """A number held in a tensor is read at every call; a size that is no integer is refused, not cut."""
    from triton_augment_b200 import _functional_features as FF
    q = torch.zeros(1, 4, 1, 8)
    patch, before = torch.tensor(2.0), len(FF._ROTARY_CACHE)
    for value in (3.25, 5.75):
        patch.fill_(value)
        with pytest.raises(ValueError, match="CUDA"):
            ta.rotary_embedding(q, sections=(4, 4), grid=(2, 2), patch=patch)
    assert len(FF._ROTARY_CACHE) == min(64, before + 2)
    assert all(type(v) in (float, int, str, tuple, type(None)) for key in FF._ROTARY_CACHE for v in key)
    for kw in (dict(sections=(4.5, 4)), dict(sections=(4, 4), prefix=0.5), dict(sections=(4, 4), grid=(2.0, 2))):
        with pytest.raises(TypeError):
            ta.rotary_embedding(q, **{"grid": (2, 2), **kw})
