"""Operators on what a network makes of the augmented batch: features and patch tokens.

``group_norm`` (channels-last features, with an activation), ``dropout`` (mask computed from a counter,
never stored) and ``rotary_embedding`` (positions with one to three axes).  float32, float16 and
bfloat16 CUDA tensors, differentiable once (backward mode only); each call is one call into libta_b200.so on torch's
current stream.  No counterpart in the reference.

A CUDA graph may hold forward and backward of these operators.  As with any torch operator, no graph
of eager calls on the same leaf tensors may be alive while a backward pass is being captured (drop
the results of warm-up calls first): autograd would make the capturing stream wait for the stream
of the eager call.
"""
from __future__ import annotations

import math
from operator import index

import torch

from . import _lib
from . import functional as _F

__all__ = ["group_norm", "dropout", "rotary_embedding"]


# ----------------------------------------------------------------------------- checks
def _validate_feature_tensor(tensor, name: str) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(tensor)}")
    if tensor.dtype not in _lib.FEATURE_TYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {tensor.dtype}")


def _on_cuda(tensor, name: str) -> None:
    """Checked last: everything else about a call can be refused without a GPU."""
    if not tensor.is_cuda:
        raise ValueError(f"{name} must be on CUDA device")


def _like(tensor, other, name: str, shape=None) -> None:
    """``tensor`` on the device of ``other``, with ``shape``."""
    if tensor.device != other.device:
        raise ValueError(f"{name} must be on {other.device}, got {tensor.device}")
    if shape is not None and tuple(tensor.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(tensor.shape)}")


def _choice(value, table, name: str) -> int:
    code = table.get(value) if isinstance(value, str) else None
    if code is None:
        raise ValueError(f"{name} must be one of {', '.join(repr(k) for k in table)}, got {value!r}")
    return code


# ----------------------------------------------------------------------------- group norm
def group_norm(x, num_groups: int, weight=None, bias=None, eps: float = 1e-5, activation: str = "none", *,
               same_on_frame: bool = False) -> torch.Tensor:
    """Group normalisation and an activation in one pass: ``act((x - mean) / sqrt(var + eps) * weight + bias)``.

    ``x``: features ``(C, H, W)``, ``(N, C, H, W)`` or ``(N, T, C, H, W)`` of any channel count, channels
    last in memory (``torch.channels_last``; each frame of a clip likewise) - any other layout is
    copied to that one first, and the result has it.  ``mean`` and ``var`` (biased) are taken over the
    pixels and the ``C / num_groups`` channels of a group, per image, and per frame of a clip or, with
    ``same_on_frame=True``, over all its frames.  ``weight`` and ``bias``: ``(C,)``, both in one of the three
    types, which need not be the features'.  ``activation``: ``"none"``, ``"relu"``, ``"silu"`` or ``"gelu"`` (exact).

    Statistics and arithmetic are float32, the result is rounded once.  Differentiable in ``x``, ``weight``
    and ``bias``; sums run in a fixed order, so results and gradients repeat bit for bit.
    """
    _validate_feature_tensor(x, "x")
    if x.ndim not in (3, 4, 5):
        raise ValueError(f"Expected 3D, 4D, or 5D tensor, got {x.ndim}D tensor with shape {x.shape}")
    channels = x.shape[-3]
    if isinstance(num_groups, bool) or not isinstance(num_groups, int) or num_groups <= 0:
        raise ValueError(f"num_groups must be a positive integer, got {num_groups}")
    if channels == 0 or channels % num_groups:
        raise ValueError(f"{channels} channels cannot be split into {num_groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _validate_feature_tensor(t, name)
            _like(t, x, name, (channels,))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    act = _choice(activation, _lib.ACTIVATIONS, "activation")
    _on_cuda(x, "x")
    samples = 1 if x.ndim == 3 else x.shape[0] * (x.shape[1] if x.ndim == 5 and not same_on_frame else 1)
    return _lib.torch_binding().group_norm(x, weight, bias, num_groups, float(eps), act, samples)


# ----------------------------------------------------------------------------- dropout
_MODES = {"element": 0, "channel": 1, "pixel": 2, "sample": 3}


def _mask_layout(shape, channels_last, mode, same_on_batch, same_on_frame):
    """Four sizes of the tensor in memory order and the bit set of those the mask is shared along."""
    n = shape[0] if len(shape) >= 4 else 1
    t = shape[1] if len(shape) == 5 else 1
    c, plane = shape[-3], shape[-2] * shape[-1]
    chan_bit, plane_bit = (8, 4) if channels_last else (4, 8)
    shared = ((1 if same_on_batch else 0) | (2 if same_on_frame else 0) | (plane_bit if mode in (1, 3) else 0)
              | (chan_bit if mode in (2, 3) else 0))
    return ((n, t, plane, c) if channels_last else (n, t, c, plane)), shared


def dropout(x, p: float = 0.5, seed=None, *, offset: int = 0, mode: str = "element", same_on_batch: bool = False,
            same_on_frame: bool = False, residual=None) -> torch.Tensor:
    """``residual + keep * x / (1 - p)`` with a mask that is a function of ``(seed, offset, position)`` and is
    computed where it is needed: no mask is stored, and the backward pass computes it again.

    ``seed``: an integer (taken modulo 2^64), a one-element int64 tensor on ``x``'s device (read when the
    kernel runs, so a captured graph can be replayed with another seed; do not overwrite it between a
    forward pass and its backward pass), or None: one draw from torch's generator for that device, so
    ``torch.manual_seed`` repeats it and replays of a captured graph differ.  ``offset`` (0 to 2^32 - 1)
    separates calls that share a seed, such as the layers of a network.

    ``mode``: what is dropped together - ``"element"`` (``x`` of any shape), or, for ``(C, H, W)``, ``(N, C, H, W)``
    and ``(N, T, C, H, W)`` features, ``"channel"`` (whole planes), ``"pixel"`` (all channels of a pixel) or
    ``"sample"`` (whole images; with ``residual``: stochastic depth).  ``same_on_batch`` / ``same_on_frame``: one
    mask for all samples / for all frames of a clip, as in the transform classes (no meaning for a
    single image; same_on_frame none for images).

    A dropped element contributes exactly 0, whatever it held; ``p = 1`` drops everything.  Mask entries are
    numbered in memory order (row-major, or channels last where ``x`` has that layout; other layouts are
    copied to row-major), so the same values in another layout get another mask.  An element is kept
    when its 32-bit number is not below ``round(p * 2^32)``.  The result has ``x``'s layout and is rounded
    once.  Differentiable in ``x`` and ``residual``.
    """
    _validate_feature_tensor(x, "x")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p ({p}) must be in [0, 1]")
    code = _choice(mode, _MODES, "mode")
    if x.ndim not in (3, 4, 5) and (code or same_on_batch or same_on_frame):
        raise ValueError(f"mode={mode!r} and same_on_* need a 3D, 4D, or 5D tensor, got {x.ndim}D tensor with shape {x.shape}")
    if isinstance(offset, bool) or not isinstance(offset, int) or not 0 <= offset < 2 ** 32:
        raise ValueError(f"offset must be an integer in [0, 2^32), got {offset}")
    if residual is not None:
        _validate_feature_tensor(residual, "residual")
        _like(residual, x, "residual", x.shape)
        if residual.dtype != x.dtype:
            raise TypeError(f"residual must be {x.dtype} like x, got {residual.dtype}")
    number, tensor = 0, None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise TypeError(f"a seed tensor must hold one int64, got {seed.dtype} of shape {tuple(seed.shape)}")
        _like(seed, x, "seed")
        tensor = seed
    elif isinstance(seed, int) and not isinstance(seed, bool):
        number = seed & (2 ** 64 - 1)
    elif seed is not None:
        raise TypeError(f"seed must be an integer, an int64 tensor or None, got {type(seed)}")
    _on_cuda(x, "x")
    if seed is None:
        tensor = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), dtype=torch.int64, device=x.device)
    same_on_batch, same_on_frame = bool(same_on_batch) and x.ndim >= 4, bool(same_on_frame) and x.ndim == 5
    return _lib.torch_binding().dropout(x, residual, p, number, tensor, offset, code, same_on_batch, same_on_frame, _mask_layout)


# ----------------------------------------------------------------------------- rotary positions
class _Rotary:
    """What of a call does not depend on its tensors, checked and laid out once per configuration."""
    __slots__ = ("sections", "grid", "prefix", "call")

    def __init__(self, sections, grid, patch, base, pairing, spectrum, prefix):
        self.sections = sections
        axes = len(self.sections)
        if not 1 <= axes <= 3:
            raise ValueError(f"sections must name one to three axes, got {axes}")
        if any(s < 0 or s % 2 for s in self.sections) or sum(self.sections) > 512:
            raise ValueError(f"sections must be even, not negative, and add up to at most 512, got {self.sections}")
        if not 0.0 < base < float("inf"):
            raise ValueError(f"base must be positive, got {base}")
        pairing, spectrum = _choice(pairing, _lib.PAIRINGS, "pairing"), _choice(spectrum, _lib.SPECTRA, "spectrum")
        self.prefix = prefix
        self.grid = grid
        if grid is not None:
            if len(self.grid) != axes or any(g < 0 for g in self.grid):
                raise ValueError(f"grid must have {axes} sizes like sections, got {grid}")
            if not 0.0 < patch < float("inf"):
                raise ValueError(f"patch must be positive, got {patch}")
        self.call = _lib.torch_binding().rotary_spec(list(self.sections), pairing, spectrum, self.prefix, base, self.grid, patch)


_ROTARY_CACHE = {}


def _rotary_spec(*key) -> _Rotary:
    spec = _ROTARY_CACHE.get(key)
    if spec is None:
        spec = _Rotary(*key)
        if len(_ROTARY_CACHE) < 64:
            _ROTARY_CACHE[key] = spec
    return spec


def _per_sample(value, neutral, n, dtype, device, name):
    """A scalar or ``(N,)`` window argument; None where it is the neutral scalar."""
    if not isinstance(value, torch.Tensor) and value == neutral:
        return None
    return _F._convert_to_tensor(value, n, dtype, device, name)


def rotary_embedding(q, k=None, *, sections, positions=None, grid=None, patch: float = 1, top=0, left=0,
                     flip_horizontal=False, base: float = 10000.0, pairing: str = "interleaved", spectrum: str = "axis",
                     prefix: int = 0):
    """Rotary positions with one to three axes on queries ``(N, L, heads, D)`` and, in the same launch, keys
    ``(N, L, key heads, D)``.  Returns the rotated ``q``, or ``(q, k)`` when keys are given.

    ``sections``: for each axis (time, height, width or fewer) how many elements of a head it rotates, even
    numbers whose sum is at most ``D`` (and 512); what is left is copied.  ``pairing="interleaved"`` turns elements
    ``(2j, 2j + 1)``, ``"halves"`` elements ``(j, j + sum(sections) / 2)``; pairs go to the axes in order.  With
    ``spectrum="axis"`` pair ``m`` of an axis has frequency ``base ** (-2m / its section)``, with ``"joint"`` pair ``j`` of
    the head has ``base ** (-2j / sum(sections))``.

    Positions come from one of two arguments.  ``positions``: an int64, int32 or float32 tensor ``(L, axes)`` or
    ``(N, L, axes)`` (tokens of text and of images mixed, single tokens while generating, frame times).
    ``grid``: the patch grid, one size per axis, tokens in row-major order; the index is the position.
    With ``grid``, the window arguments of :func:`fused_augment` keep the patches of a crop at the places
    they had in the whole image: ``top`` and ``left`` (pixels, numbers or ``(N,)`` tensors) move the height and
    width axes by ``top / patch`` and ``left / patch``, where a patch is ``patch`` pixels wide, and for samples
    selected by ``flip_horizontal`` the columns count from the other side.

    The first ``prefix`` tokens of every sample (class or register tokens) are copied; ``grid`` does not
    count them, ``positions`` has (unused) entries for them.  Angles are reduced before they are rounded, so
    positions up to 2^24 in size lose nothing; strided views, such as slices of a fused projection or transposed
    ``(N, heads, L, D)`` tensors, are read in place, and results have the layout ``torch.empty_like`` gives.
    Differentiable in ``q`` and ``k``, not in positions.
    """
    _validate_feature_tensor(q, "q")
    if q.ndim != 4:
        raise ValueError(f"q must have shape (N, L, heads, D), got {tuple(q.shape)}")
    n, length, _, dim = q.shape
    if k is not None:
        _validate_feature_tensor(k, "k")
        if k.ndim != 4:
            raise ValueError(f"k must have shape (N, L, heads, D), got {tuple(k.shape)}")
        _like(k, q, "k", (n, length, k.shape[2], dim))
        if k.dtype != q.dtype:
            raise TypeError(f"k must be {q.dtype} like q, got {k.dtype}")
    if isinstance(grid, int):
        grid = (grid,)
    patch = float(patch)                                  # (numbers only: a tensor in the key would stand for its identity)
    spec = _rotary_spec(tuple(map(index, sections)), None if grid is None else tuple(map(index, grid)), patch, float(base),
                        pairing, spectrum, index(prefix))
    axes, prefix = len(spec.sections), spec.prefix
    if sum(spec.sections) > dim:
        raise ValueError(f"sections must be even, not negative, and add up to at most {dim}, got {spec.sections}")
    if not 0 <= prefix <= length:
        raise ValueError(f"prefix must be in [0, {length}], got {prefix}")
    if (positions is None) == (grid is None):
        raise ValueError("exactly one of positions and grid must be given")
    top_t = left_t = flip_t = None
    window = [name for name, v in (("top", top), ("left", left), ("flip_horizontal", flip_horizontal))
              if isinstance(v, torch.Tensor) or v]
    if positions is not None:
        if not isinstance(positions, torch.Tensor):
            raise TypeError(f"positions must be a torch.Tensor, got {type(positions)}")
        if positions.dtype not in _lib.POSITION_TYPES:
            raise TypeError(f"positions must be int64, int32 or float32, got {positions.dtype}")
        if tuple(positions.shape) not in ((length, axes), (n, length, axes)):
            raise ValueError(f"positions must have shape ({length}, {axes}) or ({n}, {length}, {axes}), got {tuple(positions.shape)}")
        _like(positions, q, "positions")
        if positions.requires_grad:
            raise ValueError("positions must not require gradients")
        if window or patch != 1:
            raise ValueError(f"{', '.join(window) or 'patch'} belongs to grid, not to positions")
    else:
        if math.prod(spec.grid) != length - prefix:
            raise ValueError(f"grid {spec.grid} has {math.prod(spec.grid)} patches for {length - prefix} tokens")
        if axes < 2 and "top" in window:
            raise ValueError("top needs a height axis")
        _on_cuda(q, "q")
        top_t = _per_sample(top, 0, n, torch.float32, q.device, "top")
        left_t = _per_sample(left, 0, n, torch.float32, q.device, "left")
        flip_t = _per_sample(flip_horizontal, False, n, torch.bool, q.device, "flip_horizontal")
    _on_cuda(q, "q")
    return _lib.torch_binding().rotary(q, k, positions, top_t, left_t, flip_t, spec.call)
