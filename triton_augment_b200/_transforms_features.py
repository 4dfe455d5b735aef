"""Module classes of the feature operators (re-exported by transforms.py)."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import functional as F
from . import transforms as T

__all__ = ["TritonGroupNorm", "TritonDropout", "TritonRotaryEmbedding"]


class TritonGroupNorm(nn.Module):
    """Group normalisation with an activation on channels-last features (``functional.group_norm``), with a
    learned weight and bias unless ``affine=False``.  ``same_on_frame=True``: the frames of a clip share statistics."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True, activation: str = "none",
                 same_on_frame: bool = False, device=None, dtype=None):
        super().__init__()
        if num_groups <= 0 or num_channels <= 0 or num_channels % num_groups:
            raise ValueError(f"{num_channels} channels cannot be split into {num_groups} groups")
        F._choice(activation, F._lib.ACTIVATIONS, "activation")
        self.num_groups, self.num_channels, self.eps = num_groups, num_channels, eps
        self.activation, self.same_on_frame = activation, same_on_frame
        self.weight = nn.Parameter(torch.ones(num_channels, device=device, dtype=dtype)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels, device=device, dtype=dtype)) if affine else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.ndim >= 3 and x.shape[-3] != self.num_channels:
            raise ValueError(f"expected {self.num_channels} channels, got {x.shape[-3]}")
        return F.group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation,
                            same_on_frame=self.same_on_frame)

    def extra_repr(self):
        return (f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.weight is not None}, "
                f"activation={self.activation!r}, same_on_frame={self.same_on_frame}")


class TritonDropout(T._BatchAware):
    """Dropout with a computed mask (``functional.dropout``), seeded by one draw from torch's generator per call.
    ``same_on_batch`` / ``same_on_frame`` share the mask like the random transforms share their parameters.
    Returns the input (plus ``residual``) unchanged in evaluation mode or for ``p == 0``."""

    def __init__(self, p: float = 0.5, mode: str = "element", same_on_batch: bool = False, same_on_frame: bool = True):
        super().__init__(same_on_batch, same_on_frame)
        if not (0.0 <= p <= 1.0):
            raise ValueError(f"p ({p}) must be in [0, 1]")
        F._choice(mode, F._MODES, "mode")
        self.p, self.mode = p, mode

    def forward(self, x: torch.Tensor, residual=None) -> torch.Tensor:
        if not self.training or self.p == 0:
            return x if residual is None else F.dropout(x, 0.0, 0, residual=residual)
        image = x.ndim in (3, 4, 5)
        return F.dropout(x, self.p, mode=self.mode, same_on_batch=self.same_on_batch and (image or self.mode != "element"),
                         same_on_frame=self.same_on_frame and x.ndim == 5, residual=residual)

    def __repr__(self):
        return f"{self.__class__.__name__}(p={self.p}, mode={self.mode!r}, " + self._tail()


class TritonRotaryEmbedding(nn.Module):
    """Rotary positions on queries and keys (``functional.rotary_embedding``) with a fixed split of the head."""

    def __init__(self, sections, base: float = 10000.0, pairing: str = "interleaved", spectrum: str = "axis", patch: float = 1,
                 prefix: int = 0):
        super().__init__()
        self.sections = tuple(int(s) for s in sections)
        if not 1 <= len(self.sections) <= 3 or any(s < 0 or s % 2 for s in self.sections):
            raise ValueError(f"sections must be one to three even sizes, got {sections}")
        F._choice(pairing, F._lib.PAIRINGS, "pairing")
        F._choice(spectrum, F._lib.SPECTRA, "spectrum")
        self.base, self.pairing, self.spectrum, self.patch, self.prefix = base, pairing, spectrum, patch, prefix

    def forward(self, q, k=None, *, positions=None, grid=None, top=0, left=0, flip_horizontal=False):
        return F.rotary_embedding(q, k, sections=self.sections, positions=positions, grid=grid,
                                  patch=1 if grid is None else self.patch, top=top, left=left,
                                  flip_horizontal=flip_horizontal, base=self.base, pairing=self.pairing,
                                  spectrum=self.spectrum, prefix=self.prefix)

    def extra_repr(self):
        return (f"sections={self.sections}, base={self.base}, pairing={self.pairing!r}, spectrum={self.spectrum!r}, "
                f"patch={self.patch}, prefix={self.prefix}")
