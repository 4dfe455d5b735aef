"""The feature operators' definitions in 64 bits (torch, any device), and the error that float32
arithmetic with one final rounding may leave."""
import math

import numpy as np
import torch

U = 2.0 ** -24          # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ----------------------------------------------------------------------------- group norm
def act_and_slope(z, name):
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def group_norm(x, groups, weight, bias, eps, act, same_on_frame=False, dy=None):
    """dict of y and, with dy, dx, dweight, dbias; each with '<name>_tol', the error bound for x's
    (the parameters') type."""
    c = x.shape[-3]
    samples = 1 if x.ndim == 3 else x.shape[0] * (x.shape[1] if x.ndim == 5 and not same_on_frame else 1)
    last = x.movedim(-3, -1).shape
    rows = lambda t: t.movedim(-3, -1).reshape(samples, -1, groups, c // groups).double()
    back = lambda t: t.reshape(last).movedim(-1, -3)
    v = rows(x)
    w = (torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.double()).reshape(groups, -1)
    b = (torch.zeros(c, dtype=torch.float64, device=x.device) if bias is None else bias.double()).reshape(groups, -1)
    mean = v.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((v - mean).square().mean((1, 3), keepdim=True) + eps)
    xhat = (v - mean) * rstd
    z = xhat * w + b
    y, slope = act_and_slope(z, act)
    # |error of z| <= 64 u scale: the mean is off by a few roundings of |mean| + spread (sums of up to 32
    # terms in a row, joined in trees), rstd by a few relative ones, then three roundings; the
    # activations' slopes are below 1.13 and their own error is below 32 u |y|
    scale = (xhat.abs() + mean.abs() * rstd + 1) * w.abs() + b.abs()
    out = dict(y=back(y), y_tol=back(half_step(x.dtype) * y.abs() + 64 * U * scale + tiny(x.dtype)))
    if dy is None:
        return out
    d = rows(dy)
    g = d * slope
    u = g * w
    mu, mux = u.mean((1, 3), keepdim=True), (u * xhat).mean((1, 3), keepdim=True)
    dx = rstd * (u - mu - xhat * mux)
    # slopes change by less than 1.2 per unit of z, so g is off by |dy| (64 u scale 1.2 + 32 u)
    g_err = 128 * U * d.abs() * (scale + 1)
    u_err = g_err * w.abs()
    dx_err = rstd * (u_err + u_err.mean((1, 3), keepdim=True) + xhat.abs() * (u_err * (xhat.abs() + 1)).mean((1, 3), keepdim=True)
                     + 64 * U * (u.abs() + u.abs().mean((1, 3), keepdim=True)
                                 + xhat.abs() * (u * xhat).abs().mean((1, 3), keepdim=True)
                                 + (1 + mean.abs() * rstd) * mux.abs()))
    out.update(dx=back(dx), dx_tol=back(half_step(x.dtype) * dx.abs() + dx_err + tiny(x.dtype)))
    for name, term, err, p in (("dweight", g * xhat, g_err * xhat.abs() + g.abs() * 64 * U * (xhat.abs() + mean.abs() * rstd + 1), weight),
                               ("dbias", g, g_err, bias)):
        if p is None:
            continue
        total = term.sum((0, 1)).reshape(c)
        tol = (err + 64 * U * term.abs()).sum((0, 1)).reshape(c)
        out[name], out[name + "_tol"] = total, half_step(p.dtype) * total.abs() + tol + tiny(p.dtype)
    return out


def tiny(dtype):
    """Half the spacing of the type's subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


# ----------------------------------------------------------------------------- dropout
def philox(counter, key):
    """Philox4x32-10 on numpy uint64 arrays of 32-bit words: counter (4 arrays), key (2 numbers)."""
    m, mask = (np.uint64(0xD2511F53), np.uint64(0xCD9E8D57)), np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(key[0]), int(key[1])]
    for _ in range(10):
        p0, p1 = c[0] * m[0], c[2] * m[1]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & mask, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def mask_numbers(count, seed, offset=0, first=0):
    """32-bit numbers of mask entries first .. first + count - 1."""
    seed &= 2 ** 64 - 1
    entry = np.arange(first, first + count, dtype=np.uint64)
    block, slot = entry >> np.uint64(3), (entry & np.uint64(7)).astype(np.int64)
    out = np.zeros(count, dtype=np.uint64)
    for tag, shift in ((0x64726F70, 16), (0x64726F71, 0)):
        words = philox([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), np.full_like(block, offset), np.full_like(block, tag)],
                       (seed & 0xFFFFFFFF, seed >> 32))
        word = np.choose(slot // 2, words)
        half = np.where(slot % 2 == 0, word & np.uint64(0xFFFF), word >> np.uint64(16))
        out |= half.astype(np.uint64) << np.uint64(shift)
    return out


def dropout_keep(shape, p, seed, offset=0, shared=(), order=None):
    """Boolean mask of a tensor of ``shape``; ``order``: its axes from outermost to innermost in memory;
    ``shared``: axes along which the mask is one value."""
    order = list(range(len(shape))) if order is None else list(order)
    mshape = [1 if a in shared else shape[a] for a in order]
    keep = mask_numbers(math.prod(mshape), seed, offset) >= np.uint64(round(p * 2 ** 32))
    keep = torch.from_numpy(keep.reshape(mshape))
    return keep.permute([order.index(a) for a in range(len(shape))]).expand(shape)


# ----------------------------------------------------------------------------- rotary positions
def rotary_angles(positions, sections, base=10000.0, spectrum="axis"):
    """positions (..., axes) in float64 -> angles (..., pairs)."""
    cols, first, rot = [], 0, sum(sections)
    for a, s in enumerate(sections):
        for m in range(s // 2):
            power = 2.0 * m / s if spectrum == "axis" else 2.0 * (first + m) / rot
            cols.append(positions[..., a] * base ** -power)
        first += s // 2
    return torch.stack(cols, -1) if cols else positions[..., :0]


def rotary(x, angles, sections, pairing, prefix=0, inverse=False):
    """x (N, L, H, D); angles (N or 1, L - prefix, pairs).  Returns the result and its error bound."""
    rot = sum(sections)
    out, tol = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    v = x.double()[:, prefix:, :, :rot]
    c, s = torch.cos(angles)[:, :, None], torch.sin(angles)[:, :, None]
    s = -s if inverse else s
    sl = (slice(0, None, 2), slice(1, None, 2)) if pairing == "interleaved" else (slice(0, rot // 2), slice(rot // 2, None))
    a, b = v[..., sl[0]], v[..., sl[1]]
    for where, val in ((sl[0], a * c - b * s), (sl[1], b * c + a * s)):
        out[:, prefix:, :, :rot][..., where] = val
        # turns: three roundings of numbers below one (2 pi 3 2^-25 = 9.5 u), cosine and sine within 3 u,
        # products and their sum 2 u: below 16 u of |a| + |b|
        tol[:, prefix:, :, :rot][..., where] = half_step(x.dtype) * val.abs() + 16 * U * (a.abs() + b.abs()) + tiny(x.dtype)
    return out, tol


def grid_positions(grid, n, patch=1.0, top=None, left=None, flip=None, device="cpu"):
    """(n, cells, axes) positions of a patch grid, windows as in fused_augment."""
    cols = torch.meshgrid(*[torch.arange(g, dtype=torch.float64, device=device) for g in grid], indexing="ij")
    pos = torch.stack([c.reshape(-1) for c in cols], -1).unsqueeze(0).repeat(n, 1, 1)
    if flip is not None:
        f = torch.as_tensor(flip, device=device).expand(n).bool()
        pos[f, :, -1] = grid[-1] - 1 - pos[f, :, -1]
    if left is not None:
        pos[..., -1] += (torch.as_tensor(left, device=device).double().expand(n) / patch)[:, None]
    if top is not None:
        pos[..., -2] += (torch.as_tensor(top, device=device).double().expand(n) / patch)[:, None]
    return pos


def assert_within(got, want, tol, what=""):
    """Every element within its bound; NaN where NaN is expected.

    A type rounds to infinity from half a step above its largest value M on.  The last step below M is
    M eps / (2 - eps) (M = (2 - eps) 2^e, step eps 2^e), so that is M (1 + eps / (4 - 2 eps)): 65520 for float16.  Infinity
    is right where the exact value and its bound reach that."""
    top = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / (4 - 2 * torch.finfo(got.dtype).eps))
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, (what, tuple(got.shape), tuple(want.shape))
    over = got.isinf() & (got.sign() == want.sign()) & (want.abs() + tol >= top)
    bad = ~((got - want).abs() <= tol) & ~((got == want) | (got.isnan() & want.isnan()) | over)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / tol)[bad].max()), got[bad][:4].tolist(), want[bad][:4].tolist())
