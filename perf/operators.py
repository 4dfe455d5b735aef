"""Feature operators next to the augmentations: what is timed, on which sizes, and against what.

Three operators that a network applies to the images, clips and patch tokens this package prepares:

* ``group_norm``: group normalisation with an activation on channels-last features, forward and
  backward;
* ``dropout``: dropout whose mask is a function of (seed, element) and is never stored, per element or
  shared by channels, pixels, frames or the batch, with an optional residual, forward and backward;
* ``rotary_embedding``: rotary positions with one to three axes (time, height, width) on the queries
  and keys of patch tokens, forward and backward.

``run`` computes them with elementary torch operations in 32 bits (``own = False``) or through the
package's entry points (``own = True``); ``exact`` gives the operators' definitions in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_MASK32 = 0xFFFFFFFF


# ----------------------------------------------------------------------------- cases
def _gn(name, dtype, n, c, h, w, groups, activation, t=0, train=False, same_on_frame=False):
    """t = 0: images (n, c, h, w); t > 0: clips (n, t, c, h, w)."""
    return dict(name=name, op="group_norm", dtype=dtype, n=n, t=t, c=c, h=h, w=w, groups=groups, activation=activation,
                train=train, same_on_frame=same_on_frame)


def _dr(name, dtype, shape, p, mode="element", train=False, residual=False, channels_last=False, same_on_batch=False,
        same_on_frame=False):
    """shape: tokens (n, l, d), images (n, c, h, w) or clips (n, t, c, h, w), as text "nxlxd"."""
    return dict(name=name, op="dropout", dtype=dtype, shape=shape, p=p, mode=mode, train=train, residual=residual,
                channels_last=channels_last, same_on_batch=same_on_batch, same_on_frame=same_on_frame)


def _ro(name, dtype, n, grid, heads, kv_heads, dim, sections, pairing="interleaved", spectrum="axis", train=False, prefix=0,
        patch=1, window=False, positions="grid"):
    """grid: "14x14" or "8x14x14" tokens; kv_heads = 0: queries only; positions "grid", "int64" or "float32"
    (a tensor of that type with one entry per sample, token and axis); window: crop offsets and flips per sample."""
    return dict(name=name, op="rotary", dtype=dtype, n=n, grid=grid, heads=heads, kv_heads=kv_heads, dim=dim,
                sections=sections, pairing=pairing, spectrum=spectrum, train=train, prefix=prefix, patch=patch, window=window,
                positions=positions)


def listed():
    return [
        # one image's late feature map while serving: latency counts
        _gn("gn_one_image", "float16", 1, 64, 14, 14, 8, "silu"),
        # the early blocks of a network on a batch of 224-pixel crops
        _gn("gn_batch", "bfloat16", 32, 256, 56, 56, 32, "silu"),
        # full-resolution features of a decoder: a sample is larger than an SM's memory many times over
        _gn("gn_full_resolution", "float16", 16, 128, 224, 224, 32, "silu"),
        # a training step at a quarter of the resolution, ten channels to a group
        _gn("gn_train", "bfloat16", 64, 320, 28, 28, 32, "silu", train=True),
        # clips normalised over their frames, odd sizes, single precision
        _gn("gn_train_clips", "float32", 4, 96, 35, 35, 12, "gelu", t=8, train=True, same_on_frame=True),
        # the tokens of one 224-pixel image with a class token
        _dr("dropout_one_image", "bfloat16", "1x197x768", 0.1),
        # a transformer block's residual branch in training
        _dr("dropout_residual_train", "bfloat16", "128x197x768", 0.1, train=True, residual=True),
        # clips whose frames lose the same pixels: odd planes, channels last
        _dr("dropout_clip_pixels", "float16", "8x16x24x57x57", 0.25, mode="pixel", channels_last=True, same_on_frame=True),
        # serving: one new token for each of 32 requests, three-axis positions, few key heads
        _ro("rotary_one_token", "bfloat16", 32, "1x1x1", 16, 4, 128, "32x48x48", pairing="halves", spectrum="joint",
            positions="int64"),
        # training on clips of 16 frames in tubes of two, 14 x 14 patches
        _ro("rotary_train_clips", "bfloat16", 8, "8x14x14", 12, 12, 64, "16x24x24", train=True),
        # large images, 64 x 64 patches: bandwidth counts
        _ro("rotary_large_images", "bfloat16", 16, "64x64", 16, 16, 128, "64x64", pairing="halves"),
        # patches of random crop windows keep the places they had in the whole image; odd grid, class token
        _ro("rotary_crop_windows", "float32", 24, "15x21", 6, 2, 72, "32x36", prefix=1, patch=16, window=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("group_norm", "dropout", "rotary"))
    dtype = rng.choice(("float32", "float16", "bfloat16"))
    train = rng.random() < 0.5
    limit = 32_000_000                                  # elements; the largest listed case has 268 435 456 of them
    if op == "group_norm":
        while True:
            groups = rng.choice((1, 2, 4, 8, 12, 16, 32))
            c = groups * _log_int(rng, 1, 40)
            n, h, w = _log_int(rng, 1, 128), _log_int(rng, 1, 224), _log_int(rng, 1, 224)
            t = rng.choice((0, 0, _log_int(rng, 1, 16)))
            if 64 <= n * max(t, 1) * c * h * w <= limit:
                break
        # (relu's slope jumps at zero, where the last bit decides: forward only)
        activation = rng.choice(("none", "silu", "gelu") if train else ("none", "relu", "silu", "gelu"))
        return _gn(None, dtype, n, c, h, w, groups, activation, t, train, t > 0 and rng.random() < 0.5)
    if op == "dropout":
        while True:
            kind = rng.choice(("tokens", "images", "clips"))
            if kind == "tokens":
                dims = [_log_int(rng, 1, 256), _log_int(rng, 1, 1024), _log_int(rng, 16, 2048)]
            else:
                dims = [_log_int(rng, 1, 128), _log_int(rng, 1, 512), _log_int(rng, 1, 128), _log_int(rng, 1, 128)]
                if kind == "clips":
                    dims.insert(1, _log_int(rng, 1, 16))
            if 64 <= math.prod(dims) <= limit:
                break
        image = kind != "tokens"
        return _dr(None, dtype, "x".join(map(str, dims)), rng.choice((0.05, 0.1, 0.25, 0.5, 0.9)),
                   rng.choice(("element", "channel", "pixel", "sample")) if image else "element", train,
                   rng.random() < 0.5, image and rng.random() < 0.5, image and rng.random() < 0.25,
                   kind == "clips" and rng.random() < 0.5)
    while True:
        axes = rng.choice((1, 2, 3))
        grid = [_log_int(rng, 1, 4096)] if axes == 1 else [_log_int(rng, 1, 64) for _ in range(axes)]
        n, heads = _log_int(rng, 1, 64), _log_int(rng, 1, 32)
        sections = [2 * _log_int(rng, 1, 32) for _ in range(axes)]
        dim = sum(sections) + rng.choice((0, 0, 0, 1, 8, 16))
        kv = rng.choice((0, 1, max(1, heads // 4), heads))
        if n * math.prod(grid) * (heads + kv) * dim <= limit:
            break
    positions = rng.choice(("grid", "grid", "int64", "float32"))
    return _ro(None, dtype, n, "x".join(map(str, grid)), heads, kv, dim, "x".join(map(str, sections)),
               rng.choice(("interleaved", "halves")), rng.choice(("axis", "joint")), train, rng.choice((0, 0, 1, 4)),
               rng.choice((8, 14, 16)) if positions == "grid" else 1,
               positions == "grid" and axes >= 2 and rng.random() < 0.5, positions)


# ----------------------------------------------------------------------------- sizes and work
def _ints(text):
    return tuple(int(v) for v in text.split("x"))


def _image_shape(case):
    return (case["n"], case["t"], case["c"], case["h"], case["w"]) if case["t"] else (case["n"], case["c"], case["h"], case["w"])


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    train = case["train"]
    if case["op"] == "group_norm":
        numel = math.prod(_image_shape(case))
        # forward: read x, write y; training step: read x and dy, write y and dx (x twice: the forward
        # pass is over before dy exists)
        tensors = 5 if train else 2
        flops = {"none": 0, "relu": 1, "silu": 5, "gelu": 12}[case["activation"]]
        return {"bytes": tensors * numel * size, "flops": numel * ((7 + flops) * (3 if train else 1))}
    if case["op"] == "dropout":
        numel = math.prod(_ints(case["shape"]))
        tensors = 2 + (1 if case["residual"] else 0) + (2 if train else 0)
        return {"bytes": tensors * numel * size, "flops": 2 * numel * (2 if train else 1)}
    tokens = case["n"] * (math.prod(_ints(case["grid"])) + case["prefix"])
    numel = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
    pos = tokens * len(_ints(case["sections"])) * {"grid": 0, "int64": 8, "float32": 4}[case["positions"]]
    return {"bytes": (4 if train else 2) * numel * size + pos, "flops": 3 * numel * (2 if train else 1)}


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev, dt = torch.device("cuda"), _DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    host = torch.Generator()
    host.manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)
    state = {"case": case}
    if case["op"] == "group_norm":
        c, shape = case["c"], _image_shape(case)
        last = shape[:-3] + shape[-2:] + (c,)                            # memory order: channels last
        back = (0, 1, 4, 2, 3) if case["t"] else (0, 3, 1, 2)
        # a convolution's output: channels with their own mean and spread
        x = torch.empty(last, dtype=dt, device=dev)
        x.copy_(normal(*last).mul_(0.5 + torch.rand(c, generator=gen, device=dev)).add_(normal(c)))
        state["x"] = x.permute(back)
        # parameters: single precision in training, the features' type while serving
        param = torch.float32 if case["train"] else dt
        state["weight"] = (1.0 + 0.2 * normal(c)).to(param)
        state["bias"] = (0.2 * normal(c)).to(param)
        if case["train"]:
            state["dy"] = normal(*last).to(dt).permute(back)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_(True)
        return state
    if case["op"] == "dropout":
        shape = _ints(case["shape"])
        def tensor():
            if not case["channels_last"]:
                return normal(*shape).to(dt)
            last = shape[:-3] + shape[-2:] + shape[-3:-2]
            return normal(*last).to(dt).permute((0, 1, 4, 2, 3) if len(shape) == 5 else (0, 3, 1, 2))
        state["x"] = tensor()
        state["residual"] = tensor() if case["residual"] else None
        state["seed"] = int(torch.randint(0, 2 ** 62, (1,), generator=host))
        if case["train"]:
            state["dy"] = tensor()
            state["x"].requires_grad_(True)
            if case["residual"]:
                state["residual"].requires_grad_(True)
        return state
    grid, sections = _ints(case["grid"]), _ints(case["sections"])
    n, length = case["n"], math.prod(grid) + case["prefix"]
    state["q"] = normal(n, length, case["heads"], case["dim"]).to(dt)
    state["k"] = normal(n, length, case["kv_heads"], case["dim"]).to(dt) if case["kv_heads"] else None
    if case["positions"] == "int64":                                     # requests that are up to 32768 tokens long
        state["positions"] = torch.randint(0, 32768, (n, length, len(sections)), generator=gen, device=dev)
    elif case["positions"] == "float32":
        state["positions"] = torch.rand(n, length, len(sections), generator=gen, device=dev) * 1024.0
    if case["window"]:
        state["top"] = torch.randint(0, 800, (n,), generator=gen, device=dev).float()
        state["left"] = torch.randint(0, 800, (n,), generator=gen, device=dev).float()
        state["flip"] = torch.rand(n, generator=gen, device=dev) < 0.5
    if case["train"]:
        state["dq"] = normal(n, length, case["heads"], case["dim"]).to(dt)
        state["q"].requires_grad_(True)
        if case["kv_heads"]:
            state["dk"] = normal(n, length, case["kv_heads"], case["dim"]).to(dt)
            state["k"].requires_grad_(True)
    return state


# ----------------------------------------------------------------------------- the plain forms
def _plain_activation(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _plain_group_norm(x, weight, bias, case):
    shape, g = x.shape, case["groups"]
    n = case["n"] if case["same_on_frame"] or not case["t"] else case["n"] * case["t"]
    last = x.movedim(-3, -1).float()
    v = last.reshape(n, -1, g, shape[-3] // g)
    mean = v.mean(dim=(1, 3), keepdim=True)
    d = v - mean
    var = (d * d).mean(dim=(1, 3), keepdim=True)
    z = (d * (1.0 / torch.sqrt(var + 1e-5))).reshape(last.shape) * weight.float() + bias.float()
    return _plain_activation(z, case["activation"]).to(x.dtype).movedim(-1, -3)


def _philox(block, seed, offset, tag):
    """Philox4x32-10 of counter (block, offset, tag) with 32-bit words in int64 tensors.  A product of
    two 32-bit words wraps modulo 2^64; its upper word is still right after the mask."""
    c = [block & _MASK32, block >> 32, torch.full_like(block, offset), torch.full_like(block, tag)]
    k0, k1 = seed & _MASK32, (seed >> 32) & _MASK32
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & _MASK32) ^ c[1] ^ k0, p1 & _MASK32, ((p0 >> 32) & _MASK32) ^ c[3] ^ k1, p0 & _MASK32]
        k0, k1 = (k0 + 0x9E3779B9) & _MASK32, (k1 + 0xBB67AE85) & _MASK32
    return c


def _halves(words):
    """Four 32-bit words -> eight 16-bit numbers, low half first."""
    return torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], dim=-1)


def _shared_axes(case, ndim):
    """Axes (of the tensor in memory order) along which the mask is one value."""
    axes = set()
    if ndim >= 4 or case["mode"] != "element":
        inner = (ndim - 3, ndim - 2, ndim - 1)
        chan, space = (inner[2], inner[:2]) if case["channels_last"] else (inner[0], inner[1:])
        if case["mode"] in ("channel", "sample"):
            axes.update(space)
        if case["mode"] in ("pixel", "sample"):
            axes.add(chan)
        if case["same_on_batch"]:
            axes.add(0)
        if case["same_on_frame"] and ndim == 5:
            axes.add(1)
    return axes


def _plain_keep(x_mem, case, seed):
    shared = _shared_axes(case, x_mem.ndim)
    mask_shape = [1 if a in shared else s for a, s in enumerate(x_mem.shape)]
    count = math.prod(mask_shape)
    block = torch.arange((count + 7) // 8, device=x_mem.device)
    number = _halves(_philox(block, seed, 0, 0x64726F70)) * 65536 + _halves(_philox(block, seed, 0, 0x64726F71))
    return (number.reshape(-1)[:count] >= int(round(case["p"] * 2.0 ** 32))).reshape(mask_shape)


def _plain_dropout(x, residual, seed, case):
    mem = (lambda v: v.movedim(-3, -1)) if case["channels_last"] else (lambda v: v)
    xm = mem(x).float()
    y = torch.where(_plain_keep(xm, case, seed), xm * (1.0 / (1.0 - case["p"])), torch.zeros_like(xm))
    if residual is not None:
        y = y + mem(residual).float()
    y = y.to(x.dtype)
    return y.movedim(-1, -3) if case["channels_last"] else y


def _plain_positions(state):
    """Positions (n, grid tokens, axes) in 64 bits."""
    case = state["case"]
    if "positions" in state:
        return state["positions"][:, case["prefix"]:].double()
    grid, patch, dev = _ints(case["grid"]), float(case["patch"]), state["q"].device
    n = case["n"]
    cols = []
    for a, size in enumerate(grid):
        index = torch.arange(size, device=dev, dtype=torch.float64).expand(n, size)
        from_end = len(grid) - 1 - a                                     # 0: width, 1: height
        if case["window"] and from_end == 0:
            index = torch.where(state["flip"][:, None], size - 1 - index, index) + state["left"].double()[:, None] / patch
        elif case["window"] and from_end == 1:
            index = index + state["top"].double()[:, None] / patch
        view = [n] + [1] * len(grid)
        view[1 + a] = size
        cols.append(index.reshape(view).expand(n, *grid).reshape(n, -1))
    return torch.stack(cols, dim=-1)


def _plain_cos_sin(state):
    case = state["case"]
    sections = _ints(case["sections"])
    pos, rot = _plain_positions(state), sum(sections)
    angles, first = [], 0
    for a, s in enumerate(sections):
        j = torch.arange(s // 2, device=pos.device, dtype=torch.float64)
        power = 2.0 * j / s if case["spectrum"] == "axis" else 2.0 * (j + first) / rot
        angles.append(pos[:, :, a, None] * torch.exp(-power * math.log(10000.0)))
        first += s // 2
    angle = torch.cat(angles, dim=-1)[:, :, None, :]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_rotate(x, cos, sin, case):
    prefix, rot = case["prefix"], sum(_ints(case["sections"]))
    head, v, tail = x[:, :prefix].float(), x[:, prefix:, :, :rot].float(), x[:, prefix:, :, rot:].float()
    if case["pairing"] == "interleaved":
        a, b = v[..., 0::2], v[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = v[..., :rot // 2], v[..., rot // 2:]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((head, torch.cat((out, tail), dim=-1)), dim=1).to(x.dtype)


# ----------------------------------------------------------------------------- one pass
def _forward(state):
    """The operator's outputs, and the leaves and incoming gradients of a training step."""
    case = state["case"]
    if case["op"] == "group_norm":
        if own:
            import triton_augment_b200 as ta
            y = ta.group_norm(state["x"], case["groups"], state["weight"], state["bias"], eps=1e-5,
                              activation=case["activation"], same_on_frame=case["same_on_frame"])
        else:
            y = _plain_group_norm(state["x"], state["weight"], state["bias"], case)
        return [y], [state["x"], state["weight"], state["bias"]], [state.get("dy")]
    if case["op"] == "dropout":
        if own:
            import triton_augment_b200 as ta
            y = ta.dropout(state["x"], case["p"], state["seed"], mode=case["mode"], same_on_batch=case["same_on_batch"],
                           same_on_frame=case["same_on_frame"], residual=state["residual"])
        else:
            y = _plain_dropout(state["x"], state["residual"], state["seed"], case)
        return [y], [state["x"]] + ([state["residual"]] if case["residual"] else []), [state.get("dy")]
    if own:
        import triton_augment_b200 as ta
        where = dict(positions=state["positions"]) if "positions" in state else dict(grid=_ints(case["grid"]), patch=case["patch"])
        if case["window"]:
            where.update(top=state["top"], left=state["left"], flip_horizontal=state["flip"])
        out = ta.rotary_embedding(state["q"], state["k"], sections=_ints(case["sections"]), base=10000.0,
                                  pairing=case["pairing"], spectrum=case["spectrum"], prefix=case["prefix"], **where)
        out = list(out) if case["kv_heads"] else [out]
    else:
        cos, sin = _plain_cos_sin(state)
        out = [_plain_rotate(state["q"], cos, sin, case)]
        if case["kv_heads"]:
            out.append(_plain_rotate(state["k"], cos, sin, case))
    leaves, grads = [state["q"]], [state.get("dq")]
    if case["kv_heads"]:
        leaves.append(state["k"])
        grads.append(state.get("dk"))
    return out, leaves, grads


def run(state):
    out, leaves, grads = _forward(state)
    if not state["case"]["train"]:
        return out
    back = torch.autograd.grad(out, leaves, grads)
    return [o.detach() for o in out] + list(back)


# ----------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"group_norm": _exact_group_norm, "dropout": _exact_dropout, "rotary": _exact_rotary}[case["op"]](case, state)


def _exact_group_norm(case, s):
    """y = act(z), z = xhat * weight + bias, xhat = (x - mean) / sqrt(var + eps) over each sample's group.
    With g = dy * act'(z) and u = g * weight: dweight = sum g * xhat, dbias = sum g, and
    dx = (u - mean(u) - xhat * mean(u * xhat)) / sqrt(var + eps), the means over the group."""
    n = case["n"] * (1 if case["same_on_frame"] or not case["t"] else case["t"])
    c, groups = case["c"], case["groups"]
    rows = math.prod(_image_shape(case)) // (n * c)
    to_rows = lambda v: v.detach().movedim(-3, -1).reshape(n, rows, groups, c // groups).double()
    from_rows = lambda v: v.reshape(s["x"].movedim(-3, -1).shape).movedim(-1, -3)
    x = to_rows(s["x"])
    weight, bias = (s[k].detach().double().reshape(groups, c // groups) for k in ("weight", "bias"))
    count = rows * (c // groups)
    centred = x - x.sum((1, 3), keepdim=True) / count
    rstd = torch.rsqrt(centred.square().sum((1, 3), keepdim=True) / count + 1e-5)
    xhat = centred * rstd
    z = xhat * weight + bias
    act = case["activation"]
    if act == "silu":
        sig = torch.sigmoid(z)
        y, slope = z * sig, sig * (1.0 + z * (1.0 - sig))
    elif act == "relu":
        y, slope = z.clamp(min=0.0), (z > 0).double()
    elif act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    else:
        y, slope = z, torch.ones_like(z)
    if not case["train"]:
        return [from_rows(y)]
    g = to_rows(s["dy"]) * slope
    u = g * weight
    dx = rstd * (u - u.sum((1, 3), keepdim=True) / count - xhat * ((u * xhat).sum((1, 3), keepdim=True) / count))
    return [from_rows(y), from_rows(dx), (g * xhat).sum((0, 1)).reshape(c), g.sum((0, 1)).reshape(c)]


def _exact_words(index, seed, tag):
    """16-bit number of each mask entry: Philox4x32-10 on its block of eight, products from 16-bit limbs."""
    def product(v, m):
        lo, hi = (v & 0xFFFF) * m, (v >> 16) * m                          # both below 2^48
        full_lo = lo + ((hi & 0xFFFF) << 16)
        return full_lo & _MASK32, (full_lo >> 32) + (hi >> 16)
    block = torch.div(index, 8, rounding_mode="floor")
    a, b, c, d = block % (1 << 32), block // (1 << 32), torch.zeros_like(block), torch.zeros_like(block) + tag
    for r in range(10):
        lo0, hi0 = product(a, 0xD2511F53)
        lo1, hi1 = product(c, 0xCD9E8D57)
        ka = (seed + r * 0x9E3779B9) % (1 << 32)
        kb = ((seed >> 32) + r * 0xBB67AE85) % (1 << 32)
        a, b, c, d = hi1 ^ b ^ ka, lo1, hi0 ^ d ^ kb, lo0
    slot = index % 8
    word = torch.where(slot < 2, a, torch.where(slot < 4, b, torch.where(slot < 6, c, d)))
    return torch.where(slot % 2 == 0, word % 65536, word // 65536)


def _exact_dropout(case, s):
    """out = residual + keep * x / (1 - p), dx = keep * dy / (1 - p); keep: the mask entry's 32-bit number is
    not below round(p 2^32).  Mask entries count in memory order over the axes that are not shared."""
    x = s["x"].detach()
    to_mem = (lambda v: v.detach().movedim(-3, -1)) if case["channels_last"] else (lambda v: v.detach())
    back = (lambda v: v.movedim(-1, -3)) if case["channels_last"] else (lambda v: v)
    xm = to_mem(x)
    names = {3: "ntc", 4: "ncss", 5: "nfcss"}[xm.ndim] if not case["channels_last"] else {4: "nssc", 5: "nfssc"}[xm.ndim]
    free = {"element": "nfcst", "channel": "nfc", "pixel": "nfs", "sample": "nf"}[case["mode"]]
    if case["same_on_batch"]:
        free = free.replace("n", "")
    if case["same_on_frame"]:
        free = free.replace("f", "")
    index, stride = torch.zeros([1] * xm.ndim, dtype=torch.int64, device=x.device), 1
    for a in reversed(range(xm.ndim)):
        if names[a] in free:
            view = [1] * xm.ndim
            view[a] = xm.shape[a]
            index = index + torch.arange(xm.shape[a], device=x.device).reshape(view) * stride
            stride *= xm.shape[a]
    number = (_exact_words(index, s["seed"], 0x64726F70) << 16) + _exact_words(index, s["seed"], 0x64726F71)
    factor = (number >= round(case["p"] * 2 ** 32)).double() / (1.0 - case["p"])
    y = xm.double() * factor
    if case["residual"]:
        y = y + to_mem(s["residual"]).double()
    out = [back(y)]
    if case["train"]:
        out.append(back(to_mem(s["dy"]).double() * factor))
        if case["residual"]:
            out.append(s["dy"].double())
    return out


def _exact_rotary(case, s):
    """Each pair (a, b) of a token becomes (a cos - b sin, a sin + b cos) with the angle position * frequency
    of the pair's axis, as a complex product; gradients are multiplied by the conjugate."""
    grid, sections, prefix = _ints(case["grid"]), _ints(case["sections"]), case["prefix"]
    n, dev, rot = case["n"], s["q"].device, sum(sections)
    length = math.prod(grid)
    axis = torch.tensor([a for a, v in enumerate(sections) for _ in range(v // 2)], device=dev)
    inner = [j / v for v in sections for j in range(0, v, 2)] if case["spectrum"] == "axis" else [j / rot for j in range(0, rot, 2)]
    freq = torch.tensor([10000.0 ** -e for e in inner], dtype=torch.float64, device=dev)
    if "positions" in s:
        pos = s["positions"][:, prefix:].double()
    else:
        pos = torch.cartesian_prod(*[torch.arange(v, dtype=torch.float64, device=dev) for v in grid]).reshape(1, length, len(grid))
        pos = pos.repeat(n, 1, 1)
        if case["window"]:
            flipped = grid[-1] - 1 - pos[..., -1]
            pos[..., -1] = torch.where(s["flip"].view(n, 1), flipped, pos[..., -1]) + s["left"].double().view(n, 1) / case["patch"]
            pos[..., -2] += s["top"].double().view(n, 1) / case["patch"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=dev), pos[..., axis] * freq).unsqueeze(2)

    def rotate(x, phase):
        out = x.detach().double()
        v = out[:, prefix:, :, :rot]
        if case["pairing"] == "interleaved":
            pair = torch.complex(v[..., 0::2].contiguous(), v[..., 1::2].contiguous()) * phase
            v[..., 0::2], v[..., 1::2] = pair.real, pair.imag
        else:
            pair = torch.complex(v[..., :rot // 2].contiguous(), v[..., rot // 2:].contiguous()) * phase
            v[..., :rot // 2], v[..., rot // 2:] = pair.real, pair.imag
        return out

    names = ["q", "k"] if case["kv_heads"] else ["q"]
    out = [rotate(s[v], turn) for v in names]
    if case["train"]:
        out += [rotate(s["d" + v], turn.conj()) for v in names]
    return out
