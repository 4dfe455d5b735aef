"""The operators in a row, as a network's first block uses them on an augmented batch: augment, convolve,
group norm + activation, dropout, patch tokens, rotary positions of the crop's patches, attention."""
import pytest
import torch

import feature_reference as R
import triton_augment_b200 as ta

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _block(images, conv, w, b, proj, top, left, flip, ops):
    """ops: (group norm, dropout, rotary) in one precision."""
    f = torch.nn.functional.conv2d(images.to(conv.dtype), conv, stride=2, padding=1)
    f = f.contiguous(memory_format=torch.channels_last)
    f = ops[1](ops[0](f, w, b))
    n, c, hh, ww = f.shape
    tok = f.unfold(2, 4, 4).unfold(3, 4, 4).permute(0, 2, 3, 1, 4, 5).reshape(n, (hh // 4) * (ww // 4), c * 16)
    q, k = (tok @ proj).view(n, tok.shape[1], 2, 2, 16).unbind(2)
    q, k = ops[2](q, k, (hh // 4, ww // 4), top, left, flip)
    return torch.einsum("nihd,njhd->nhij", q, k).softmax(-1).square().mean(), q


def test_block_against_64_bits():
    """Loss and parameter gradients of the float32 chain against the same chain in 64 bits.  The chain is
    conv, norm, attention logits of order one: float32 leaves some 1e-5 of each gradient's size; 1e-3 is asked."""
    torch.backends.cuda.matmul.allow_tf32 = torch.backends.cudnn.allow_tf32 = False
    g = torch.Generator(device=DEV).manual_seed(0)
    batch = torch.rand(4, 3, 80, 96, generator=g, device=DEV)
    top, left = torch.tensor([0., 5., 16., 9.], device=DEV), torch.tensor([3., 0., 31., 8.], device=DEV)
    flip = torch.tensor([True, False, False, True], device=DEV)
    images = ta.fused_augment(batch, top, left, 64, 64, flip, brightness_factor=1.1, mean=(0.5,) * 3, std=(0.25,) * 3)
    conv = (torch.randn(16, 3, 3, 3, generator=g, device=DEV) * 0.3).requires_grad_()
    w, b = (1 + 0.1 * torch.randn(16, generator=g, device=DEV)).requires_grad_(), (0.1 * torch.randn(16, generator=g, device=DEV)).requires_grad_()
    proj = (torch.randn(256, 64, generator=g, device=DEV) * 0.06).requires_grad_()
    leaves = (conv, w, b, proj)
    own = (lambda f, w, b: ta.group_norm(f, 4, w, b, activation="silu"),
           lambda f: ta.dropout(f, 0.1, 99, mode="channel"),
           lambda q, k, grid, t, l, fl: ta.rotary_embedding(q, k, sections=(8, 8), grid=grid, patch=8, top=t, left=l, flip_horizontal=fl))

    def gn64(f, w, b):
        v = f.reshape(f.shape[0], 4, -1)
        v = ((v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5)).reshape(f.shape)
        return torch.nn.functional.silu(v * w.view(1, -1, 1, 1) + b.view(1, -1, 1, 1))

    def drop64(f):
        keep = R.dropout_keep(tuple(f.shape), 0.1, 99, shared={2, 3}, order=(0, 2, 3, 1)).to(DEV)
        return f * keep / 0.9

    def rope64(q, k, grid, t, l, fl):
        ang = R.rotary_angles(R.grid_positions(grid, q.shape[0], 8.0, t, l, fl, device=DEV), (8, 8))[:, :, None]
        turn = lambda x: torch.stack((x[..., 0::2] * ang.cos() - x[..., 1::2] * ang.sin(), x[..., 1::2] * ang.cos() + x[..., 0::2] * ang.sin()), -1).flatten(-2)
        return turn(q), turn(k)
    loss, q = _block(images, *leaves, top, left, flip, own)
    grads = torch.autograd.grad(loss, leaves)
    leaves64 = [t.detach().double().requires_grad_() for t in leaves]
    loss64, q64 = _block(images, *leaves64, top, left, flip, (gn64, drop64, rope64))
    grads64 = torch.autograd.grad(loss64, leaves64)
    assert abs(float((loss - loss64).detach())) <= 1e-4 * abs(float(loss64))
    assert float((q - q64).abs().max()) <= 1e-4 * float(q64.abs().max())
    for got, want in zip(grads, grads64):
        assert float((got - want).norm()) <= 1e-3 * float(want.norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_in_16_bits_runs_and_repeats(dtype):
    """Same modules in 16 bits: finite gradients of every parameter, equal bits on a second run with the seed reset."""
    torch.manual_seed(1)
    norm, drop = ta.TritonGroupNorm(4, 16, activation="silu").to(DEV), ta.TritonDropout(0.2, mode="channel")
    rope = ta.TritonRotaryEmbedding((8, 8), patch=8)
    aug = ta.TritonRandomCropFlip(64)
    conv = (torch.randn(16, 3, 3, 3, device=DEV) * 0.3).to(dtype).requires_grad_()
    proj = (torch.randn(256, 64, device=DEV) * 0.06).to(dtype).requires_grad_()
    batch = torch.rand(4, 3, 80, 96, device=DEV)
    ops = (lambda f, w, b: norm(f), drop, lambda q, k, grid, t, l, fl: rope(q, k, grid=grid, top=t, left=l, flip_horizontal=fl))
    leaves = [conv, proj, norm.weight, norm.bias]
    results = []
    for _ in range(2):
        torch.manual_seed(7)
        loss, _ = _block(aug(batch), conv, norm.weight, norm.bias, proj, 4, 8, False, ops)
        results.append([loss.detach()] + list(torch.autograd.grad(loss, leaves)))
    assert all(bool(torch.isfinite(t).all()) and bool(t.any()) for t in results[0])
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][2], results[1][2])


def _calls():
    w = torch.ones(16, device="cuda")
    grid = dict(sections=(4, 4), grid=(2, 2))
    return {"group_norm": ((2, 16, 6, 6), lambda x: ta.group_norm(x, 4, w, activation="silu")),
            "dropout": ((2, 16, 6, 6), lambda x: ta.dropout(x, 0.3, 5)),
            "rotary": ((2, 4, 3, 8), lambda x: ta.rotary_embedding(x, **grid))}


@pytest.mark.parametrize("name", ["group_norm", "dropout", "rotary"])
def test_negated_views(name):
    """Tensors whose values torch keeps negated, features and gradients alike."""
    shape, f = _calls()[name]
    x, dy = torch.randn(shape, device="cuda"), torch.randn(shape, device="cuda")
    plain = (-x).requires_grad_()
    neg = torch._neg_view(x).requires_grad_()
    assert neg.is_neg()
    a, b = f(plain), f(neg)
    assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(a, plain, -dy)[0], torch.autograd.grad(b, neg, torch._neg_view(dy))[0])


@pytest.mark.parametrize("name", ["group_norm", "dropout", "rotary"])
def test_forward_mode_is_refused(name):
    import torch.autograd.forward_ad as fw
    shape, f = _calls()[name]
    with fw.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        f(fw.make_dual(torch.randn(shape, device="cuda"), torch.randn(shape, device="cuda")))


@pytest.mark.parametrize("name", ["group_norm", "dropout", "rotary"])
def test_threads_share_a_graph(name):
    """Four threads go backward through one graph, and through graphs of their own."""
    from concurrent.futures import ThreadPoolExecutor
    shape, f = _calls()[name]
    x, dy = torch.randn(shape, device="cuda").requires_grad_(), torch.randn(shape, device="cuda")
    y = f(x)
    want = torch.autograd.grad(y, x, dy, retain_graph=True)[0]
    with ThreadPoolExecutor(4) as pool:
        got = list(pool.map(lambda i: torch.autograd.grad(y if i % 2 else f(x), x, dy, retain_graph=True)[0], range(32)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
