"""The attention block of attn_block.py: forward and backward through the norms, the 1×1 convs and attention against the
same graph in torch in 64 bits, and a short training run.

Tolerance: every tensor between two operators is rounded to fp16 once (2^-11 relative to its size, at most six deep, each
passed on with a gain of order one by norms and projections), so a relative 2-norm error of 6·2^-11·2 ≈ 0.6 % bounds
the outputs; the gradients pass as many again: 1.2 %."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(block, x, dy, dh):
    B, H, W, C = block.shape
    heads, L, D = block.heads, H * W, C // block.heads
    p = {n: (block.weights[n] if n in block.weights else block.params[n]).double().requires_grad_(True) for n in block.params}
    x = x.double().requires_grad_(True)
    rms = lambda t, g: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + block.eps) * g  # noqa: E731
    n = rms(x, p["g1"]).reshape(B, L, C)
    q, k, v = ((n @ p[m].reshape(C, C).T).view(B, L, heads, D).transpose(1, 2) for m in "qkv")
    i = torch.arange(L, device=x.device)
    far = (i[:, None] // W - i // W).abs() + (i[:, None] % W - i % W).abs()
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device=x.device, dtype=torch.float64)
    s = q @ k.transpose(2, 3) / math.sqrt(D) - slopes[None, :, None, None] * far
    a = (torch.softmax(s, 3) @ v).transpose(1, 2).reshape(B, L, C)
    h = x + (a @ p["out"].reshape(C, C).T).view(B, H, W, C)
    y = rms(h, p["g2"])
    ((y * dy.double()).sum() + (h * dh.double()).sum()).backward()
    return h.detach(), y.detach(), x.grad, {n: t.grad for n, t in p.items()}


@pytest.mark.parametrize("B,H,W,C,heads", [(2, 20, 20, 512, 8), (1, 13, 9, 128, 4), (3, 8, 5, 64, 1)])
def test_block(cuda_lib, B, H, W, C, heads):
    from objectsam_b200.attn_block import AttnBlock
    block = AttnBlock(B, H, W, C, heads, seed=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy, dh = (torch.randn(B, H, W, C, generator=g, device="cuda").half() for _ in range(3))
    h, y = block.forward(x)
    dx = block.backward(dy, dh)
    rh, ry, rdx, rg = reference(block, x, dy, dh)
    far = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert far(h, rh) < 0.006 and far(y, ry) < 0.006
    assert far(dx, rdx) < 0.012
    for n in rg:
        assert far(block.grads[n], rg[n].reshape(block.grads[n].shape)) < 0.012, n


def test_training_brings_the_loss_down(cuda_lib):
    from objectsam_b200.attn_block import main
    losses = main(steps=60)
    assert all(math.isfinite(v) for v in losses) and losses[-1] < 0.6 * losses[0], (losses[0], losses[-1])


def test_refusals(cuda_lib):
    from objectsam_b200.attn_block import AttnBlock
    for C, heads in ((100, 4), (256, 3), (512, 2), (48, 4), (1024, 8)):
        with pytest.raises(ValueError):
            AttnBlock(1, 4, 4, C, heads)
