"""A trainable attention block over an NHWC feature map, made of the token operators and the 1×1 convs: the pieces run
together as a model uses them.

    n = rms(x)·g1;  q, k, v = conv1×1(n);  a = attention(q, k, v);  h = x + conv1×1(a);  y = rms(h)·g2

A map of H×W pixels in NHWC is H·W tokens × C channels, so no layout changes: the 1×1 convs are the projections, their
outputs are read as heads in place, and positions enter as a distance bias |Δy| + |Δx| on the map with a slope per
head (2^(−8·(h+1)/heads)).  The residual's addition and the second norm are one pass.

    block = AttnBlock(B, H, W, C, heads)          # fp32 master weights, fp16 copies, AdamW over all of them
    h, y = block.forward(x)                       # x: (B, H, W, C) fp16, e.g. model.act("model.9")
    dx = block.backward(dy, dh)                   # gradients of y and, optionally, of h
    block.step(max_norm=10.0, grad_scale=1/scale)

`python -m objectsam_b200.attn_block` trains one on synthetic maps and prints its loss.
"""
from __future__ import annotations

import math

import torch

from .attn import AttnGeom, AttnOp
from .conv import ConvGeom, ConvOp
from .norm import rms_norm_bwd, rms_norm_fwd
from .optim import AdamW

__all__ = ["AttnBlock"]


class AttnBlock:
    PROJ = ("q", "k", "v", "out")

    def __init__(self, batch: int, height: int, width: int, channels: int, heads: int, cap: float = 0.0, eps: float = 1e-5,
                 lr: float = 1e-3, weight_decay: float = 0.01, bits: int = 32, seed: int = 0, device="cuda"):
        if channels % heads or (channels // heads) % 8 or channels // heads > 128 or channels % 32 or channels > 512:
            raise ValueError("channels are a multiple of 32 and of heads, at most 512 (the convs'); channels / heads a "
                             "multiple of 8, at most 128")
        B, H, W, C = batch, height, width, channels
        L, D = H * W, C // heads
        self.shape, self.heads, self.eps = (B, H, W, C), heads, eps
        g = torch.Generator(device="cpu").manual_seed(seed)
        sizes = {"g1": (C,), "g2": (C,)} | {n: (C, 1, 1, C) for n in self.PROJ}  # conv weights KRSC
        init = {n: torch.ones(s) if len(s) == 1 else torch.randn(s, generator=g) / math.sqrt(C) for n, s in sizes.items()}
        self.params = {n: t.to(device) for n, t in init.items()}
        self.weights = {n: self.params[n].half() for n in self.PROJ}
        f16 = lambda *s: torch.empty(*s, dtype=torch.float16, device=device)  # noqa: E731
        self.grads = {n: torch.empty(sizes[n], device=device) if n in ("g1", "g2") else f16(*sizes[n]) for n in sizes}
        names = list(sizes)
        self.opt = AdamW([self.params[n] for n in names], [self.grads[n] for n in names],
                         copies=[self.weights.get(n) for n in names], lr=lr, weight_decay=weight_decay, bits=bits,
                         decay=[n in self.weights for n in names])
        self.conv = ConvOp().init(ConvGeom(B, H, W, C, C, 1, 1, 1, 0))  # all four projections
        slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], device=device)
        self.attn = AttnOp().init(AttnGeom(B, L, L, heads, heads, D), cap=cap, grid_w=W, slopes=slopes)
        nbytes = max(self.conv.workspace_size(), self.attn.workspace_size(), 256)
        self.ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        self.n1, self.a, self.z, self.h, self.y = (f16(B, H, W, C) for _ in range(5))
        self.qkv, self.dqkv = ([f16(B, H, W, C) for _ in range(3)] for _ in range(2))
        self.rstd1, self.rstd2 = (torch.empty(B * L, device=device) for _ in range(2))
        self.lse = torch.empty(B, heads, L, device=device)
        self.dhid, self.da, self.dn1, self.dx = (f16(B, H, W, C) for _ in range(4))

    def _heads(self, t):
        """A map as (batch, tokens, heads, dim)."""
        B, H, W, C = self.shape
        return t.view(B, H * W, self.heads, C // self.heads)

    def forward(self, x, stream=None):
        """(h, y): the residual stream and its norm, both (B, H, W, C) fp16 and the block's own buffers."""
        p, w = self.params, self.weights
        self.x = x
        rms_norm_fwd(x, p["g1"], self.eps, self.n1, rstd=self.rstd1, stream=stream)
        for n, t in zip(self.PROJ, self.qkv):
            self.conv.fwd(self.n1, w[n], t, self.ws, stream=stream)
        self.attn.fwd(*map(self._heads, self.qkv), self._heads(self.a), self.lse, ws=self.ws, stream=stream)
        self.conv.fwd(self.a, w["out"], self.z, self.ws, stream=stream)
        rms_norm_fwd(self.z, p["g2"], self.eps, self.y, res=x, total=self.h, rstd=self.rstd2, stream=stream)
        return self.h, self.y

    def backward(self, dy, dh=None, stream=None):
        """dx for the gradients of y and of h; the parameters' gradients into self.grads (written)."""
        p, w, g, ws = self.params, self.weights, self.grads, self.ws
        rms_norm_bwd(dy, self.h, p["g2"], self.rstd2, self.dhid, g["g2"], dtotal=dh, stream=stream)
        self.conv.wgrad(self.a, self.dhid, g["out"], ws, stream=stream)
        self.conv.dgrad(self.dhid, w["out"], self.da, ws, stream=stream)
        self.attn.bwd(*map(self._heads, self.qkv), self._heads(self.a), self.lse, self._heads(self.da),
                      *map(self._heads, self.dqkv), ws=ws, stream=stream)
        # dn1 is summed in fp16 over the three projections (dgrad's beta): two roundings beside those of its terms, of one size
        for i, (n, d) in enumerate(zip(self.PROJ, self.dqkv)):
            self.conv.wgrad(self.n1, d, g[n], ws, stream=stream)
            self.conv.dgrad(d, w[n], self.dn1, ws, beta=float(i > 0), stream=stream)
        rms_norm_bwd(self.dn1, self.x, p["g1"], self.rstd1, self.dx, g["g1"], dtotal=self.dhid, stream=stream)
        return self.dx

    def step(self, lr=None, max_norm=None, grad_scale: float = 1.0, stream=None) -> None:
        self.opt.step(lr=lr, max_norm=max_norm, grad_scale=grad_scale, stream=stream)


def main(steps: int = 60, batch: int = 4, size: int = 20, channels: int = 256, heads: int = 4) -> list:
    """Fits a block to another one's outputs on random maps; returns the losses."""
    scale = 128.0  # of the loss, so that small gradients stay in fp16's range
    teacher = AttnBlock(batch, size, size, channels, heads, seed=1)
    block = AttnBlock(batch, size, size, channels, heads, seed=2, bits=8)
    g = torch.Generator(device="cuda").manual_seed(0)
    losses = []
    for i in range(steps):
        x = torch.randn(batch, size, size, channels, generator=g, device="cuda").half()
        want = teacher.forward(x)[1].float()
        diff = block.forward(x)[1].float() - want
        losses.append(float((diff * diff).mean()))
        block.backward((diff * (2 * scale / want[0].numel())).half())
        block.step(max_norm=1.0, grad_scale=1 / scale)
        if i % 10 == 0 or i == steps - 1:
            print(f"step {i}: loss {losses[-1]:.5f}, gradient norm {float(block.opt.norm):.4f}")
    return losses


if __name__ == "__main__":
    main()
