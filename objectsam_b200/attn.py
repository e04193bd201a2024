"""Attention over tokens on the C ABI: capped scores, a distance bias, document / prefix / causal masks, forward,
backward, and single tokens over a long cache (osam_attn_fwd / osam_attn_bwd in include/osam.h give the formulas).

    op = AttnOp().init(AttnGeom(B, H*W, H*W, heads, heads, dim, torch.float16), grid_w=W, slopes=slopes)
    ws = torch.empty(op.workspace_size(), dtype=torch.uint8, device="cuda")
    op.fwd(q, k, v, o, lse, ws=ws)
    op.bwd(q, k, v, o, lse, do, dq, dk, dv, ws=ws)

Tensors are (batch, tokens, heads, dim) CUDA tensors of the plan's type with dim contiguous: slices of a fused
projection (batch, tokens, (q, k, v) heads, dim) and of a cache are taken as they lie.  slopes, lens, prefix and
the document ids are device tensors that the plan keeps and every call reads anew.  Without `ws` the plan makes
one per device and stream and keeps it.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._lib import AttnDesc, View, check, lib, stream_ptr

__all__ = ["AttnGeom", "AttnOp"]

_DTYPE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_MASK = {"none": _lib.ATTN_NONE, "causal": _lib.ATTN_CAUSAL, "prefix": _lib.ATTN_PREFIX}


@dataclass(frozen=True)
class AttnGeom:
    batch: int
    len_q: int
    len_k: int
    heads_q: int
    heads_k: int
    dim: int
    dtype: torch.dtype = torch.float16


class AttnOp:
    def __init__(self):
        self._d: Optional[AttnDesc] = None

    def init(self, g: AttnGeom, scale: Optional[float] = None, cap: float = 0.0, mask: str = "none", grid_w: int = 0,
             slopes=None, lens=None, prefix=None, doc_q=None, doc_k=None) -> "AttnOp":
        """scale: 1/√dim unless given.  lens, prefix: int32 (batch,); slopes: float32 (heads_q,); doc_q (batch, len_q)
        and doc_k (batch, len_k): int32."""
        if g.dtype not in _DTYPE:
            raise ValueError("attention takes float16 or bfloat16")
        if cap > 0 and not ctypes.c_float(cap).value:
            raise ValueError("cap is below float32's range: it would be taken as none")
        if mask not in _MASK:
            raise ValueError(f"mask is one of {sorted(_MASK)}")
        for name, t, dtype, shape in (("slopes", slopes, torch.float32, (g.heads_q,)),
                                      ("lens", lens, torch.int32, (g.batch,)),
                                      ("prefix", prefix, torch.int32, (g.batch,)),
                                      ("doc_q", doc_q, torch.int32, (g.batch, g.len_q)),
                                      ("doc_k", doc_k, torch.int32, (g.batch, g.len_k))):
            if t is not None and (t.dtype != dtype or tuple(t.shape) != shape or not t.is_cuda or not t.is_contiguous()):
                raise ValueError(f"{name}: contiguous CUDA {dtype} of shape {shape} expected")
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        d = AttnDesc(_DTYPE[g.dtype], g.batch, g.len_q, g.len_k, g.heads_q, g.heads_k, g.dim, _MASK[mask],
                     1.0 / math.sqrt(max(g.dim, 1)) if scale is None else scale, cap, grid_w, p(slopes), p(lens),
                     p(prefix), p(doc_q), p(doc_k))
        self._ws_bytes = int(lib().osam_attn_workspace_size(ctypes.byref(d)))
        if not self._ws_bytes:  # refused, unless there are no queries (and this call does nothing)
            check(lib().osam_attn_fwd(ctypes.byref(d), View(), View(), View(), View(), None, None, 0, None))
        self._keep = (slopes, lens, prefix, doc_q, doc_k)
        self._g, self._d, self._ref, self._ws = g, d, ctypes.byref(d), {}
        self._dtype = g.dtype
        self._q = torch.Size((g.batch, g.len_q, g.heads_q, g.dim))
        self._k = torch.Size((g.batch, g.len_k, g.heads_k, g.dim))
        return self

    def geom(self) -> AttnGeom:
        return self._g

    def workspace_size(self) -> int:
        return self._ws_bytes

    tune = workspace_size  # as ConvOp.tune: nothing is timed

    def _view(self, t, shape, name: str) -> View:
        if t.dtype is not self._dtype or t.shape != shape or not t.is_cuda:
            raise ValueError(f"{name}: CUDA {self._dtype} of shape {tuple(shape)} expected")
        sb, st, sh, sd = t.stride()
        if sd != 1 and shape[3] > 1:
            raise ValueError(f"{name}: the head dimension is contiguous")
        return View(t.data_ptr(), sb, st, sh)

    def _workspace(self, ws, stream):
        if ws is None:
            s = stream if stream is not None else torch.cuda.current_stream()
            key = s.device.index, s.cuda_stream  # the default stream's handle is 0 on every device
            ws = self._ws.get(key)
            if ws is None:
                with torch.cuda.stream(s):
                    ws = self._ws[key] = torch.empty(max(self._ws_bytes, 256), dtype=torch.uint8, device=s.device)
        elif not ws.is_cuda or not ws.is_contiguous():
            raise ValueError("workspace: a contiguous CUDA tensor expected")
        return ws.data_ptr(), ws.numel() * ws.element_size()

    def _lse(self, lse):
        if lse.dtype != torch.float32 or lse.numel() != self._g.batch * self._g.heads_q * self._g.len_q or \
                not lse.is_contiguous() or not lse.is_cuda:
            raise ValueError("lse: contiguous CUDA float32 (batch, heads_q, len_q) expected")
        return lse.data_ptr()

    def fwd(self, q, k, v, o, lse=None, ws=None, stream=None) -> None:
        """o (and lse, float32 (batch, heads_q, len_q)) ← attention of q over k, v."""
        w, n = self._workspace(ws, stream)
        check(lib().osam_attn_fwd(self._ref, self._view(q, self._q, "q"), self._view(k, self._k, "k"),
                                  self._view(v, self._k, "v"), self._view(o, self._q, "o"),
                                  None if lse is None else self._lse(lse), w, n, stream_ptr(stream)))

    def bwd(self, q, k, v, o, lse, do, dq, dk, dv, ws=None, stream=None) -> None:
        """dq, dk, dv ← gradients for do, the gradient of o; o and lse are the forward's."""
        w, n = self._workspace(ws, stream)
        check(lib().osam_attn_bwd(self._ref, self._view(q, self._q, "q"), self._view(k, self._k, "k"),
                                  self._view(v, self._k, "v"), self._view(o, self._q, "o"), self._lse(lse),
                                  self._view(do, self._q, "do"), self._view(dq, self._q, "dq"),
                                  self._view(dk, self._k, "dk"), self._view(dv, self._k, "dv"), w, n,
                                  stream_ptr(stream)))
