"""AdamW over many tensors in one launch on the C ABI (osam_adamw_* in include/osam.h give the formulas).

    opt = AdamW(params, grads, copies=weights_fp16, lr=1e-3, weight_decay=0.05, bits=8, decay=[t.dim() > 1 for t in params])
    opt.step(max_norm=10.0, grad_scale=1 / loss_scale)

params: contiguous float32 CUDA tensors; grads: float32, float16 or bfloat16, one per parameter (views of a gradient
arena will do, unaligned ones too); copies: 16-bit tensors that receive the new parameters (operands of convs that
take their weights from the caller, as attn_block.py's do), None where a parameter has none.  The tensors' memory is read at every step and must stay in place.
States: opt.m, opt.v (float32, or float8_e4m3fn with opt.m_scale, opt.v_scale per 256 elements, where v holds √v).
opt.norm: the gradients' norm of the last step with max_norm.  A captured step replays with its capture's count and rate.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import AdamWTensor, check, lib, stream_ptr

__all__ = ["AdamW"]

_TYPE = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


class AdamW:
    def __init__(self, params: Sequence, grads: Sequence, copies: Optional[Sequence] = None, lr: float = 1e-3,
                 betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, bits: int = 32,
                 decay: Optional[Sequence[bool]] = None, step: int = 0, stream=None):
        n = len(params)
        self._plan = ctypes.c_void_p()
        if not n:
            raise ValueError("no parameters")
        copies = [None] * n if copies is None else list(copies)
        decay = [True] * n if decay is None else list(decay)
        if not n == len(grads) == len(copies) == len(decay):
            raise ValueError("one gradient, copy and decay flag for each parameter")
        tab = (AdamWTensor * n)()
        dev = params[0].device
        for i, (p, g, c) in enumerate(zip(params, grads, copies)):
            for t, name, types in ((p, "parameter", (torch.float32,)), (g, "gradient", tuple(_TYPE)),
                                   (c, "copy", (torch.float16, torch.bfloat16))):
                if t is not None and (t.dtype not in types or t.numel() != p.numel() or not t.is_contiguous() or
                                      not t.is_cuda or t.device != dev):
                    raise ValueError(f"{name} {i}: a contiguous CUDA tensor of {p.numel()} elements, one of {types}")
            tab[i] = AdamWTensor(p.data_ptr(), g.data_ptr(), None if c is None else c.data_ptr(), p.numel(),
                                 _TYPE[g.dtype], _lib.F16 if c is None else _TYPE[c.dtype], int(bool(decay[i])))
        nbytes, elems = ctypes.c_size_t(), ctypes.c_int64()
        check(lib().osam_adamw_sizes(tab, n, bits, ctypes.byref(nbytes), ctypes.byref(elems)))
        self._keep = (list(params), list(grads), copies)
        self.bits, self.steps = bits, int(step)
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        s = stream if stream is not None else torch.cuda.current_stream(dev)
        with torch.cuda.stream(s):
            self._table = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
            kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
            self.m, self.v = (torch.zeros(elems.value, dtype=torch.float32 if bits == 32 else torch.uint8,
                                          device=dev).view(kind) for _ in range(2))
            self.m_scale, self.v_scale = ((torch.zeros(elems.value // 256, device=dev) for _ in range(2))
                                          if bits == 8 else (None, None))
            self.norm = torch.zeros(1, device=dev)
        check(lib().osam_adamw_create(tab, n, bits, self._table.data_ptr(), nbytes.value, s.cuda_stream,
                                      ctypes.byref(self._plan)))
        self._scales = (None, None) if bits == 32 else (self.m_scale.data_ptr(), self.v_scale.data_ptr())
        self._streams = {s.cuda_stream}  # that the allocator knows to use the optimizer's own tensors

    def close(self) -> None:
        if self._plan:
            lib().osam_adamw_destroy(self._plan)
            self._plan = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def load_state(self, m, v, m_scale=None, v_scale=None, step: Optional[int] = None) -> None:
        """Copies saved states (of this layout) in."""
        for to, src in ((self.m, m), (self.v, v), (self.m_scale, m_scale), (self.v_scale, v_scale)):
            if (to is None) != (src is None):
                raise ValueError("8-bit states come with their scales")
            if to is not None:
                if src.dtype != to.dtype or src.numel() != to.numel():
                    raise ValueError(f"state: {to.numel()} elements of {to.dtype} expected")
                to.copy_(src.reshape(-1))
        if step is not None:
            self.steps = int(step)

    def step(self, lr: Optional[float] = None, max_norm: Optional[float] = None, grad_scale: float = 1.0,
             stream=None) -> None:
        """One step; with max_norm the gradients (times grad_scale) are clipped to that norm, and a norm that is
        not finite leaves everything but the step count as it was."""
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm is positive")
        st = stream_ptr(stream)
        if st not in self._streams:
            s = stream if stream is not None else torch.cuda.current_stream()
            for t in (self._table, self.m, self.v, self.m_scale, self.v_scale, self.norm):
                if t is not None:
                    t.record_stream(s)
            self._streams.add(st)
        check(lib().osam_adamw_step(self._plan, self.m.data_ptr(), self.v.data_ptr(), *self._scales, self.steps + 1,
                                    self.lr if lr is None else lr, self.betas[0], self.betas[1], self.eps,
                                    self.weight_decay, grad_scale, max_norm or 0.0, self.norm.data_ptr(), st))
        self.steps += 1
