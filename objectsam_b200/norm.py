"""RMS norm over the channels of each row with the residual's addition, in 16 bits or e4m3 with a scale per 128
channels, and its backward pass, on the C ABI (osam_rms_* in include/osam.h give the formulas).

    rms_norm_fwd(x, w, eps, y, res=r, total=h, rstd=rstd)         # h = x + r, y = h·rstd·w
    rms_norm_fwd_q8(x, w, eps, q, qscale, res=r, total=h)         # y ≈ q·qscale[:, channel // 128]
    rms_norm_bwd(dy, h, w, rstd, dx, dw, dtotal=dh)               # dx = dh + the norm's gradient

Any leading shape: an NHWC map (N, H, W, C) is N·H·W rows.  A tensor may be a channel slice of a wider buffer (its
rows equally spaced); w, dw and rstd are float32 and contiguous.  total may be x or res.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check, lib, stream_ptr

__all__ = ["rms_norm_fwd", "rms_norm_fwd_q8", "rms_norm_bwd", "workspace", "GROUP"]

GROUP = 128  # channels that share an e4m3 scale
_DTYPE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_ws_cache: dict = {}


def _rows(t, shape, dtype, name: str):
    """(pointer, elements from row to row) of a tensor whose leading dimensions are equally spaced rows."""
    if t.dtype is not dtype or t.shape != shape or not t.is_cuda:
        raise ValueError(f"{name}: CUDA {dtype} of shape {tuple(shape)} expected")
    if t.is_contiguous():
        return t.data_ptr(), shape[-1]
    stride = t.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}: channels are contiguous")
    ld, n = None, 1
    for size, step in zip(shape[-2::-1], stride[-2::-1]):
        if size == 1:
            continue
        if ld is None:
            ld, n = step, size
            if ld < shape[-1]:  # a row repeated by broadcasting, too: stride 0
                raise ValueError(f"{name}: rows do not overlap")
        elif step != ld * n:
            raise ValueError(f"{name}: rows are equally spaced")
        else:
            n *= size
    return t.data_ptr(), shape[-1] if ld is None else ld


def _f32(t, n: int, name: str):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.numel() != n or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"{name}: contiguous CUDA float32 of {n} elements expected")
    return t.data_ptr()


def _in(x):
    """(type code, type, shape, channels, rows)"""
    dtype, shape = x.dtype, x.shape
    code = _DTYPE.get(dtype)
    if code is None:
        raise ValueError("rms norm takes float16 or bfloat16")
    C = shape[-1]
    return code, dtype, shape, C, x.numel() // max(C, 1)


def rms_norm_fwd(x, w, eps: float, y, res=None, total=None, rstd=None, stream=None) -> None:
    code, dtype, shape, C, rows = _in(x)
    r = (None, 0) if res is None else _rows(res, shape, dtype, "res")
    t = (None, 0) if total is None else _rows(total, shape, dtype, "total")
    check(lib().osam_rms_fwd(code, *_rows(x, shape, dtype, "x"), *r, _f32(w, C, "w"), rows, C, eps, *t,
                             *_rows(y, shape, dtype, "y"), _f32(rstd, rows, "rstd"), stream_ptr(stream)))


def rms_norm_fwd_q8(x, w, eps: float, q, qscale, res=None, total=None, rstd=None, stream=None) -> None:
    """q: float8_e4m3fn like x; qscale: float32 (rows, ⌈C/128⌉)."""
    code, dtype, shape, C, rows = _in(x)
    r = (None, 0) if res is None else _rows(res, shape, dtype, "res")
    t = (None, 0) if total is None else _rows(total, shape, dtype, "total")
    check(lib().osam_rms_fwd_q8(code, *_rows(x, shape, dtype, "x"), *r, _f32(w, C, "w"), rows, C, eps, *t,
                                *_rows(q, shape, torch.float8_e4m3fn, "q"), _f32(qscale, rows * -(-C // GROUP), "qscale"),
                                _f32(rstd, rows, "rstd"), stream_ptr(stream)))


def workspace(C: int, device, stream=None) -> torch.Tensor:
    """The backward's workspace for C channels, one per (device, stream, size).  None is ever replaced: a captured graph may
    hold its address."""
    dev = torch.device(device)
    s = stream if stream is not None else torch.cuda.current_stream(dev)
    nbytes = max(int(lib().osam_rms_bwd_workspace_size(C)), 1 << 20)
    key = (dev.index, s.cuda_stream, nbytes)
    buf = _ws_cache.get(key)
    if buf is None:
        with torch.cuda.stream(s):
            buf = _ws_cache[key] = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return buf


def rms_norm_bwd(dy, h, w, rstd, dx, dw, dtotal=None, ws=None, stream=None) -> None:
    """h: the forward's total (its x where there was no residual); dtotal: the gradient that reaches h by the
    residual path."""
    code, dtype, shape, C, rows = _in(dy)
    d = (None, 0) if dtotal is None else _rows(dtotal, shape, dtype, "dtotal")
    if ws is None:
        ws = workspace(C, dy.device, stream)
    elif not ws.is_cuda or not ws.is_contiguous():
        raise ValueError("ws: a contiguous CUDA tensor expected")
    check(lib().osam_rms_bwd(code, *_rows(dy, shape, dtype, "dy"), *_rows(h, shape, dtype, "h"), _f32(w, C, "w"),
                             _f32(rstd, rows, "rstd"), *d, rows, C, *_rows(dx, shape, dtype, "dx"), _f32(dw, C, "dw"),
                             ws.data_ptr(), ws.numel() * ws.element_size(), stream_ptr(stream)))
