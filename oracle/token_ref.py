"""CPU/torch restatements in 64 bits of the token operators (test infrastructure): attention with its masks and
gradients, the RMS norm, the AdamW step.  Written from the formulas in include/osam.h; every function takes and
returns float64 tensors unless it says otherwise."""
from __future__ import annotations

import math

import torch


def attn_visible(batch, len_q, len_k, mask="none", lens=None, prefix=None, doc_q=None, doc_k=None):
    """bool [batch][len_q][len_k]: which keys each query sees."""
    out = torch.zeros(batch, len_q, len_k, dtype=torch.bool)
    for b in range(batch):
        n = len_k if lens is None else max(0, min(len_k, int(lens[b])))
        for i in range(len_q):
            pos = i + n - len_q
            end = n
            if mask == "causal":
                end = min(n, pos + 1)
            elif mask == "prefix":
                end = min(n, max(pos + 1, int(prefix[b])))
            out[b, i, :max(0, end)] = True
    if doc_q is not None:
        dq, dk = doc_q.cpu(), doc_k.cpu()
        out &= (dq[:, :, None] == dk[:, None, :]) & (dq[:, :, None] >= 0)
    return out


def attn_distance(batch, len_q, len_k, grid_w=0, lens=None):
    """[batch][len_q][len_k] distances of query and key positions."""
    j = torch.arange(len_k)
    out = torch.zeros(batch, len_q, len_k, dtype=torch.float64)
    for b in range(batch):
        n = len_k if lens is None else max(0, min(len_k, int(lens[b])))
        i = torch.arange(len_q) + n - len_q
        if grid_w:
            fl = lambda t: torch.div(t, grid_w, rounding_mode="floor")  # noqa: E731
            out[b] = ((fl(i)[:, None] - fl(j)).abs() + ((i - fl(i) * grid_w)[:, None] - (j - fl(j) * grid_w)).abs())
        else:
            out[b] = (i[:, None] - j).abs()
    return out


def attention(q, k, v, visible, scale, cap=0.0, slopes=None, distance=None, do=None, unit=0.0):
    """q [B][Lq][Hq][D], k, v [B][Lk][Hk][D] → dict(o, lse [B][Hq][Lq], score_max) and, with do, dq, dk, dv.  Hidden
    keys' contents are not used.  With `unit` (a 16-bit type's rounding unit u) also, for each output x, `tol_x`: how
    far it may be when P, dS, o and the outputs are rounded to that type once each and all else is exact:
      |Δo|  ≤ u·Σ p|v| + u|o|              |Δdv| ≤ u·Σ_i p|do| + u|dv|
      |Δds| ≤ u|ds| + p·(1−t²)·u·Σ|o||do|   (the rounded o enters δ)
      |Δdq| ≤ scale·Σ_j |Δds||k| + u|dq|,  dk likewise."""
    B, Lq, Hq, D = q.shape
    Hk = k.shape[2]
    G = Hq // Hk
    see = visible.to(q.device)[:, None]
    kk, vv = (t.permute(0, 2, 1, 3).repeat_interleave(G, 1) for t in (k, v))
    seen = see.any(2)[:, 0]  # keys that some query sees
    kk, vv = (torch.where(seen[:, None, :, None], t, 0.0) for t in (kk, vv))
    qq = torch.where(see.any(3)[:, 0, :, None, None], q, 0.0).permute(0, 2, 1, 3)
    s = scale * qq @ kk.transpose(2, 3)
    t = torch.tanh(s / cap) if cap else torch.zeros_like(s)
    x = cap * t if cap else s
    if slopes is not None:
        x = x - slopes.to(q)[None, :, None, None] * distance.to(q)[:, None]
    x = x.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(x, 3)
    p = torch.where(see, torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
    o = p @ vv
    back = lambda a: a.permute(0, 2, 1, 3)  # noqa: E731
    group = lambda a: a.reshape(B, Hk, G, *a.shape[2:]).sum(2)  # noqa: E731
    out = {"o": back(o), "lse": lse, "tol_o": back(unit * (p @ vv.abs()) + unit * o.abs()),
           "score_sum": (scale * qq.abs() @ kk.abs().transpose(2, 3)).amax() if Lq and k.shape[1] else 0.0}
    if do is None:
        return out
    g = torch.where(see.any(3)[:, 0, :, None, None], do, 0.0).permute(0, 2, 1, 3)
    dv = p.transpose(2, 3) @ g
    dp = g @ vv.transpose(2, 3)
    ds = p * (dp - (g * o).sum(3, keepdim=True)) * (1 - t * t)
    eds = unit * ds.abs() + p * (1 - t * t) * unit * (g * o).abs().sum(3, keepdim=True)
    dq, dk = scale * ds @ kk, scale * ds.transpose(2, 3) @ qq
    out |= {"dq": back(dq), "dk": back(group(dk)), "dv": back(group(dv))}
    out["tol_dq"] = back(scale * eds @ kk.abs() + unit * dq.abs())
    out["tol_dk"] = back(group(scale * eds.transpose(2, 3) @ qq.abs()) + unit * group(dk).abs())
    out["tol_dv"] = back(group(unit * (p.transpose(2, 3) @ g.abs())) + unit * group(dv).abs())
    return out


def rms_norm(x, w, eps, res=None, dy=None, dtotal=None, stored=None):
    """x [rows][C] → dict(h, rstd, y) and, with dy, dx and dw from the stored total (h as the forward rounded it)."""
    h = x if res is None else x + res
    rstd = 1 / torch.sqrt((h * h).mean(1) + eps)
    out = {"h": h, "rstd": rstd, "y": h * rstd[:, None] * w}
    if dy is not None:
        hs = h if stored is None else stored
        n = hs * rstd[:, None]
        c = (dy * w * n).mean(1, keepdim=True)
        out["dx"] = rstd[:, None] * (dy * w - n * c) + (0 if dtotal is None else dtotal)
        out["dw"] = (dy * n).sum(0)
    return out


def adamw(p, g, m, v, t, lr, betas, eps, weight_decay, mul=1.0, decay=True):
    """New (p, m, v) of one step (t counts from 1)."""
    b1, b2 = betas
    g = g * mul
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    step = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p * (1 - lr * weight_decay * bool(decay)) - lr * step, m, v
