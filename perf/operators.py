"""The token-mixing and optimizer operators as measured work: attention (capped scores, distance bias, document /
prefix / causal masks), the RMS norm with the residual's addition, and the AdamW step over many tensors.

`own` false: every pass in its plain form, elementary torch operations in 32 bits, rounded once at the end.
`own` true: the calls a user makes of objectsam_b200.  Both take the same state and return the same outputs.
"""
import itertools
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the 20x20 map of 640-pixel images (stride 32, 512 channels = 8 heads of 64), inference, batch 16
        dict(name="attn_map20", op="attn", dir="fwd", batch=16, lq=400, lk=400, hq=8, hk=8, dim=64, type="f16",
             mask="none", cap=0.0, bias="grid", width=20, doc=0, pad=0),
        # the 40x40 map (stride 16, 256 channels = 4 heads of 64), a training step's forward and backward
        dict(name="attn_map40_train", op="attn", dir="train", batch=8, lq=1600, lk=1600, hq=4, hk=4, dim=64,
             type="f16", mask="none", cap=0.0, bias="grid", width=40, doc=0, pad=0),
        # long packed sequences: documents of uneven lengths and a padded end, shared key heads, capped scores
        dict(name="attn_packed_train", op="attn", dir="train", batch=2, lq=4096, lk=4096, hq=16, hk=4, dim=128,
             type="bf16", mask="causal", cap=30.0, bias="none", width=0, doc=2500, pad=57),
        # one long prompt with a prefix that sees itself both ways, odd length, distance bias
        dict(name="attn_prefix", op="attn", dir="fwd", batch=1, lq=8191, lk=8191, hq=8, hk=2, dim=64, type="bf16",
             mask="prefix", cap=0.0, bias="line", width=0, doc=0, pad=0),
        # a single new token over a short cache: the latency of a call
        dict(name="attn_token", op="attn", dir="fwd", batch=1, lq=1, lk=517, hq=8, hk=8, dim=64, type="f16",
             mask="causal", cap=0.0, bias="line", width=0, doc=0, pad=0),
        # single new tokens of 16 sequences over long caches of uneven lengths, shared key heads
        dict(name="attn_token_long", op="attn", dir="fwd", batch=16, lq=1, lk=32768, hq=32, hk=8, dim=128,
             type="bf16", mask="causal", cap=50.0, bias="none", width=0, doc=0, pad=0),
        # norm and residual in front of one 20x20 map's attention: the latency of a call
        dict(name="rms_map20", op="rms", dir="fwd", rows=400, cols=512, type="f16", res=True),
        # the same for a training batch of 40x40 maps, forward and backward
        dict(name="rms_train", op="rms", dir="train", rows=25600, cols=256, type="f16", res=True),
        # wide rows into 8 bits with a scale per 128 channels
        dict(name="rms_q8", op="rms", dir="q8", rows=16397, cols=4096, type="bf16", res=True),
        # this network's own parameters: 32-bit states, fp16 weight copies, clipped to a norm of 10
        dict(name="adamw_model", op="adamw", net=True, tensors=0, largest=0, bits=32, grad="f32", copy="f16",
             clip=10.0, packed=False),
        # many small and odd tensors that lie in one array without gaps, 8-bit states
        dict(name="adamw_small", op="adamw", net=False, tensors=61, largest=5003, bits=8, grad="f32", copy="f16",
             clip=0.0, packed=True),
        # large matrices with 8-bit states and 16-bit gradients
        dict(name="adamw_large", op="adamw", net=False, tensors=24, largest=20_000_000, bits=8, grad="bf16",
             copy="bf16", clip=1.0, packed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["map", "packed", "prefix", "token", "token", "rms", "rms", "rms", "adamw", "adamw", "adamw"])
    t = rng.choice(["f16", "bf16"])
    heads = rng.choice([(8, 8), (4, 4), (3, 1), (8, 2), (6, 2), (16, 4), (5, 5)])
    dim = rng.choice([32, 40, 64, 64, 80, 128])
    cap = rng.choice([0.0, 0.0, 20.0, 50.0])
    if kind == "map":
        w, h = _log(rng, 5, 48), _log(rng, 5, 48)
        most = max(1, 100_000_000 // (heads[0] * (w * h) ** 2))
        return dict(op="attn", dir=rng.choice(["fwd", "train"]), batch=rng.randint(1, min(8, most)), lq=w * h, lk=w * h,
                    hq=heads[0], hk=heads[1], dim=dim, type=t, mask="none", cap=cap,
                    bias=rng.choice(["none", "grid", "grid"]), width=w, doc=0, pad=0)
    if kind == "packed":
        n = 5 * _log(rng, 60, 819)
        return dict(op="attn", dir=rng.choice(["fwd", "train"]), batch=rng.randint(1, 2), lq=n, lk=n, hq=heads[0],
                    hk=heads[1], dim=dim, type=t, mask=rng.choice(["none", "causal"]), cap=cap,
                    bias=rng.choice(["none", "line"]), width=0, doc=_log(rng, 60, 1500),
                    pad=rng.choice([0, rng.randint(1, 200)]))
    if kind == "prefix":
        n = 5 * _log(rng, 40, 1200)
        return dict(op="attn", dir=rng.choice(["fwd", "train"]) if n < 2000 else "fwd", batch=rng.randint(1, 2),
                    lq=n, lk=n, hq=heads[0], hk=heads[1], dim=dim, type=t, mask="prefix", cap=cap,
                    bias=rng.choice(["none", "line"]), width=0, doc=0, pad=0)
    if kind == "token":
        n = 5 * _log(rng, 13, 6553)
        return dict(op="attn", dir="fwd", batch=_log(rng, 1, 16), lq=rng.choice([1, 1, 1, 2, 5]), lk=n, hq=heads[0],
                    hk=heads[1], dim=dim, type=t, mask="causal", cap=cap, bias=rng.choice(["none", "line"]), width=0,
                    doc=0, pad=0)
    if kind == "rms":
        cols = 8 * (2 * _log(rng, 2, 350) + 1)
        return dict(op="rms", dir=rng.choice(["fwd", "train", "q8"]), rows=_log(rng, 1, min(200_000, 60_000_000 // cols)),
                    cols=cols, type=t, res=rng.random() < 0.7)
    largest = _log(rng, 300, 8_000_000)
    return dict(op="adamw", net=False, tensors=_log(rng, 3, 200 if largest < 100_000 else 20), largest=largest,
                bits=rng.choice([8, 32]), grad=rng.choice(["f32", "f16", "bf16"]),
                copy=rng.choice(["none", "f16", "bf16"]), clip=rng.choice([0.0, 1.0]), packed=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------ attention
def _docs(c):
    """Document ids [batch][lk] of a packed case: uneven documents, the last `pad` tokens belong to none (-1)."""
    r = random.Random(c["lk"] * 31 + c["doc"])
    out = np.full((c["batch"], c["lk"]), -1, np.int32)
    for b in range(c["batch"]):
        at, d = 0, 0
        while at < c["lk"] - c["pad"]:
            n = min(r.randint(max(1, c["doc"] // 2), c["doc"] * 3 // 2), c["lk"] - c["pad"] - at)
            out[b, at:at + n] = d
            at, d = at + n, d + 1
    return out


def _lens(c):
    """Keys in use of each sequence's cache (single tokens): between a quarter of the cache and all of it."""
    r = random.Random(c["lk"] * 7 + c["batch"])
    return np.array([c["lk"]] + [max(c["lq"], r.randint(c["lk"] // 4, c["lk"])) for _ in range(c["batch"] - 1)], np.int32)


def _prefix(c):
    return np.array([(b + 1) * c["lk"] // (3 * c["batch"]) for b in range(c["batch"])], np.int32)


def _serving(c):
    return c["lq"] != c["lk"]


def _pairs(c):
    """Visible (query, key) pairs of one head, over the batch."""
    lens = _lens(c) if _serving(c) else np.full(c["batch"], c["lk"])
    prefix = _prefix(c) if c["mask"] == "prefix" else np.zeros(c["batch"], np.int64)
    docs = _docs(c) if c["doc"] else None
    n = 0
    for b in range(c["batch"]):
        i = np.arange(c["lq"], dtype=np.int64)
        end = np.full(c["lq"], lens[b], np.int64)
        if c["mask"] != "none":
            end = np.minimum(end, np.maximum(i + lens[b] - c["lq"] + 1, prefix[b]))
        if docs is None:
            n += int(end.sum())
            continue
        at = np.flatnonzero(np.diff(docs[b], prepend=-9))
        first = np.zeros(c["lk"], np.int64)
        first[at] = at
        first = np.maximum.accumulate(first)
        last = np.append(at[1:], c["lk"])[np.searchsorted(at, i, side="right") - 1]
        n += int((np.maximum(0, np.minimum(end, last) - first) * (docs[b] >= 0)).sum())
    return n


def _prepare_attn(c, g):
    B, Lq, Lk, Hq, Hk, D, t = c["batch"], c["lq"], c["lk"], c["hq"], c["hk"], c["dim"], TYPES[c["type"]]
    s = {"c": c, "scale": 1 / math.sqrt(D)}

    def rnd(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=t) if by == 1.0
                else (torch.randn(*shape, generator=g, device=DEV) * by).to(t))

    if _serving(c):  # the new tokens' queries, and caches [batch][tokens][heads][dim]
        s["q"] = rnd(B, Lq, Hq, D, by=2.0)
        s["k"], s["v"] = rnd(B, Lk, Hk, D), rnd(B, Lk, Hk, D)
        s["lens"] = torch.from_numpy(_lens(c)).to(DEV)
    else:  # one projection's output [batch][tokens][(queries, keys, values) heads][dim]
        qkv = rnd(B, Lq, Hq + 2 * Hk, D)
        qkv[:, :, :Hq] *= 2
        s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
    if c["bias"] != "none":
        s["slopes"] = torch.tensor([2.0 ** (-6.0 * (h + 1) / Hq) * (0.25 if c["bias"] == "line" else 1.0)
                                    for h in range(Hq)], device=DEV)
    if c["mask"] == "prefix":
        s["prefix"] = torch.from_numpy(_prefix(c)).to(DEV)
    if c["doc"]:
        s["doc"] = torch.from_numpy(_docs(c)).to(DEV)
    if c["dir"] == "train":
        s["do"] = rnd(B, Lq, Hq, D)
    if own:  # the plan, its workspace and the output buffers that a program keeps
        from objectsam_b200.attn import AttnGeom, AttnOp
        s["op"] = AttnOp().init(AttnGeom(B, Lq, Lk, Hq, Hk, D, t), scale=s["scale"], cap=c["cap"], mask=c["mask"],
                                grid_w=c["width"] if c["bias"] == "grid" else 0, slopes=s.get("slopes"),
                                lens=s.get("lens"), prefix=s.get("prefix"), doc_q=s.get("doc"), doc_k=s.get("doc"))
        s["ws"] = torch.empty(s["op"].workspace_size(), dtype=torch.uint8, device=DEV)
        s["o"] = torch.empty(B, Lq, Hq, D, dtype=t, device=DEV)
        if c["dir"] == "train":
            s["lse"] = torch.empty(B, Hq, Lq, device=DEV)
            d = torch.empty(B, Lq, Hq + 2 * Hk, D, dtype=t, device=DEV)
            s["dq"], s["dk"], s["dv"] = d[:, :, :Hq], d[:, :, Hq:Hq + Hk], d[:, :, Hq + Hk:]
    return s


def _own_attn(s):
    op = s["op"]
    if s["c"]["dir"] == "fwd":
        op.fwd(s["q"], s["k"], s["v"], s["o"], ws=s["ws"])
        return {"o": s["o"]}
    op.fwd(s["q"], s["k"], s["v"], s["o"], s["lse"], ws=s["ws"])
    op.bwd(s["q"], s["k"], s["v"], s["o"], s["lse"], s["do"], s["dq"], s["dk"], s["dv"], ws=s["ws"])
    return {k: s[k] for k in ("o", "lse", "dq", "dk", "dv")}


def _plain_attn(s):
    c = s["c"]
    B, Lq, Lk, Hq, Hk, D = c["batch"], c["lq"], c["lk"], c["hq"], c["hk"], c["dim"]
    G, t = Hq // Hk, s["q"].dtype

    def rows(x):  # [batch][tokens][query heads][dim] -> [batch][key heads][heads of the group x tokens][dim]
        return x.float().reshape(B, Lq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, D)

    def back(x):
        return x.reshape(B, Hk, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, D)

    q, k, v = rows(s["q"]), s["k"].float().permute(0, 2, 1, 3), s["v"].float().permute(0, 2, 1, 3)
    j = torch.arange(Lk, device=DEV)
    n = s["lens"].long()[:, None] if "lens" in s else torch.full((B, 1), Lk, device=DEV)
    i = torch.arange(Lq, device=DEV)[None] + n - Lq  # positions of the queries [batch][Lq]
    see = (j < n)[:, None].expand(B, Lq, Lk)
    if c["mask"] != "none":
        before = j <= i[:, :, None]
        see = see & (before | (j < s["prefix"].long()[:, None, None]) if c["mask"] == "prefix" else before)
    if c["doc"]:
        see = see & (s["doc"][:, :, None] == s["doc"][:, None, :]) & (s["doc"][:, :, None] >= 0)
    see = see[:, None, None]  # [batch][1][1][Lq][Lk]

    x = (q @ k.transpose(2, 3)).mul_(s["scale"])
    if c["cap"] > 0:
        th = x.div_(c["cap"]).tanh_()
        x = th * c["cap"]
    x = x.view(B, Hk, G, Lq, Lk)
    if c["bias"] != "none":
        if c["bias"] == "grid":
            far = (i[:, :, None] // c["width"] - j // c["width"]).abs() + (i[:, :, None] % c["width"] - j % c["width"]).abs()
        else:
            far = (i[:, :, None] - j).abs()
        x = x - s["slopes"].view(1, Hk, G, 1, 1) * far.float()[:, None, None]
    x = torch.where(see, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(B, Hk, G * Lq, Lk)
    o = p @ v
    out = {"o": back(o).to(t)}
    if c["dir"] == "train":
        do = rows(s["do"])
        out["lse"] = (top + torch.log(total)).view(B, Hq, Lq)
        out["dv"] = (p.transpose(2, 3) @ do).permute(0, 2, 1, 3).to(t)
        ds = p * (do @ v.transpose(2, 3) - (do * o).sum(-1, keepdim=True))
        if c["cap"] > 0:
            ds = ds * (1 - th * th)
        ds = ds * s["scale"]
        out["dq"] = back(ds @ k).to(t)
        out["dk"] = (ds.transpose(2, 3) @ q).permute(0, 2, 1, 3).to(t)
    return out


def _exact_attn(c, seed):
    """One (sequence, key head) at a time in 64 bits; the gradients are autograd's of the softmax expression."""
    if _pairs(c) * c["hq"] * c["dim"] > 6e10:
        return None
    s = prepare(c, seed)
    B, Lq, Lk, Hq, Hk, D = c["batch"], c["lq"], c["lk"], c["hq"], c["hk"], c["dim"]
    train, G = c["dir"] == "train", Hq // Hk
    lens = _lens(c) if _serving(c) else [Lk] * B
    docs, prefix = _docs(c) if c["doc"] else None, _prefix(c) if c["mask"] == "prefix" else None
    z = lambda h: torch.zeros(B, Lq if h == Hq else Lk, h, D, dtype=torch.float64, device=DEV)  # noqa: E731
    out = {"o": z(Hq)}
    if train:
        out |= {"lse": torch.zeros(B, Hq, Lq, dtype=torch.float64, device=DEV), "dq": z(Hq), "dk": z(Hk), "dv": z(Hk)}
    for b, m in itertools.product(range(B), range(Hk)):
        n = int(lens[b])
        at = np.arange(Lq) + n - Lq
        if c["mask"] == "none":
            hidden = np.zeros((Lq, n), bool)
        else:
            hidden = np.arange(n)[None] > at[:, None]
            if prefix is not None:
                hidden &= (np.arange(n) >= prefix[b])[None]
        if docs is not None:
            hidden |= docs[b][:, None] != docs[b][None]
            hidden |= docs[b][:, None] < 0
        empty = torch.from_numpy(hidden.all(1)).to(DEV)
        hidden = torch.from_numpy(hidden).to(DEV)
        if c["bias"] == "grid":
            y, x = np.divmod(at, c["width"])
            ky, kx = np.divmod(np.arange(n), c["width"])
            far = np.abs(y[:, None] - ky) + np.abs(x[:, None] - kx)
        elif c["bias"] == "line":
            far = np.abs(at[:, None] - np.arange(n))
        k = s["k"][b, :n, m].double().requires_grad_(train)
        v = s["v"][b, :n, m].double().requires_grad_(train)
        for h in range(m * G, m * G + G):
            q = s["q"][b, :, h].double().requires_grad_(train)
            with torch.set_grad_enabled(train):
                w = torch.einsum("id,jd->ij", q, k) * s["scale"]
                if c["cap"]:
                    w = c["cap"] * torch.tanh(w / c["cap"])
                if c["bias"] != "none":
                    w = w - float(s["slopes"][h]) * torch.from_numpy(far).to(DEV)
                w = w.masked_fill(hidden, -math.inf)
                lse = torch.logsumexp(w, 1)
                p = torch.softmax(w.masked_fill(empty[:, None], 0.0), 1).masked_fill(empty[:, None], 0.0)
                o = torch.einsum("ij,jd->id", p, v)
                if train:
                    o.backward(s["do"][b, :, h].double())
            out["o"][b, :, h] = o.detach()
            if train:
                out["lse"][b, h], out["dq"][b, :, h] = lse.detach(), q.grad
        if train:
            out["dk"][b, :n, m], out["dv"][b, :n, m] = k.grad, v.grad
    return out


def _work_attn(c):
    size = 2
    keys = int(_lens(c).sum()) if _serving(c) else c["batch"] * c["lk"]
    qs, ks = c["batch"] * c["lq"] * c["hq"] * c["dim"] * size, keys * c["hk"] * c["dim"] * size
    pairs = _pairs(c) * c["hq"]
    if c["dir"] == "fwd":
        return {"bytes": 2 * qs + 2 * ks, "flops": 4 * pairs * c["dim"]}
    return {"bytes": 4 * qs + 4 * ks + 4 * c["batch"] * c["lq"] * c["hq"], "flops": 14 * pairs * c["dim"]}


# ------------------------------------------------------------------------------------------------ RMS norm
EPS = 1e-5
GROUP = 128  # channels that share a scale in 8 bits


def _prepare_rms(c, g):
    R, C, t = c["rows"], c["cols"], TYPES[c["type"]]
    s = {"c": c, "x": torch.randn(R, C, generator=g, device=DEV, dtype=t),
         "w": 1 + 0.2 * torch.randn(C, generator=g, device=DEV)}
    if c["res"]:
        s["r"] = torch.randn(R, C, generator=g, device=DEV, dtype=t) * 2
    if c["dir"] == "train":
        s["dy"] = torch.randn(R, C, generator=g, device=DEV, dtype=t)
        s["dsum"] = torch.randn(R, C, generator=g, device=DEV, dtype=t) if c["res"] else None
    if own:  # the output buffers that a program keeps
        s["h"] = torch.empty(R, C, dtype=t, device=DEV) if c["res"] else s["x"]
        s["rstd"] = torch.empty(R, device=DEV)
        if c["dir"] == "q8":
            s["q"] = torch.empty(R, C, dtype=torch.float8_e4m3fn, device=DEV)
            s["qs"] = torch.empty(R, -(-C // GROUP), device=DEV)
        else:
            s["y"] = torch.empty(R, C, dtype=t, device=DEV)
        if c["dir"] == "train":
            s["dx"], s["dw"] = torch.empty(R, C, dtype=t, device=DEV), torch.empty(C, device=DEV)
    return s


def _own_rms(s):
    from objectsam_b200 import norm
    c, r, h = s["c"], s.get("r"), s["h"]
    total = h if c["res"] else None
    if c["dir"] == "q8":
        norm.rms_norm_fwd_q8(s["x"], s["w"], EPS, s["q"], s["qs"], res=r, total=total, rstd=s["rstd"])
        out = {"q": s["q"], "qs": s["qs"], "rstd": s["rstd"]}
    else:
        norm.rms_norm_fwd(s["x"], s["w"], EPS, s["y"], res=r, total=total, rstd=s["rstd"])
        out = {"y": s["y"], "rstd": s["rstd"]}
    if c["dir"] == "train":
        norm.rms_norm_bwd(s["dy"], h, s["w"], s["rstd"], s["dx"], s["dw"], dtotal=s["dsum"])
        out |= {"dx": s["dx"], "dw": s["dw"]}
    return out | ({"h": h} if c["res"] else {})


def _plain_rms(s):
    c, t = s["c"], s["x"].dtype
    h = s["x"].float()
    if c["res"]:
        h = h + s["r"].float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    y = h * rstd * s["w"]
    out = {"rstd": rstd[:, 0]}
    if c["res"]:
        out["h"] = h.to(t)
    if c["dir"] == "q8":
        R, C = h.shape
        n = -(-C // GROUP)
        y = torch.cat([y, y.new_zeros(R, n * GROUP - C)], 1).view(R, n, GROUP)
        top = y.abs().amax(2, keepdim=True)
        out["qs"] = (top / 448)[..., 0]
        out["q"] = (y * torch.where(top > 0, 448 / top, 0.0)).view(R, -1)[:, :C].to(torch.float8_e4m3fn)
        return out
    out["y"] = y.to(t)
    if c["dir"] == "train":  # the backward pass reads the sum as it was stored
        dy = s["dy"].float()
        n = h.to(t).float() * rstd
        wdy = dy * s["w"]
        dx = (wdy - n * (wdy * n).mean(1, keepdim=True)) * rstd
        out["dx"] = (dx + s["dsum"].float() if c["res"] else dx).to(t)
        out["dw"] = (dy * n).sum(0)
    return out


def _exact_rms(c, seed):
    s = prepare(c, seed)
    h = s["x"].double() + (s["r"].double() if c["res"] else 0)
    out = {"rstd": (h.square().sum(1) / c["cols"] + EPS) ** -0.5}
    w = s["w"].double()
    if c["res"]:
        out["h"] = h
    y = torch.einsum("rc,r,c->rc", h, out["rstd"], w)
    if c["dir"] == "q8":
        y = torch.nn.functional.pad(y, (0, -c["cols"] % GROUP)).unflatten(1, (-1, GROUP))
        out["qs"] = y.abs().max(2).values / 448
        out["q"] = (y / out["qs"][..., None].clamp_min(1e-300)).flatten(1)[:, :c["cols"]]
        return out
    out["y"] = y
    if c["dir"] == "train":
        x = h.clone().requires_grad_(True)
        wp = w.clone().requires_grad_(True)
        torch.nn.functional.rms_norm(x, (c["cols"],), wp, EPS).backward(s["dy"].double())
        out["dx"] = x.grad + (s["dsum"].double() if c["res"] else 0)
        out["dw"] = wp.grad
    return out


def _work_rms(c):
    n, size = c["rows"] * c["cols"], 2
    fwd = n * size * (2 if c["res"] else 1) + n * (size if c["res"] else 0) + 4 * c["rows"] + 4 * c["cols"]
    if c["dir"] == "q8":
        return {"bytes": fwd + n + 4 * c["rows"] * -(-c["cols"] // GROUP), "flops": 6 * n}
    bwd = n * size * (4 if c["res"] else 3) + 8 * c["cols"] if c["dir"] == "train" else 0
    return {"bytes": fwd + n * size + bwd, "flops": (14 if c["dir"] == "train" else 5) * n}


# ------------------------------------------------------------------------------------------------ AdamW
LR, B1, B2, AEPS, WD, STEP0 = 1e-3, 0.9, 0.999, 1e-8, 0.05, 1000
BLOCK = {32: 64, 8: 256}  # elements that a tensor's state is rounded up to; with 8 bits, that share a scale


def _net_sizes():
    """Element counts of this network's parameters in order: conv weights, norm gains and biases."""
    def c2f(c1, c2, n):
        c = c2 // 2
        return [(c1, c2, 1)] + [(c, c, 3)] * (2 * n) + [((2 + n) * c, c2, 1)]
    convs = [(3, 32, 3), (32, 64, 3), *c2f(64, 64, 1), (64, 128, 3), *c2f(128, 128, 2), (128, 256, 3), *c2f(256, 256, 2),
             (256, 512, 3), *c2f(512, 512, 1), (512, 256, 1), (1024, 512, 1), *c2f(768, 256, 1), *c2f(384, 128, 1),
             (128, 128, 3), *c2f(384, 256, 1), (256, 256, 3), *c2f(768, 512, 1)]
    for ch in (128, 256, 512):
        convs += [(ch, 64, 3), (64, 64, 3), (64, 64, 1), (ch, 128, 3), (128, 128, 3), (128, 1, 1), (ch, 32, 3),
                  (32, 32, 3), (32, 32, 1)]
    convs += [(128, 128, 3), (128, 128, 2), (128, 128, 3), (128, 32, 1)]
    return [n for a, b, k in convs for n in (a * b * k * k, b, b)]


def _sizes(c):
    if c["net"]:
        return _net_sizes()
    r = random.Random(c["tensors"] * 1009 + c["largest"])
    return [c["largest"]] + [_log(r, max(1, c["largest"] // (4 if c["largest"] > 1_000_000 else 3000)), c["largest"])
                             for _ in range(c["tensors"] - 1)]


def _offsets(sizes, unit):
    return np.concatenate([[0], np.cumsum([-(-n // unit) * unit for n in sizes])]).astype(np.int64)


def _prepare_adamw(c, g):
    sizes, U = _sizes(c), BLOCK[c["bits"]]
    so, po = _offsets(sizes, U), _offsets(sizes, 1 if c["packed"] else U)  # of the states, of the parameters
    n = int(po[-1])
    size = torch.tensor(sizes, device=DEV)
    start = torch.from_numpy(so[:-1]).to(DEV)
    tensor_of = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.from_numpy(np.diff(po)).to(DEV),
                                        output_size=n)
    inside = torch.arange(n, device=DEV) - torch.from_numpy(po[:-1]).to(DEV)[tensor_of]
    used = inside < size[tensor_of]
    level = 10 ** (-1 - 3 * torch.rand(len(sizes), generator=g, device=DEV))  # gradients' size, tensor by tensor
    grad = torch.randn(n, generator=g, device=DEV) * level[tensor_of] * used
    s = {"c": c, "n": n, "sizes": sizes, "po": po, "p": torch.randn(n, generator=g, device=DEV) * 0.05 * used,
         "g": grad.to(TYPES[c["grad"]]), "t": STEP0}
    if c["packed"]:  # where each parameter's state lies
        s["at"] = start[tensor_of] + inside
    flat = torch.zeros(int(so[-1]), device=DEV)
    spread = lambda v: flat.index_copy(0, s["at"], v) if c["packed"] else v  # noqa: E731
    m = spread(grad * 0.3 + 0.1 * level[tensor_of] * used * torch.randn(n, generator=g, device=DEV))
    v = spread((grad * torch.rand(n, generator=g, device=DEV)).square() + (0.3 * level[tensor_of] * used).square())
    decay = torch.tensor([float(k >= 2048) for k in sizes], device=DEV)  # norm gains and biases do not decay
    s["decay"] = torch.repeat_interleave(decay, torch.from_numpy(np.diff(so) // U).to(DEV))[:, None]
    if c["bits"] == 8:
        s["m"], s["ms"] = _to8(m.view(-1, U), False)
        s["v"], s["vs"] = _to8(v.sqrt().view(-1, U), True)
    else:
        s["m"], s["v"] = m.view(-1, U), v.view(-1, U)
    if c["copy"] != "none":
        s["copy"] = s["p"].to(TYPES[c["copy"]])
    if own:  # the optimizer object, made once over the program's tensors
        from objectsam_b200.optim import AdamW
        cut = lambda x: [x[a:a + k] for a, k in zip(po[:-1].tolist(), sizes)]  # noqa: E731
        s["opt"] = opt = AdamW(cut(s["p"]), cut(s["g"]), copies=cut(s["copy"]) if "copy" in s else None, lr=LR,
                               betas=(B1, B2), eps=AEPS, weight_decay=WD, bits=c["bits"],
                               decay=[k >= 2048 for k in sizes], step=STEP0)
        opt.load_state(m=s["m"], v=s["v"], m_scale=s.get("ms"), v_scale=s.get("vs"))
    return s


def _to8(x, positive):
    """e4m3 values and a scale for each row; with `positive`, what is above zero stays above zero."""
    top = x.abs().amax(1, keepdim=True)
    live = top >= 1e-30
    q = (x * torch.where(live, 448 / top, 0.0)).to(torch.float8_e4m3fn)
    if positive:
        f = q.float()
        q = torch.where(live & (x > 0) & (f == 0), 2.0 ** -9, f).to(torch.float8_e4m3fn)
    return q, torch.where(live, top / 448, 0.0)


def _own_adamw(s):
    c, opt = s["c"], s["opt"]
    opt.step(max_norm=c["clip"] or None)
    out = {"p": s["p"], "m": opt.m, "v": opt.v}
    if c["bits"] == 8:
        out |= {"ms": opt.m_scale, "vs": opt.v_scale}
    if c["copy"] != "none":
        out["copy"] = s["copy"]
    return out | ({"norm": opt.norm} if c["clip"] else {})


def _plain_adamw(s):
    c, U = s["c"], BLOCK[s["c"]["bits"]]
    s["t"] += 1
    g = s["g"].float()
    out = {}
    if c["clip"]:
        out["norm"] = (g * g).sum().sqrt().view(1)
        g = g * torch.clamp(c["clip"] / (out["norm"] + 1e-6), max=1.0)
    p = s["p"]
    if c["packed"]:
        lay = torch.zeros(s["m"].numel(), device=DEV)
        g, p = lay.index_copy(0, s["at"], g), lay.index_copy(0, s["at"], p)
    g, p = g.view(-1, U), p.view(-1, U)
    if c["bits"] == 8:
        m, v = s["m"].view(-1, U).float() * s["ms"].view(-1, 1), (s["v"].view(-1, U).float() * s["vs"].view(-1, 1)).square()
    else:
        m, v = s["m"].view(-1, U), s["v"].view(-1, U)
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * (g * g)
    root = v.sqrt()
    p = p * (1 - LR * WD * s["decay"]) - (LR / (1 - B1 ** s["t"])) * m / (root / math.sqrt(1 - B2 ** s["t"]) + AEPS)
    p = p.view(-1)
    s["p"] = p[s["at"]] if c["packed"] else p
    if c["bits"] == 8:
        (m, ms), (v, vs) = _to8(m, False), _to8(root, True)
        s["ms"], s["vs"] = ms.view(-1), vs.view(-1)
        out |= {"ms": s["ms"], "vs": s["vs"]}
    s["m"], s["v"] = m.view(-1), v.view(-1)
    out |= {"p": s["p"], "m": s["m"], "v": s["v"]}
    if c["copy"] != "none":
        out["copy"] = s["p"].to(TYPES[c["copy"]])
    return out


def _exact_adamw(c, seed):
    s = prepare(c, seed)
    U, n8, t = BLOCK[c["bits"]], c["bits"] == 8, STEP0 + 1
    at = s["at"] if c["packed"] else slice(None)
    g = s["g"].double()
    m, v = s["m"].double().view(-1, U), s["v"].double().view(-1, U)
    if n8:
        m, v = m * s["ms"].double(), (v * s["vs"].double()) ** 2
    out = {}
    if c["clip"]:
        out["norm"] = torch.linalg.vector_norm(g).view(1)
        g = g * min(1.0, c["clip"] / (float(out["norm"]) + 1e-6))
    G = torch.zeros(m.numel(), dtype=torch.float64, device=DEV)
    G[at] = g
    m = torch.lerp(G.view(-1, U), m, B1)
    v = torch.lerp(G.view(-1, U) ** 2, v, B2)
    mh, vh = m / (1 - B1 ** t), v / (1 - B2 ** t)
    decay = (1 - LR * WD * s["decay"].double()).expand(-1, U).reshape(-1)[at]
    out["p"] = s["p"].double() * decay - LR * (mh / (vh.sqrt() + AEPS)).view(-1)[at]
    if c["copy"] != "none":
        out["copy"] = out["p"]
    if n8:
        out["ms"], out["vs"] = m.abs().max(1).values / 448, v.sqrt().max(1).values / 448
        out["m"] = (m / out["ms"].clamp_min(1e-300)[:, None]).view(-1)
        out["v"] = (v.sqrt() / out["vs"].clamp_min(1e-300)[:, None]).view(-1)
    else:
        out["m"], out["v"] = m.view(-1), v.view(-1)
    return out


def _work_adamw(c):
    n = sum(_sizes(c))
    gb, cb = {"f32": 4, "f16": 2, "bf16": 2}[c["grad"]], {"none": 0, "f16": 2, "bf16": 2}[c["copy"]]
    state = 16 if c["bits"] == 32 else 4 + 16 / 256
    return {"bytes": n * (8 + gb + cb + state), "flops": n * (16 if c["clip"] else 14)}


# ------------------------------------------------------------------------------------------------ all
_BY_OP = {"attn": (_prepare_attn, _own_attn, _plain_attn, _exact_attn, _work_attn),
          "rms": (_prepare_rms, _own_rms, _plain_rms, _exact_rms, _work_rms),
          "adamw": (_prepare_adamw, _own_adamw, _plain_adamw, _exact_adamw, _work_adamw)}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return _BY_OP[case["op"]][0](case, g)


def run(state):
    return _BY_OP[state["c"]["op"]][1 if own else 2](state)


def exact(case, seed):
    return _BY_OP[case["op"]][3](case, seed)


def work(case):
    return _BY_OP[case["op"]][4](case)
