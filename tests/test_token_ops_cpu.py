"""The token operators without a GPU: their refusals (argument checks come before any device call), and the 64-bit
restatement's gradients against differences."""
import math

import pytest
import torch

from objectsam_b200 import _lib
from objectsam_b200._lib import AdamWTensor, AttnDesc, View, lib
from oracle import token_ref

INVALID = _lib.OSAM_ERR_INVALID


def desc(**kw):
    d = dict(dtype=_lib.F16, batch=1, len_q=4, len_k=4, heads_q=2, heads_k=2, dim=64, mask=_lib.ATTN_NONE, scale=0.125,
             cap=0.0, grid_w=0)
    d.update(kw)
    return AttnDesc(**d)


def fwd(d, *views):
    import ctypes
    views = list(views) or [View(4096, 4 * 128, 128, 64)] * 4
    return lib().osam_attn_fwd(ctypes.byref(d), *views, None, None, 0, None)


@pytest.mark.parametrize("kw", [dict(dtype=_lib.F32), dict(dtype=7), dict(batch=-1), dict(len_q=-1), dict(len_k=-2),
                                dict(heads_q=0), dict(heads_q=3), dict(heads_k=0), dict(dim=0), dict(dim=12), dict(dim=136),
                                dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan),
                                dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf), dict(mask=3), dict(mask=-1),
                                dict(mask=_lib.ATTN_PREFIX), dict(doc_q=4096), dict(doc_k=4096), dict(grid_w=-1),
                                dict(len_q=1 << 30, heads_q=4), dict(len_k=(1 << 30) + 1),
                                dict(len_k=1048577, doc_q=4096, doc_k=4096)])
def test_attention_descriptions(kw):
    import ctypes
    d = desc(**kw)
    assert fwd(d) == INVALID and lib().osam_last_error().startswith(b"attention: ")
    assert lib().osam_attn_workspace_size(ctypes.byref(d)) == 0


def test_attention_views():
    good = View(4096, 512, 128, 64)
    for bad in (View(None, 512, 128, 64), View(4104, 512, 128, 64), View(4096, 512, 124, 64), View(4096, 512, 0, 64),
                View(4096, 512, -128, 64), View(4096, 512, 128, 1 << 40)):
        for at in range(4):
            assert fwd(desc(), *(bad if i == at else good for i in range(4))) == INVALID
    assert fwd(desc(), good, good, good, good) == INVALID and b"workspace" in lib().osam_last_error()
    # strides of extents of one are not looked at, and empty work is no error
    one = View(4096, 3, 5, 7)
    assert fwd(desc(len_q=1, len_k=1, heads_q=1, heads_k=1), one, one, one, one) == INVALID
    assert b"workspace" in lib().osam_last_error()
    assert fwd(desc(batch=0)) == fwd(desc(len_q=0)) == _lib.OSAM_OK


def test_rms_refusals():
    L = lib()

    def call(dtype=_lib.F16, x=4096, ldx=64, res=None, ldres=0, w=4096, rows=3, C=64, total=None, ldt=0, y=8192, ldy=64):
        return L.osam_rms_fwd(dtype, x, ldx, res, ldres, w, rows, C, 1e-5, total, ldt, y, ldy, None, None)

    for kw in (dict(dtype=_lib.F32), dict(C=60), dict(C=0), dict(C=8200, ldx=8200, ldy=8200), dict(rows=-1), dict(x=None),
               dict(x=4104), dict(ldx=56), dict(ldx=68), dict(w=None), dict(y=None), dict(ldy=8), dict(res=4100, ldres=64),
               dict(res=4096, ldres=32), dict(total=4096, ldt=60)):
        assert call(**kw) == INVALID, kw
    assert call(rows=0) == _lib.OSAM_OK
    assert L.osam_rms_fwd_q8(_lib.F16, 4096, 64, None, 0, 4096, 3, 64, 1e-5, None, 0, 8192, 64, None, None, None) == INVALID
    assert L.osam_rms_fwd_q8(_lib.F16, 4096, 64, None, 0, 4096, 3, 64, 1e-5, None, 0, 8196, 64, 4096, None, None) == INVALID
    assert L.osam_rms_bwd_workspace_size(12000) == 0 and L.osam_rms_bwd_workspace_size(64) > 0
    assert L.osam_rms_bwd(_lib.F16, 4096, 64, 4096, 64, 4096, 4096, None, 0, 3, 64, 8192, 64, 4096, None, 0, None) == INVALID
    assert L.osam_rms_bwd(_lib.F16, 4096, 64, 4096, 64, 4096, 4096, None, 0, 3, 64, 8192, 64, None, 4096, 1 << 30, None) == INVALID


def test_adamw_refusals():
    import ctypes
    L = lib()
    nbytes, elems = ctypes.c_size_t(), ctypes.c_int64()

    def sizes(bits=32, **kw):
        t = dict(p=4096, g=4096, copy=None, n=100, grad_type=_lib.F32, copy_type=_lib.F16, decay=1)
        t.update(kw)
        tab = (AdamWTensor * 2)(AdamWTensor(**t), AdamWTensor(4096, 4096, None, 65, _lib.F32, _lib.F16, 0))
        return L.osam_adamw_sizes(tab, 2, bits, ctypes.byref(nbytes), ctypes.byref(elems))

    assert sizes() == _lib.OSAM_OK and elems.value == 128 + 128
    assert sizes(8) == _lib.OSAM_OK and elems.value == 256 + 256
    for kw in (dict(bits=16), dict(n=-1), dict(p=None), dict(g=None), dict(p=4098), dict(g=4097), dict(grad_type=5),
               dict(copy=4096, copy_type=_lib.F32), dict(copy=4097)):
        assert sizes(**kw) == INVALID, kw
    plan = ctypes.c_void_p()
    tab = (AdamWTensor * 1)(AdamWTensor(4096, 4096, None, 65, _lib.F32, _lib.F16, 0))
    assert L.osam_adamw_create(tab, 1, 32, None, 0, None, ctypes.byref(plan)) == INVALID and not plan
    assert L.osam_adamw_step(None, 4096, 4096, None, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 0.0, None, None) == INVALID
    # a plan over no elements: the checks of a step need no device
    none = (AdamWTensor * 1)(AdamWTensor(None, None, None, 0, _lib.F32, _lib.F16, 0))
    assert L.osam_adamw_sizes(none, 1, 32, ctypes.byref(nbytes), ctypes.byref(elems)) == _lib.OSAM_OK and elems.value == 0


def test_python_refusals():
    from objectsam_b200 import norm
    from objectsam_b200.attn import AttnGeom, AttnOp
    from objectsam_b200.optim import AdamW
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        norm.rms_norm_fwd(x, torch.ones(64), 1e-5, x)  # not on a GPU
    with pytest.raises(ValueError):
        norm.rms_norm_fwd(x.float(), torch.ones(64), 1e-5, x)
    with pytest.raises(ValueError):
        AttnOp().init(AttnGeom(1, 4, 4, 1, 1, 64, torch.float32))
    with pytest.raises(ValueError):
        AttnOp().init(AttnGeom(1, 4, 4, 1, 1, 64), mask="window")
    with pytest.raises(ValueError):
        AttnOp().init(AttnGeom(1, 4, 4, 1, 1, 64), slopes=torch.ones(2))
    with pytest.raises(_lib.OsamError):
        AttnOp().init(AttnGeom(1, 4, 4, 1, 1, 60))
    with pytest.raises(ValueError):
        AdamW([], [])
    with pytest.raises(ValueError):
        AdamW([torch.zeros(4)], [torch.zeros(4)])


@pytest.mark.parametrize("cap,slope,mask", [(0.0, 0.0, "none"), (2.0, 0.3, "causal"), (3.0, 0.1, "prefix")])
def test_reference_attention_gradients(cap, slope, mask):
    """Σ gradient·d against central differences of the restated forward, both in 64 bits: the difference's error is
    ε²/6 of the third derivative, about 1e-9 here."""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    B, L, Hq, Hk, D = 2, 9, 4, 2, 5
    q, k, v, do = r(B, L, Hq, D), r(B, L, Hk, D), r(B, L, Hk, D), r(B, L, Hq, D)
    doc = torch.tensor([[0, 0, 0, 1, 1, -1, 1, 1, 0]] * B, dtype=torch.int32)
    vis = token_ref.attn_visible(B, L, L, mask, prefix=[3, 7], doc_q=doc, doc_k=doc)
    kw = dict(scale=0.4, cap=cap, slopes=torch.full((Hq,), slope), distance=token_ref.attn_distance(B, L, L, 3))
    out = token_ref.attention(q, k, v, vis, do=do, **kw)
    eps = 1e-5
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2)):
        d = r(*out[name].shape)
        loss = []
        for s in (eps, -eps):
            a = [q, k, v]
            a[at] = a[at] + s * d
            loss.append((token_ref.attention(*a, vis, **kw)["o"] * do).sum())
        assert abs((loss[0] - loss[1]) / (2 * eps) - (out[name] * d).sum()) < 1e-7


def test_reference_rms_gradients():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, dy = r(5, 16), r(16), r(5, 16)
    out = token_ref.rms_norm(x, w, 1e-5, dy=dy)
    eps = 1e-5
    dx, dw = r(5, 16), r(16)
    up, down = token_ref.rms_norm(x + eps * dx, w + eps * dw, 1e-5)["y"], token_ref.rms_norm(x - eps * dx, w - eps * dw, 1e-5)["y"]
    got = ((up - down) * dy).sum() / (2 * eps)
    assert abs(got - (out["dx"] * dx).sum() - (out["dw"] * dw).sum()) < 1e-7


class Strided:
    """A CUDA tensor's shape and strides, as the argument checks see them."""
    dtype, is_cuda = torch.float16, True

    def __init__(self, t):
        self.t, self.shape = t, t.shape

    def is_contiguous(self):
        return self.t.is_contiguous()

    def stride(self):
        return self.t.stride()

    def data_ptr(self):
        return 4096


def test_rows_of_a_norm():
    """Rows are taken by one distance from row to row; a row that broadcasting repeats has none."""
    from objectsam_b200 import norm
    base = torch.zeros(6, 10, 96, dtype=torch.float16)
    rows = lambda t: norm._rows(Strided(t), t.shape, torch.float16, "x")  # noqa: E731
    assert rows(base) == (4096, 96) and rows(base[..., 16:80]) == (4096, 96) and rows(base[:, 3:4, :32]) == (4096, 960)
    assert rows(base[:1, :1]) == (4096, 96) and rows(base[:, ::2, :64]) == (4096, 192)
    row = torch.zeros(1, 64, dtype=torch.float16)
    for bad in (row.expand(8, 64), base[:, :1].expand(6, 10, 96), base[:1].expand(6, 10, 96), base[:, :5], base[..., :64].as_strided((5, 64), (32, 1)),
                base.transpose(1, 2)):
        with pytest.raises(ValueError):
            rows(bad)


def test_kept_workspaces_go_by_device_and_stream(monkeypatch):
    """The default stream has the same handle on every device."""
    import contextlib
    from types import SimpleNamespace

    from objectsam_b200.attn import AttnGeom, AttnOp
    op = AttnOp().init(AttnGeom(1, 4, 4, 1, 1, 64))
    made = []
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: made.append(device) or
                        SimpleNamespace(data_ptr=lambda at=len(made): at, numel=lambda: n, element_size=lambda: 1))
    streams = [SimpleNamespace(device=torch.device("cuda", d), cuda_stream=h) for d, h in ((0, 0), (1, 0), (1, 7))]
    got = [op._workspace(None, s) for s in streams + streams]
    assert [p for p, _ in got] == [1, 2, 3] * 2 and [d.index for d in made] == [0, 1, 1]


def test_workspaces_are_looked_at():
    """A workspace in host memory, or one with gaps, is refused before anything is launched."""
    from types import SimpleNamespace

    from objectsam_b200 import norm
    from objectsam_b200.attn import AttnGeom, AttnOp
    op = AttnOp().init(AttnGeom(1, 4, 4, 1, 1, 64))
    flat = torch.zeros(op.workspace_size() * 2, dtype=torch.uint8)
    gaps = SimpleNamespace(is_cuda=True, is_contiguous=lambda: False)
    dy = torch.zeros(4, 64, dtype=torch.float16)
    for ws in (flat, gaps):
        with pytest.raises(ValueError, match="workspace"):
            op.fwd(None, None, None, None, ws=ws)
        with pytest.raises(ValueError, match="workspace"):
            op.bwd(None, None, None, None, None, None, None, None, None, ws=ws)
        with pytest.raises(ValueError, match="ws"):
            norm.rms_norm_bwd(dy, dy, None, None, dy, None, ws=ws)


@pytest.mark.parametrize("kw", [dict(batch=1 << 30, heads_q=1 << 30, heads_k=1 << 30, len_q=1 << 10, len_k=1 << 10),
                                dict(batch=1 << 16, heads_q=1 << 16, heads_k=1 << 16, len_q=1, len_k=1 << 30),
                                dict(batch=(1 << 31) - 1, heads_q=(1 << 31) - 1, heads_k=(1 << 31) - 1, len_q=1, len_k=1),
                                dict(batch=1 << 20, heads_q=1 << 20, heads_k=1 << 20, len_q=1 << 30, len_k=0),
                                dict(grid_w=(1 << 30) + 1), dict(grid_w=(1 << 31) - 1)])
def test_descriptions_past_any_size(kw):
    """Products that wrap in 64 bits are too large, not small."""
    import ctypes
    d = desc(**kw)
    assert lib().osam_attn_workspace_size(ctypes.byref(d)) == 0
    assert fwd(d) == INVALID and (b"too many tokens" in lib().osam_last_error() or b"grid_w" in lib().osam_last_error())


@pytest.mark.parametrize("sizes", [[(1 << 63) - 1], [1 << 62] * 3, [(1 << 63) - 2000] * 2, [1 << 43], [1 << 41] * 4])
def test_adamw_over_any_number_of_elements(sizes):
    """Sizes whose layout would wrap are refused, by the sizes' call and by the plan's, which would else ask for memory by them."""
    import ctypes
    L, tab = lib(), (AdamWTensor * len(sizes))(*(AdamWTensor(4096, 4096, None, n, _lib.F32, _lib.F16, 1) for n in sizes))
    nbytes, elems, plan = ctypes.c_size_t(7), ctypes.c_int64(7), ctypes.c_void_p()
    assert L.osam_adamw_sizes(tab, len(sizes), 8, ctypes.byref(nbytes), ctypes.byref(elems)) == INVALID
    assert b"too many" in L.osam_last_error() and nbytes.value == 7
    assert L.osam_adamw_create(tab, len(sizes), 8, 4096, (1 << 64) - 1, None, ctypes.byref(plan)) == INVALID and not plan
    assert b"too many" in L.osam_last_error()


def test_vanishing_caps():
    """cap·tanh(s/cap) needs s/cap: a cap that fp32 cannot divide by is refused, and one that it rounds to 0 is not `none`."""
    import ctypes

    from objectsam_b200.attn import AttnGeom, AttnOp
    for kw in (dict(cap=1e-39), dict(cap=1e-10, scale=1e30)):
        assert fwd(desc(**kw)) == INVALID and b"cap is too small" in lib().osam_last_error(), kw
    assert lib().osam_attn_workspace_size(ctypes.byref(desc(cap=1e-37))) > 0
    with pytest.raises(ValueError):
        AttnOp().init(AttnGeom(1, 4, 4, 1, 1, 64), cap=1e-50)


def test_pointers_off_their_types():
    """fp32 and int32 arrays at odd addresses, which a kernel's loads would fault on."""
    import ctypes
    L, good = lib(), View(4096, 512, 128, 64)
    for kw in (dict(slopes=4097), dict(lens=4098), dict(prefix=4099, mask=_lib.ATTN_PREFIX), dict(doc_q=4098, doc_k=4096),
               dict(doc_q=4096, doc_k=4097)):
        assert fwd(desc(**kw)) == INVALID and b"aligned" in L.osam_last_error() and b"workspace" not in L.osam_last_error(), kw
        assert L.osam_attn_workspace_size(ctypes.byref(desc(**kw))) == 0
    d = ctypes.byref(desc())
    assert L.osam_attn_fwd(d, good, good, good, good, 4098, None, 0, None) == INVALID and b"lse" in L.osam_last_error()
    assert L.osam_attn_bwd(d, good, good, good, good, 4098, good, good, good, good, None, 0, None) == INVALID
    assert b"lse" in L.osam_last_error()

    def rms(w=4096, rstd=4096, qs=None, dw=4096):
        if qs is not None:
            return L.osam_rms_fwd_q8(_lib.F16, 4096, 64, None, 0, w, 3, 64, 1e-5, None, 0, 8192, 64, qs, rstd, None)
        a = L.osam_rms_fwd(_lib.F16, 4096, 64, None, 0, w, 3, 64, 1e-5, None, 0, 8192, 64, rstd, None) if dw == 4096 else INVALID
        b = L.osam_rms_bwd(_lib.F16, 4096, 64, 4096, 64, w, rstd, None, 0, 3, 64, 8192, 64, dw, 4096, 1 << 30, None)
        return INVALID if a == b == INVALID else 0

    for kw in (dict(w=4097), dict(rstd=4098), dict(qs=4099), dict(dw=4098)):
        assert rms(**kw) == INVALID and b"aligned" in L.osam_last_error(), kw
