"""osam_rms_* against the 64-bit restatement (oracle/token_ref.py).

Tolerances: y, h, dx are one rounding to the 16-bit type (unit u) of fp32 results whose own error is a few 2^-22 of the
row's terms: |Δ| ≤ 1.02·u·|ref| + 2^-20·(the row's largest term).  rstd and the e4m3 scales: 2^-20 relative.  dw sums up
to `rows` fp32 products: |Δ| ≤ 2^-18·Σ|dy·ĥ|.  e4m3: half a step, 2^-4 of the value (2^-10 of the scale below its normal range),
with 2^-18 for the fp32 value on the other side of a rounding boundary."""
import pytest
import torch

from oracle import token_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
EPS = 1e-5


def near(x, ref, unit, scale):
    lim = 1.02 * unit * ref.abs() + 2.0 ** -20 * scale + 2.0 ** -25  # fp16's subnormal half-step
    bad = ~((x.double() - ref).abs() <= lim)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((x.double() - ref).abs() / lim).max():.3g}×"


def check(rows, C, dtype=torch.float16, res=True, train=True, wide=0, seed=0):
    from objectsam_b200 import norm
    g = torch.Generator(device=DEV).manual_seed(seed)
    nan = float("nan")

    def buf(t=None, dt=None):  # `wide`: a channel slice of rows C + wide long
        b = torch.full((rows, C + wide), nan, device=DEV).to(dt or dtype)
        v = b[:, wide // 2 // 8 * 8:][:, :C] if wide else b
        if t is not None:
            v.copy_(t)
        return v

    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)  # noqa: E731
    x, w = buf(r(rows, C)), 1 + 0.3 * torch.randn(C, generator=g, device=DEV)
    rr = buf(r(rows, C) * 3) if res else None
    y, h, rstd = buf(), buf() if res else None, torch.full((rows,), nan, device=DEV)
    norm.rms_norm_fwd(x, w, EPS, y, res=rr, total=h, rstd=rstd)
    dy, ds = (buf(r(rows, C)), buf(r(rows, C)) if res else None) if train else (None, None)
    stored = (h if res else x).double()
    ref = token_ref.rms_norm(x.double(), w.double(), EPS, rr.double() if res else None, dy.double() if train else None,
                             ds.double() if res and train else None, stored)
    u = UNIT[dtype]
    row = lambda t: t.abs().amax(1, keepdim=True)  # noqa: E731
    near(y, ref["y"], u, row(ref["y"]))
    assert ((rstd.double() - ref["rstd"]).abs() <= 2.0 ** -20 * ref["rstd"]).all()
    if res:
        near(h, ref["h"], u, 0 * row(ref["h"]))
    if train:
        dx, dw = buf(), torch.full((C,), nan, device=DEV)
        norm.rms_norm_bwd(dy, h if res else x, w, rstd, dx, dw, dtotal=ds)
        near(dx, ref["dx"], u, row(ref["dx"]) + row(dy.double()) * ref["rstd"][:, None] * row(w[None].double()) * 8)
        lim = 2.0 ** -18 * (dy.double() * stored * ref["rstd"][:, None]).abs().sum(0) + 1e-30
        assert ((dw.double() - ref["dw"]).abs() <= lim).all()
        # a second call gives the same bits
        dw2, dx2 = torch.empty_like(dw), buf()
        norm.rms_norm_bwd(dy, h if res else x, w, rstd, dx2, dw2, dtotal=ds)
        assert torch.equal(dw, dw2) and torch.equal(dx, dx2)
    # e4m3
    q, qs = buf(dt=torch.float8_e4m3fn), torch.full((rows, -(-C // 128)), nan, device=DEV)
    h2 = buf() if res else None
    norm.rms_norm_fwd_q8(x, w, EPS, q, qs, res=rr, total=h2, rstd=rstd)
    pad = -C % 128
    grouped = torch.nn.functional.pad(ref["y"], (0, pad)).view(rows, -1, 128)
    top = grouped.abs().amax(2)
    assert ((qs.double() - top / 448).abs() <= 2.0 ** -20 * top / 448).all()
    back = (torch.nn.functional.pad(q.double(), (0, pad)).view(rows, -1, 128) * qs.double()[..., None])
    lim = torch.maximum(2.0 ** -4 * grouped.abs(), 2.0 ** -10 * qs.double()[..., None]) * (1 + 2.0 ** -10) + 2.0 ** -18 * top[..., None]
    assert ((back - grouped).abs() <= lim).all()
    if res:
        assert torch.equal(h2, h)


@pytest.mark.parametrize("C", [8, 16, 24, 32, 64, 72, 96, 128, 136, 256, 264, 512, 520, 1024, 1032, 2048, 2056, 4096, 5000, 8192])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_channels(cuda_lib, C, dtype):
    check(37, C, dtype, seed=C)


@pytest.mark.parametrize("rows", [1, 2, 31, 400, 1600, 9001])
@pytest.mark.parametrize("C", [32, 256, 1280])
def test_rows(cuda_lib, rows, C):
    check(rows, C, seed=rows)


@pytest.mark.parametrize("C", [64, 384, 1536])
def test_slices_and_no_residual(cuda_lib, C):
    check(300, C, wide=40, seed=1)
    check(300, C, res=False, seed=2)
    check(300, C, res=False, train=False, wide=8, seed=3)


def test_nhwc_maps_and_aliases(cuda_lib):
    """(N, H, W, C) maps as they are; total may be x or res, dx may be dy."""
    from objectsam_b200 import norm
    g = torch.Generator(device=DEV).manual_seed(4)
    r = lambda: torch.randn(2, 20, 20, 512, generator=g, device=DEV).half()  # noqa: E731
    x, res, dy, w = r(), r(), r(), torch.rand(512, generator=g, device=DEV)
    y, h, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(800, device=DEV)
    norm.rms_norm_fwd(x, w, EPS, y, res=res, total=h, rstd=rstd)
    for which in (0, 1):
        a, b = x.clone(), res.clone()
        y2 = torch.empty_like(x)
        norm.rms_norm_fwd(a, w, EPS, y2, res=b, total=(a, b)[which])
        assert torch.equal((a, b)[which], h) and torch.equal(y2, y)
    dx, dw = torch.empty_like(x), torch.empty(512, device=DEV)
    norm.rms_norm_bwd(dy, h, w, rstd, dx, dw)
    norm.rms_norm_bwd(dy, h, w, rstd, dy, dw)
    assert torch.equal(dx, dy)
    with pytest.raises(ValueError):  # rows that are not equally spaced
        norm.rms_norm_fwd(torch.empty(2, 22, 20, 512, dtype=torch.half, device=DEV)[:, :20], w, EPS, y)


def test_values(cuda_lib):
    """Zero rows give zeros; infinities and NaN stay in their rows."""
    from objectsam_b200 import norm
    x = torch.randn(6, 256, device=DEV).half()
    x[1] = 0
    x[3, 7] = float("inf")
    x[4, 9] = float("nan")
    w = torch.ones(256, device=DEV)
    y, q, qs = torch.empty_like(x), torch.empty(6, 256, dtype=torch.float8_e4m3fn, device=DEV), torch.empty(6, 2, device=DEV)
    norm.rms_norm_fwd(x, w, EPS, y)
    norm.rms_norm_fwd_q8(x, w, EPS, q, qs)
    assert (y[1] == 0).all() and (q[1].float() == 0).all() and (qs[1] == 0).all()
    assert torch.isfinite(y[[0, 2, 5]]).all() and torch.isfinite(q[[0, 2, 5]].float()).all()
    assert torch.isnan(y[3, 7]) and torch.isnan(y[4]).all()


def test_gradients_against_differences(cuda_lib):
    """Σ dx·d and Σ dw·e against central differences of the kernel's forward along d = sign(dx), e = sign(dw).  Steps and
    inputs are exact in fp16; the forward's rounding is a noise of 2^-11·√(Σ y²dy²) ≈ 0.03 against differences of
    hundreds, the third-order term of a step of 2^-5 under 1 %."""
    from objectsam_b200 import norm
    g = torch.Generator(device=DEV).manual_seed(5)
    x = (torch.randn(64, 96, generator=g, device=DEV) * 64).round().div(64).half()
    dy = torch.randn(64, 96, generator=g, device=DEV).half()
    w = 1 + 0.2 * torch.randn(96, generator=g, device=DEV)
    y, rstd, dx, dw = torch.empty_like(x), torch.empty(64, device=DEV), torch.empty_like(x), torch.empty(96, device=DEV)
    norm.rms_norm_fwd(x, w, EPS, y, rstd=rstd)
    norm.rms_norm_bwd(dy, x, w, rstd, dx, dw)
    eps = 2.0 ** -5

    def loss(a, b):
        norm.rms_norm_fwd(a, b, EPS, y)
        return (y.double() * dy.double()).sum().item()

    d, e = torch.sign(dx.float()), torch.sign(dw)
    got = (loss((x.float() + eps * d).half(), w) - loss((x.float() - eps * d).half(), w)) / (2 * eps)
    assert abs(got - dx.double().abs().sum().item()) <= 0.02 * abs(got)
    got = (loss(x, w + eps * e) - loss(x, w - eps * e)) / (2 * eps)
    assert abs(got - dw.double().abs().sum().item()) <= 0.02 * abs(got)


def test_empty_and_many(cuda_lib):
    from objectsam_b200 import norm
    x = torch.empty(0, 64, dtype=torch.half, device=DEV)
    w, dw = torch.ones(64, device=DEV), torch.full((64,), float("nan"), device=DEV)
    norm.rms_norm_fwd(x, w, EPS, x)
    norm.rms_norm_bwd(x, x, w, torch.empty(0, device=DEV), x, dw)
    torch.cuda.synchronize()
    assert (dw == 0).all()
    # element offsets past 2^31
    rows, C = 270_000, 8192
    x = torch.zeros(rows, C, dtype=torch.half, device=DEV)
    x[-3:] = torch.randn(3, C, device=DEV).half()
    norm.rms_norm_fwd(x, torch.ones(C, device=DEV), EPS, x)
    tail = x[-3:].double()
    assert ((tail * tail).mean(1) - 1).abs().max() < 1e-2 and not x[:8].any()


@pytest.mark.parametrize("C", [128, 264, 2048])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_vanishing_groups(cuda_lib, C, dtype):
    """A group whose largest |y| is near fp32's smallest normal number keeps its values' proportions, and its zeros; y there is
    ±2^-125·rstd and halves of it, normal numbers, so q is off by e4m3's half step and the scale by its own subnormal step."""
    from objectsam_b200 import norm
    x = torch.randn(5, C, device=DEV).to(dtype)
    w = torch.ones(C, device=DEV)
    part = torch.tensor([1.0, 0.0, -0.5, 0.25], device=DEV).repeat(32)
    x[:, :128] = part.to(dtype)
    x[:, 128:] *= 0.25
    w[:128] = 2.0 ** -124
    q, qs = torch.empty(5, C, dtype=torch.float8_e4m3fn, device=DEV), torch.empty(5, -(-C // 128), device=DEV)
    norm.rms_norm_fwd_q8(x, w, EPS, q, qs)
    assert torch.isfinite(q.float()).all()
    got, want = q[:, :128].double(), 448.0 * part.double()
    assert ((got - want).abs() <= 2.0 ** -4 * want.abs()).all()
    rstd = torch.rsqrt(x.double().square().mean(1) + EPS)
    assert ((qs[:, 0].double() - 2.0 ** -124 * rstd / 448).abs() <= 2.0 ** -149).all()


def test_captured_backward_keeps_its_workspace(cuda_lib):
    """A graph holds the address of the workspace that the norm keeps for its stream: wider calls on that stream take others."""
    from objectsam_b200 import norm
    g = torch.Generator(device=DEV).manual_seed(6)
    s = torch.cuda.Stream()

    def case(C):
        dy, x = (torch.randn(700, C, generator=g, device=DEV).half() for _ in range(2))
        return dy, x, torch.ones(C, device=DEV), torch.rand(700, device=DEV), torch.empty_like(x), torch.empty(C, device=DEV)

    small, large = case(64), case(8192)
    norm.rms_norm_bwd(*small)
    want = small[4].clone(), small[5].clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        norm.rms_norm_bwd(*small)
        held = norm.workspace(64, DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            norm.rms_norm_bwd(*small)
        for _ in range(2):
            norm.rms_norm_bwd(*large)
            assert norm.workspace(64, DEV) is held and norm.workspace(8192, DEV) is not held
            small[4].zero_(), small[5].zero_()
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(small[4], want[0]) and torch.equal(small[5], want[1])


def test_graph_capture(cuda_lib):
    """Forward, e4m3 form and backward in one graph that reads its inputs anew."""
    from objectsam_b200 import norm
    g = torch.Generator(device=DEV).manual_seed(7)
    R, C = 300, 264
    x, r, dy = (torch.randn(R, C, generator=g, device=DEV).half() for _ in range(3))
    w = torch.rand(C, generator=g, device=DEV)
    new = lambda: dict(y=torch.zeros_like(x), h=torch.zeros_like(x), rstd=torch.zeros(R, device=DEV), dx=torch.zeros_like(x),  # noqa: E731
                       dw=torch.zeros(C, device=DEV), q=torch.zeros(R, C, device=DEV).to(torch.float8_e4m3fn), qs=torch.zeros(R, 3, device=DEV))

    def step(o):
        norm.rms_norm_fwd(x, w, EPS, o["y"], res=r, total=o["h"], rstd=o["rstd"])
        norm.rms_norm_fwd_q8(x, w, EPS, o["q"], o["qs"], res=r)
        norm.rms_norm_bwd(dy, o["h"], w, o["rstd"], o["dx"], o["dw"])

    got = new()
    step(got)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(got)
    for by in (1.0, 0.5):
        x.mul_(by)
        graph.replay()
        want = new()
        step(want)
        torch.cuda.synchronize()
        for n in got:
            assert torch.equal(got[n].view(torch.uint8), want[n].view(torch.uint8)), n
