"""Attention (osam_attn_fwd / osam_attn_bwd) against the 64-bit restatement oracle/token_ref.py.

Tolerances: token_ref.attention's elementwise bounds for one rounding of P, dS, o and the outputs to the 16-bit type,
times 1.3 for what is exact there and fp32 here (score sums, exponentials: relative 2^-16 at most on these scores, below
a third of bf16's and fp16's units after the sum), plus 2^-20 of the largest value for results near zero."""
import math

import pytest
import torch

from objectsam_b200 import _lib
from oracle import token_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(B, Lq, Lk, Hq, Hk, D, dtype=torch.float16, seed=0, fused=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    if fused:
        qkv = r(B, Lq, Hq + 2 * Hk, D)
        q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
    else:
        q, k, v = r(B, Lq, Hq, D), r(B, Lk, Hk, D), r(B, Lk, Hk, D)
    return q * 2 if not fused else q, k, v, r(B, Lq, Hq, D)


def slopes_of(Hq):
    return torch.tensor([2.0 ** (-1 - h) for h in range(Hq)], device=DEV)


def close(x, ref, tol, what):
    x, ref = x.double().cpu(), ref.cpu()
    if not ref.numel():
        return
    lim = 1.3 * tol.cpu() + 2.0 ** -20 * ref.abs().max()
    bad = ~((x - ref).abs() <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((x - ref).abs() / lim).max():.3g}×"


def run(q, k, v, do, *, train=True, scale=None, cap=0.0, mask="none", grid_w=0, slopes=None, lens=None, prefix=None,
        doc_q=None, doc_k=None, stream=None):
    from objectsam_b200.attn import AttnGeom, AttnOp
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1:3]
    op = AttnOp().init(AttnGeom(B, Lq, Lk, Hq, Hk, D, q.dtype), scale=scale, cap=cap, mask=mask, grid_w=grid_w,
                       slopes=slopes, lens=lens, prefix=prefix, doc_q=doc_q, doc_k=doc_k)
    nan = float("nan")
    ws = torch.full((max(op.workspace_size(), 256),), 255, dtype=torch.uint8, device=DEV)
    out = {"o": torch.full_like(q, nan, memory_format=torch.contiguous_format),
           "lse": torch.full((B, Hq, Lq), nan, device=DEV)}
    op.fwd(q, k, v, out["o"], out["lse"], ws=ws, stream=stream)
    if train:
        out |= {"dq": torch.full(q.shape, nan, dtype=q.dtype, device=DEV), "dk": torch.full(k.shape, nan, dtype=q.dtype, device=DEV),
                "dv": torch.full(k.shape, nan, dtype=q.dtype, device=DEV)}
        op.bwd(q, k, v, out["o"], out["lse"], do, out["dq"], out["dk"], out["dv"], ws=ws, stream=stream)
    torch.cuda.synchronize()
    return out


def check(q, k, v, do, *, train=True, scale=None, cap=0.0, mask="none", grid_w=0, slopes=None, lens=None, prefix=None,
          doc_q=None, doc_k=None):
    B, Lq, Hq, D = q.shape
    Lk = k.shape[1]
    out = run(q, k, v, do, train=train, scale=scale, cap=cap, mask=mask, grid_w=grid_w, slopes=slopes, lens=lens,
              prefix=prefix, doc_q=doc_q, doc_k=doc_k)
    vis = token_ref.attn_visible(B, Lq, Lk, mask, lens, prefix, doc_q, doc_k)
    dist = token_ref.attn_distance(B, Lq, Lk, grid_w, lens)
    ref = token_ref.attention(q.double(), k.double(), v.double(), vis, scale or 1 / math.sqrt(D), cap,
                              None if slopes is None else slopes.double(), dist, do.double() if train else None,
                              UNIT[q.dtype])
    close(out["o"], ref["o"], ref["tol_o"], "o")
    # lse: the scores' fp32 sums (D terms) and the row's sum
    lse, want = out["lse"].double().cpu(), ref["lse"].cpu()
    assert torch.equal(lse == -math.inf, want == -math.inf)
    fine = want != -math.inf
    lim = float(ref["score_sum"]) * D * 2.0 ** -23 + 2.0 ** -17
    if fine.any():
        assert (lse - want)[fine].abs().max() <= lim
    if train:
        for name in ("dq", "dk", "dv"):
            close(out[name], ref[name], ref["tol_" + name], name)
    return out


# ---------------------------------------------------------------- lengths and head layouts
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 2), (2, 1), (7, 129), (64, 64), (65, 63), (127, 128), (128, 129), (200, 333),
                                   (257, 255), (400, 400), (513, 640)])
def test_lengths(cuda_lib, Lq, Lk):
    check(*make(2, Lq, Lk, 2, 2, 64, seed=Lq * 1000 + Lk))


@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 56, 64, 72, 80, 96, 120, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_dims(cuda_lib, D, dtype):
    check(*make(1, 150, 200, 2, 1, D, dtype, seed=D), mask="causal")


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (3, 1), (6, 2), (5, 5), (8, 2), (16, 1), (130, 1)])
@pytest.mark.parametrize("Lq", [1, 2, 77])
def test_shared_heads(cuda_lib, Hq, Hk, Lq):
    check(*make(2, Lq, 190, Hq, Hk, 64 if Hq < 100 else 32, seed=Hq), mask="causal")


# ---------------------------------------------------------------- scores and masks
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cap", [0.0, 2.0, 30.0])
@pytest.mark.parametrize("bias", ["none", "line", "grid"])
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
def test_scores(cuda_lib, D, dtype, cap, bias, mask):
    B, H, W = 2, 13, 15
    L = H * W
    check(*make(B, L, L, 4, 2, D, dtype, seed=3, fused=True), cap=cap, mask=mask,
          slopes=None if bias == "none" else slopes_of(4), grid_w=W if bias == "grid" else 0,
          prefix=torch.tensor([0, 150], dtype=torch.int32, device=DEV) if mask == "prefix" else None)


@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
@pytest.mark.parametrize("Hq,Hk,D", [(2, 2, 64), (6, 2, 32), (4, 1, 128)])
def test_documents(cuda_lib, mask, Hq, Hk, D):
    """Uneven documents, tokens of none, ids out of order and repeated, a sequence without any document; what the
    tokens without a document hold is NaN."""
    B, L = 3, 391
    q, k, v, do = make(B, L, L, Hq, Hk, D, seed=11)
    doc = torch.full((B, L), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate((100, 3, 1, 129, 64, 60)):
        doc[0, at:at + n] = 5 - i
        at += n
    doc[1] = torch.randint(-1, 3, (L,), generator=torch.Generator().manual_seed(1))
    for t in (q, k, v, do):
        t[(doc < 0).to(DEV)] = float("nan")
    doc = doc.to(DEV)
    check(q, k, v, do, mask=mask, doc_q=doc, doc_k=doc, cap=5.0 if D == 32 else 0.0, slopes=slopes_of(Hq) if D == 64 else None,
          prefix=torch.tensor([130, 0, 391], dtype=torch.int32, device=DEV) if mask == "prefix" else None)


def test_documents_across(cuda_lib):
    """Queries and keys with documents of their own (cross attention), another length on each side."""
    q, k, v, do = make(2, 140, 300, 4, 2, 64, seed=5)
    dq = torch.arange(140, dtype=torch.int32, device=DEV).div(50, rounding_mode="floor").int().expand(2, -1).contiguous()
    dk = torch.arange(300, dtype=torch.int32, device=DEV).div(70, rounding_mode="floor").int().expand(2, -1).contiguous()
    check(q, k, v, do, doc_q=dq, doc_k=dk)


@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
@pytest.mark.parametrize("grid_w", [0, 9])
def test_lens(cuda_lib, mask, grid_w):
    """Keys in use of each sequence: none, one, fewer than the queries, more than the cache; what lies past them is
    NaN or infinite."""
    lens = torch.tensor([0, 1, 5, 130, 300, 9999, -3], dtype=torch.int32, device=DEV)
    B, Lq, Lk = len(lens), 20, 300
    q, k, v, do = make(B, Lq, Lk, 4, 2, 64, seed=8)
    for b, n in enumerate(lens.clamp(0, Lk).tolist()):
        k[b, n:] = float("nan")
        v[b, n:] = float("inf")
    check(q, k, v, do, mask=mask, lens=lens, slopes=slopes_of(4), grid_w=grid_w,
          prefix=torch.tensor([3] * B, dtype=torch.int32, device=DEV) if mask == "prefix" else None)


@pytest.mark.parametrize("Lq,Lk,Hq,Hk,D", [(1, 517, 8, 8, 64), (1, 4096, 4, 1, 128), (3, 1025, 6, 2, 40), (1, 20000, 2, 1, 64),
                                           (40, 3000, 2, 2, 64)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_tokens_over_a_cache(cuda_lib, Lq, Lk, Hq, Hk, D, cap):
    """Few queries: the keys are split and joined; uneven caches leave splits without a key."""
    q, k, v, do = make(3, Lq, Lk, Hq, Hk, D, seed=Lk)
    lens = torch.tensor([Lk, Lk // 3, 2], dtype=torch.int32, device=DEV)
    check(q, k, v, do, mask="causal", lens=lens, cap=cap, slopes=slopes_of(Hq), train=Lk < 5000)


@pytest.mark.parametrize("lens,Lk,Hq,Hk", [([5000, 3, 0, 1, 64, 65], 5000, 4, 2), ([0, 0, -1], 900, 2, 2),
                                           ([1100] * 36, 1100, 2, 1), ([7 * i for i in range(140)], 960, 2, 2),
                                           ([9000, 1024, 5555, 9001, 700], 9001, 6, 3)])
@pytest.mark.parametrize("Lq", [1, 70])
def test_caches_of_any_lengths(cuda_lib, lens, Lk, Hq, Hk, Lq):
    """The splits follow the sequences' own lengths: more sequences than a warp, one long beside short ones, none."""
    q, k, v, do = make(len(lens), Lq, Lk, Hq, Hk, 64, seed=Lk + Lq)
    lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for b, n in enumerate(lens.clamp(0, Lk).tolist()):
        k[b, n:] = float("nan")
        v[b, n:] = float("nan")
    check(q, k, v, do, mask="causal", lens=lens, train=False)


def test_split_documents(cuda_lib):
    q, k, v, do = make(1, 2, 5000, 2, 1, 64, seed=2)
    dk = torch.arange(5000, dtype=torch.int32, device=DEV).div(600, rounding_mode="floor").int()[None].contiguous()
    check(q, k, v, do, doc_q=torch.tensor([[3, -1]], dtype=torch.int32, device=DEV), doc_k=dk)


def test_many_heads(cuda_lib):
    """Causal calls whose keys and values pass L2 go over the heads in groups: the same results as in two halves."""
    t = make(64, 400, 400, 16, 16, 128, seed=4)
    whole = run(*t, mask="causal")
    for part in (slice(0, 32), slice(32, 64)):
        half = run(*(x[part] for x in t), mask="causal")
        for name, x in half.items():
            assert torch.equal(whole[name][part], x), name


# ---------------------------------------------------------------- ranges
def test_growing_scores(cuda_lib):
    """Row maxima that grow by far more than the lazy rescale's bound from tile to tile, and shrink again."""
    q, k, v, do = make(1, 256, 900, 2, 1, 64, seed=4)
    k *= torch.linspace(0.05, 3.0, 900, device=DEV).half()[None, :, None, None]
    check(q, k, v, do)
    check(q, k.flip(1), v, do)


def test_gradients_scale_with_do(cuda_lib):
    """The backward is linear in dO, and its power of two follows dO's size: with dO·2^-12 every step before the last
    rounding is the same times 2^-12, though fp16 could not hold dS as it stands.  So the results differ by the two
    roundings alone: 2^-11 relative in all, and half of fp16's smallest step, 2^-25·2^12.  dO is a multiple of 2^-6
    (exact on both sides)."""
    q, k, v, do = make(1, 300, 1500, 2, 2, 64, seed=6)
    do = (do.float() * 64).round().div(64).half()
    big, small = run(q, k, v, do), run(q, k, v, do * 2.0 ** -12)
    for n in ("dq", "dk", "dv"):
        x, y = big[n].double(), small[n].double() * 2.0 ** 12
        assert ((x - y).abs() <= 2.0 ** -11 * x.abs() * 1.001 + 2.0 ** -13).all(), n


def test_large_gradients(cuda_lib):
    q, k, v, do = make(1, 130, 200, 2, 1, 64, seed=7)
    check(q, k, v, do * 512)


def test_nan_stays_in_its_row(cuda_lib):
    """A query that holds NaN gives NaN in its own output row and nowhere else."""
    q, k, v, do = make(1, 200, 200, 1, 1, 64, seed=9)
    q[0, 77, 0, 3] = float("nan")
    o = run(q, k, v, do, train=False)["o"]
    assert torch.isnan(o[0, 77]).all() and torch.isfinite(o[0, :77]).all() and torch.isfinite(o[0, 78:]).all()


# ---------------------------------------------------------------- strides, streams, order
def test_strides_and_orders(cuda_lib):
    """Head-major storage, spare heads and tokens between, a batch of stride 0 nowhere: same numbers as packed."""
    B, L, H, D = 2, 150, 3, 48
    q, k, v, do = make(B, L, L, H, H, D, seed=12)
    base = run(q, k, v, do, mask="causal")
    hm = lambda t: t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # noqa: E731

    def wide(t):
        w = torch.full((B, L + 5, H + 2, D + 8), float("nan"), dtype=t.dtype, device=DEV)
        w[:, 2:L + 2, 1:H + 1, 8:] = t
        return w[:, 2:L + 2, 1:H + 1, 8:]

    for f in (hm, wide):
        got = run(f(q), f(k), f(v), f(do), mask="causal")
        for n in base:
            assert torch.equal(got[n], base[n]), n


def test_same_result_every_time(cuda_lib):
    q, k, v, do = make(2, 300, 300, 8, 2, 128, torch.bfloat16, seed=13)
    first = run(q, k, v, do, mask="causal", cap=10.0)
    for _ in range(5):
        again = run(q, k, v, do, mask="causal", cap=10.0)
        for n in first:
            assert torch.equal(first[n], again[n]), n


def test_other_stream(cuda_lib):
    """A call on a stream of its own, behind work that is still writing its inputs there."""
    q, k, v, do = make(1, 500, 500, 2, 2, 64, seed=14)
    base = run(q, k, v, do)
    s = torch.cuda.Stream()
    q2, big = torch.empty_like(q), torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            big = big @ big * 1e-3
        q2.copy_(q)
    got = run(q2, k, v, do, stream=s)
    for n in base:
        assert torch.equal(got[n], base[n]), n


def test_graph_capture(cuda_lib):
    from objectsam_b200.attn import AttnGeom, AttnOp
    q, k, v, do = make(1, 1, 2000, 4, 4, 64, seed=15)
    lens = torch.tensor([700], dtype=torch.int32, device=DEV)
    op = AttnOp().init(AttnGeom(1, 1, 2000, 4, 4, 64), mask="causal", lens=lens)
    o, ws = torch.empty_like(q), torch.empty(op.workspace_size(), dtype=torch.uint8, device=DEV)
    op.fwd(q, k, v, o, ws=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.fwd(q, k, v, o, ws=ws)
    for n in (1, 700, 1999):  # the plan reads the lengths anew at every call
        lens.fill_(n)
        g.replay()
        torch.cuda.synchronize()
        want = run(q, k, v, do, train=False, mask="causal", lens=torch.tensor([n], dtype=torch.int32, device=DEV))["o"]
        assert torch.equal(o, want)


def test_gradients_against_differences(cuda_lib):
    """(L(x + εd) − L(x − εd)) / 2ε of the kernel's own forward, L = Σ o·do, along d = sign of the gradient, against
    Σ|gradient|.  Inputs and steps are multiples of 2^-8 (exact in fp16); the forward's rounding gives L a noise of
    2^-11·√N·|o·do| ≈ 0.06 against differences of tens, the step's third-order term stays under 2 %."""
    B, L, Hq, Hk, D = 1, 96, 4, 2, 32
    q, k, v, do = make(B, L, L, Hq, Hk, D, seed=16)
    grid = lambda t: (t.float() * 64).round().div(64).half()  # noqa: E731
    q, k, v = grid(q), grid(k), grid(v)
    kw = dict(mask="causal", cap=4.0, slopes=slopes_of(Hq))
    out = run(q, k, v, do, **kw)
    eps = 2.0 ** -6
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        d = torch.sign(out[name].float())
        loss = []
        for sgn in (1, -1):
            moved = (t.float() + sgn * eps * d).half()
            a = dict(q=q, k=k, v=v)
            a[name[1]] = moved
            o = run(a["q"], a["k"], a["v"], do, train=False, **kw)["o"]
            loss.append((o.double() * do.double()).sum().item())
        got, want = (loss[0] - loss[1]) / (2 * eps), out[name].double().abs().sum().item()
        assert abs(got - want) <= 0.03 * want, (name, got, want)


def test_empty(cuda_lib):
    for Lq, Lk in ((0, 5), (5, 0), (0, 0)):
        q, k, v, do = make(2, Lq, Lk, 2, 2, 64)
        out = run(q, k, v, do)
        for n in ("o", "dq", "dk", "dv"):
            assert (out[n] == 0).all(), n
        assert (out["lse"] == -math.inf).all()
    q, k, v, do = make(0, 4, 4, 2, 2, 64)
    run(q, k, v, do)


def test_refusals_with_tensors(cuda_lib):
    from objectsam_b200.attn import AttnGeom, AttnOp
    q, k, v, do = make(2, 16, 16, 2, 2, 64)
    op = AttnOp().init(AttnGeom(2, 16, 16, 2, 2, 64))
    o = torch.empty_like(q)
    ws = torch.empty(op.workspace_size(), dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError):
        op.fwd(q.float(), k, v, o, ws=ws)
    with pytest.raises(ValueError):
        op.fwd(q[:, :8], k, v, o, ws=ws)
    with pytest.raises(ValueError):
        op.fwd(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, o, ws=ws)
    with pytest.raises(_lib.OsamError):  # a batch of stride 0
        op.fwd(q, k[:1].expand(2, -1, -1, -1), v, o, ws=ws)
    with pytest.raises(_lib.OsamError):  # 8-byte alignment
        flat = torch.zeros(q.numel() + 4, dtype=q.dtype, device=DEV)
        op.fwd(flat[4:].view(q.shape), k, v, o, ws=ws)
    with pytest.raises(_lib.OsamError):  # short workspace
        op.fwd(q, k, v, o, ws=ws[:8])
    with pytest.raises(_lib.OsamError):  # strides of 12 elements
        flat = torch.zeros(2 * 16 * 2 * 76, dtype=q.dtype, device=DEV)
        op.fwd(torch.as_strided(flat, (2, 16, 2, 64), (16 * 2 * 76, 2 * 76, 76, 1)), k, v, o, ws=ws)


@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
@pytest.mark.parametrize("D", [40, 128])
def test_long_rows_of_few_heads(cuda_lib, mask, D):
    """Few tiles and long rows: a key tile's queries (and a query tile's keys) are shared among CTAs and summed."""
    L = 1150
    q, k, v, do = make(1, L, L, 4, 1, D, seed=17)
    doc = torch.arange(L, dtype=torch.int32, device=DEV).div(500, rounding_mode="floor").int()[None].contiguous()
    check(q, k, v, do, mask=mask, doc_q=doc, doc_k=doc,
          prefix=torch.tensor([600], dtype=torch.int32, device=DEV) if mask == "prefix" else None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bias", ["none", "line", "grid"])
@pytest.mark.parametrize("tiles", [2, 3, 4])
def test_documents_of_a_few_tiles(cuda_lib, D, bias, tiles):
    """Key tiles that compare ids alternate with tiles of one document: the same bits every time, and the masks' results."""
    B, L = 2, 1000
    q, k, v, do = make(B, L, L, 4, 2, D, seed=18)
    doc = (torch.arange(L, device=DEV) + 32).div(64 * tiles, rounding_mode="floor").int().expand(B, -1).contiguous()
    kw = dict(doc_q=doc, doc_k=doc, slopes=None if bias == "none" else slopes_of(4), grid_w=25 if bias == "grid" else 0)
    first = check(q, k, v, do, **kw)
    for _ in range(10):
        again = run(q, k, v, do, **kw)
        for n in first:
            assert torch.equal(first[n], again[n]), n


# ---------------------------------------------------------------- sizes of v
@pytest.mark.parametrize("mask", ["none", "causal"])
def test_two_keys_of_opposite_values(cuda_lib, mask):
    """p = ½ on v = +8 and −8 at 128 dims: dS = ±512 in fp16, twice what dO's size alone would leave room for."""
    q, k, v, do = make(2, 3, 2, 2, 1, 128, seed=21)
    q.zero_(), do.fill_(1.0)
    v[:, 0], v[:, 1] = 8.0, -8.0
    check(q, k, v, do, mask=mask)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [2.0 ** -8, 256.0, 1024.0])
@pytest.mark.parametrize("mask", ["none", "causal"])
def test_size_of_v(cuda_lib, D, dtype, size, mask):
    """dP and dS grow with v; a row of large values that nothing may see changes nothing.  dO brings the gradients of queries and
    keys to one size, within fp16's normal numbers, where the bounds hold."""
    q, k, v, do = make(1, 200, 230, 4, 2, D, dtype, seed=22)
    doc_q, doc_k = (torch.zeros(1, n, dtype=torch.int32, device=DEV) for n in (200, 230))
    doc_k[0, 100] = -1
    v *= size
    v[0, 100] = 60000.0
    check(q, k, v, do * (16 if size < 1 else 1 / 64), mask=mask, doc_q=doc_q, doc_k=doc_k)


# ---------------------------------------------------------------- large caps
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cap", [100.0, 150.0, 1e4, 1e7, 3e38])
@pytest.mark.parametrize("bias", ["none", "line", "grid"])
def test_large_caps(cuda_lib, D, dtype, cap, bias):
    """A cap far above the scores leaves them as they are."""
    H, W = 13, 15
    q, k, v, do = make(1, H * W, H * W, 4, 2, D, dtype, seed=23)
    check(q, k, v, do, cap=cap, mask="causal", slopes=None if bias == "none" else slopes_of(4), grid_w=W if bias == "grid" else 0)


@pytest.mark.parametrize("cap", [50.0, 128.0, 129.0, 200.0, 1000.0])
@pytest.mark.parametrize("Lq", [1, 90])
def test_scores_near_a_large_cap(cuda_lib, cap, Lq):
    """Scores up to twice the cap and a row's largest just below it: whole products, exact in fp32, so that only the cap's form
    is in the error (4e-7 of a score of at most 1000: below the 0.3 of a rounding unit that `check` leaves for it with bf16)."""
    g = torch.Generator().manual_seed(24)
    Lk, D = 200, 64
    q = torch.randint(1, 4, (1, Lq, 2, D), generator=g).to(torch.bfloat16).to(DEV)
    k = torch.randint(-8, 9, (1, Lk, 2, D), generator=g).to(torch.bfloat16).to(DEV)
    k[0, ::3] = k[0, ::3].abs()
    v, do = (torch.randn(1, n, 2, D, generator=g).to(torch.bfloat16).to(DEV) for n in (Lk, Lq))
    check(q, k, v, do, cap=cap, scale=2.0 ** round(math.log2(cap / 500)))


# ---------------------------------------------------------------- slopes of either sign
@pytest.mark.parametrize("cap", [0.0, 20.0, 1e4])
@pytest.mark.parametrize("bias", ["line", "grid"])
@pytest.mark.parametrize("mask", ["none", "prefix"])
@pytest.mark.parametrize("Lq", [3, 195])
def test_slopes_of_either_sign(cuda_lib, cap, bias, mask, Lq):
    """A negative slope favours distant keys: s − slope·distance as it stands."""
    H, W = 13, 15
    q, k, v, do = make(2, Lq, H * W, 4, 2, 64, seed=25)
    slopes = torch.tensor([-0.06, 0.11, 0.0, -0.01], device=DEV)
    check(q, k, v, do, cap=cap, mask=mask, slopes=slopes, grid_w=W if bias == "grid" else 0,
          prefix=torch.tensor([0, 150], dtype=torch.int32, device=DEV) if mask == "prefix" else None)


@pytest.mark.parametrize("Lq", [1, 40, 200])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_small_weights(cuda_lib, Lq, dtype):
    """One key of weight 1 with v = 0 and 700 of weight 2^-26 with v = 60000: o is what the small ones add up to.  The weights
    are powers of two that fp16 holds with a shift of 2^2 and more, so o's rounding is the only one, and 2^-11 covers the
    score's (−26·ln 2·log2 e, off by 2^-23 of 26)."""
    D, N = 8, 700
    q, k, v = (torch.zeros(1, n, 1, D, dtype=dtype, device=DEV) for n in (Lq, N + 1, N + 1))
    q[..., 0], k[:, 1:, :, 0], v[:, 1:] = 1.0, -26.0, 60000.0
    out = run(q, k, v, None, train=False, scale=math.log(2.0))
    want = float(v[0, 1, 0, 0]) * N * 2.0 ** -26 / (1 + N * 2.0 ** -26)
    assert ((out["o"].double() - want).abs() <= (UNIT[dtype] + 2.0 ** -11) * want).all(), (out["o"].double().mean().item(), want)
    assert (out["lse"].double() - math.log(1 + N * 2.0 ** -26)).abs().max() <= 2.0 ** -20


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mask", ["causal", "prefix"])
def test_contents_of_queries_that_see_nothing(cuda_lib, D, dtype, mask):
    """Queries in front of the first key (fewer keys than queries), or of a document that no key has: q and dO may hold NaN or
    infinities there, and the keys' gradients are those of the other queries."""
    lens = torch.tensor([150, 3, 0, 90], dtype=torch.int32, device=DEV)
    B, Lq, Lk = len(lens), 150, 160
    q, k, v, do = make(B, Lq, Lk, 4, 2, D, dtype, seed=26)
    for b, n in enumerate(lens.tolist()):
        q[b, :Lq - n] = float("nan")
        do[b, :Lq - n] = float("inf")
    check(q, k, v, do, mask=mask, lens=lens, prefix=torch.zeros(B, dtype=torch.int32, device=DEV) if mask == "prefix" else None)
    q, k, v, do = make(1, Lq, Lk, 4, 2, D, dtype, seed=27)
    dq, dk = (torch.arange(n, dtype=torch.int32, device=DEV).div(40, rounding_mode="floor").int()[None].contiguous() for n in (Lq, Lk))
    dq[0, 20:30], dq[0, 70:100] = 77, 78
    q[0, 20:30], do[0, 70:100] = float("nan"), float("nan")
    check(q, k, v, do, doc_q=dq, doc_k=dk)


def test_without_a_workspace(cuda_lib):
    """The plan's own workspace, on the current stream and on another, forward and backward."""
    from objectsam_b200.attn import AttnGeom, AttnOp
    q, k, v, do = make(2, 40, 900, 4, 2, 64, seed=28)
    want = run(q, k, v, do, mask="causal")
    op = AttnOp().init(AttnGeom(2, 40, 900, 4, 2, 64), mask="causal")
    for s in (None, torch.cuda.Stream()):
        out = {n: torch.full_like(t, float("nan")) for n, t in want.items()}
        torch.cuda.synchronize()
        op.fwd(q, k, v, out["o"], out["lse"], stream=s)
        op.bwd(q, k, v, out["o"], out["lse"], do, out["dq"], out["dk"], out["dv"], stream=s)
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(out[n], want[n]), n
    assert len(op._ws) == 2


def test_graph_capture_of_a_training_step(cuda_lib):
    """Forward and backward in one graph, over documents that the plan reads anew, on the plan's own workspace."""
    from objectsam_b200.attn import AttnGeom, AttnOp
    q, k, v, do = make(2, 300, 300, 4, 2, 64, seed=29)
    doc = torch.zeros(2, 300, dtype=torch.int32, device=DEV)
    op = AttnOp().init(AttnGeom(2, 300, 300, 4, 2, 64), mask="causal", doc_q=doc, doc_k=doc)
    out = {"o": torch.empty_like(q), "lse": torch.empty(2, 4, 300, device=DEV), "dq": torch.empty_like(q),
           "dk": torch.empty_like(k), "dv": torch.empty_like(v)}

    def step():
        op.fwd(q, k, v, out["o"], out["lse"])
        op.bwd(q, k, v, out["o"], out["lse"], do, out["dq"], out["dk"], out["dv"])

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for cut in (300, 130, 1):
        doc[:, cut:] = 1
        for t in out.values():
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        want = run(q, k, v, do, mask="causal", doc_q=doc, doc_k=doc)
        for n in out:
            assert torch.equal(out[n], want[n]), (cut, n)


def test_offsets_past_32_bits(cuda_lib):
    """A cache whose second sequence lies past 2^31 elements, one of whose heads and tokens are spread as far: the same bits
    as over a small copy of the rows in use."""
    Lk, Hk, D, n = 40_000, 448, 128, 130
    cache = torch.empty(2, Lk, Hk, D, dtype=torch.bfloat16, device=DEV)  # 4.6e9 elements
    assert cache.stride(0) > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(30)
    q, do = (torch.randn(2, 3, 4, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    k, v = cache[:, :, 5:9:2], cache[:, :, Hk - 2:]
    for t in (k, v):
        t[:, :n] = torch.randn(2, n, 2, D, generator=g, device=DEV).bfloat16()
        t[1, Lk - 900:] = torch.randn(900, 2, D, generator=g, device=DEV).bfloat16()
    lens = torch.tensor([n, n], dtype=torch.int32, device=DEV)
    big = run(q, k, v, do, train=False, mask="causal", lens=lens)
    small = run(q, k[:, :n].contiguous(), v[:, :n].contiguous(), do, train=False, mask="causal", lens=lens)
    assert (big["o"].double() - small["o"].double()).abs().max() <= 2.0 ** -7 * small["o"].double().abs().max()
    assert (big["lse"] - small["lse"]).abs().max() <= 2.0 ** -17
    # forward and backward over a window at the far end, whose gradients go to views as wide
    k, v = k[1:, Lk - 900:], v[1:, Lk - 900:]
    got, want = run(q[1:], k, v, do[1:]), run(q[1:], k.contiguous(), v.contiguous(), do[1:])
    for x in want:
        assert torch.equal(got[x], want[x]), x


@pytest.mark.parametrize("bias", ["line", "grid"])
@pytest.mark.parametrize("docs", [False, True])
def test_slopes_of_either_sign_in_one_tile(cuda_lib, bias, docs):
    """More heads to a key head than a warp has rows: warps of one tile with and without a negative slope keep step."""
    q, k, v, do = make(1, 5, 300, 130, 1, 32, seed=31)
    slopes = torch.full((130,), 0.02, device=DEV)
    slopes[40:45], slopes[100:] = -0.03, -0.01
    dq, dk = (torch.arange(n, dtype=torch.int32, device=DEV).div(n // 2, rounding_mode="floor").int()[None].contiguous() for n in (5, 300))
    check(q, k, v, do, slopes=slopes, grid_w=20 if bias == "grid" else 0, doc_q=dq if docs else None, doc_k=dk if docs else None)
