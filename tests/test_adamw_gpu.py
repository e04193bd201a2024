"""osam_adamw_* against the 64-bit restatement (oracle/token_ref.adamw).

Tolerances: with 32-bit states every intermediate is one fp32 rounding of positive-and-negative sums of two terms:
|Δm|, |Δv| ≤ 2^-21 of the terms' sizes, |Δp| ≤ 2^-22·|p| + 2^-18·|step|.  8-bit states come back within half an e4m3 step
(2^-4 of the value, 2^-10 of the scale below the normal range) of the moments that the step used; for those the test feeds
the kernel's own stored states into the restatement."""
import math

import pytest
import torch

from oracle import token_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
SIZES = [1, 2, 7, 8, 63, 64, 65, 255, 256, 257, 2047, 2048, 2049, 5000, 100_003]


def tensors(sizes, grad=torch.float32, copy=torch.float16, packed=False, seed=0, level=1e-2):
    """Parameters, gradients and copies: on their own, or as slices without gaps of one array each."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    if packed:  # one element in front: nothing is aligned
        n = sum(sizes) + 1
        cut = lambda t: [t[1 + sum(sizes[:i]):1 + sum(sizes[:i + 1])] for i in range(len(sizes))]  # noqa: E731
        p, gr = cut(torch.randn(n, generator=g, device=DEV)), cut((torch.randn(n, generator=g, device=DEV) * level).to(grad))
        c = cut(torch.zeros(n, dtype=copy, device=DEV)) if copy else None
    else:
        p = [torch.randn(n, generator=g, device=DEV) for n in sizes]
        gr = [(torch.randn(n, generator=g, device=DEV) * level).to(grad) for n in sizes]
        c = [torch.zeros(n, dtype=copy, device=DEV) for n in sizes] if copy else None
    return p, gr, c


def states(opt, sizes):
    """Each tensor's (m, v) as float64, from the optimizer's arrays."""
    U = 256 if opt.bits == 8 else 64
    at, out = 0, []
    for n in sizes:
        e = at + -(-n // U) * U
        m, v = opt.m[at:e].double(), opt.v[at:e].double()
        if opt.bits == 8:
            m = (m.view(-1, U) * opt.m_scale[at // U:e // U].double()[:, None]).view(-1)
            v = (v.view(-1, U) * opt.v_scale[at // U:e // U].double()[:, None]).view(-1).square()
        assert not m[n:].any() and not v[n:].any()
        out.append((m[:n], v[:n]))
        at = e
    assert at == opt.m.numel()
    return out


def run(sizes, bits, grad, copy, packed, clip, steps=4, grad_scale=1.0):
    from objectsam_b200.optim import AdamW
    kw = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    p, g, c = tensors(sizes, grad, copy, packed)
    decay = [i % 2 == 0 for i in range(len(sizes))]
    opt = AdamW(p, g, copies=c, bits=bits, decay=decay, **kw)
    gen = torch.Generator(device=DEV).manual_seed(9)
    for t in range(1, steps + 1):
        for x in g:
            x.copy_(torch.randn(x.numel(), generator=gen, device=DEV) * 10.0 ** -t)
        before, old = [x.double().clone() for x in p], states(opt, sizes)
        opt.step(max_norm=clip, grad_scale=grad_scale)
        mul = grad_scale
        if clip:
            norm = grad_scale * math.sqrt(sum(float(x.double().square().sum()) for x in g))
            assert abs(opt.norm.item() - norm) <= 2.0 ** -18 * norm
            mul *= min(1.0, clip / (norm + 1e-6))
        new = states(opt, sizes)
        at = 0
        for i, n in enumerate(sizes):
            want, m, v = token_ref.adamw(before[i], g[i].double(), *old[i], t, decay=decay[i], mul=mul, **kw)
            step = (want - before[i]).abs()
            lim = 2.0 ** -22 * before[i].abs() + 2.0 ** -18 * (step + kw["lr"]) + (2.0 ** -16 * step if clip else 0)
            assert ((p[i].double() - want).abs() <= lim).all(), (t, i)
            if c:
                assert torch.equal(c[i], p[i].to(copy)), (t, i)
            msize = 0.9 * old[i][0].abs() + 0.1 * (g[i].double() * mul).abs()
            if bits == 32:
                assert ((new[i][0] - m).abs() <= 2.0 ** -18 * msize).all() and ((new[i][1] - v).abs() <= 2.0 ** -18 * v).all()
                continue
            U, k = 256, -(-n // 256)
            blocks = lambda a: torch.nn.functional.pad(a, (0, k * U - n)).view(k, U)  # noqa: E731
            for x, got, sc in ((m, new[i][0], opt.m_scale), (v.sqrt(), new[i][1].sqrt(), opt.v_scale)):
                s = sc[at:at + k].double()[:, None]
                top = blocks(x).abs().amax(1, keepdim=True)
                assert ((s - top / 448).abs() <= 2.0 ** -17 * top / 448).all()
                least = 2.0 ** -9 if x is not m else 2.0 ** -10  # a root above zero keeps at least the smallest value
                lim = torch.maximum(2.0 ** -4 * blocks(x).abs(), least * s) * (1 + 2.0 ** -8) + 2.0 ** -16 * top
                assert ((blocks(got) - blocks(x)).abs() <= lim).all(), (t, i)
            assert ((new[i][1] > 0) == (v > 0)).all()
            at += k
    return opt


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_steps(cuda_lib, bits, grad, packed, clip):
    run(SIZES, bits, grad, torch.float16, packed, clip)


@pytest.mark.parametrize("copy", [None, torch.bfloat16])
def test_copies(cuda_lib, copy):
    run([300, 5000], 32, torch.float32, copy, False, None)
    run([300, 5000], 8, torch.float32, copy, True, 1.0)


def test_one_element_and_scaled_gradients(cuda_lib):
    run([1], 8, torch.float32, None, False, 0.1)
    run([4096], 32, torch.float16, torch.float16, False, 1.0, grad_scale=1 / 128)
    run([4096], 32, torch.float16, torch.float16, False, None, grad_scale=1 / 128)


def test_many_tensors(cuda_lib):
    run([(i * 37) % 500 + 1 for i in range(700)], 8, torch.float32, torch.float16, True, 1.0, steps=2)


def test_no_elements_among_others(cuda_lib):
    run([0, 5, 0, 300], 8, torch.float32, None, False, 1.0, steps=2)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_gradient_that_is_not_finite_skips_the_step(cuda_lib, bits, bad):
    from objectsam_b200.optim import AdamW
    p, g, c = tensors([1000, 3000])
    opt = AdamW(p, g, copies=c, bits=bits)
    opt.step(max_norm=1.0)
    keep = [t.clone() for t in (*p, *c, opt.m.view(torch.uint8), opt.v.view(torch.uint8))]
    g[1][2999] = bad
    opt.step(max_norm=1.0)
    assert not math.isfinite(opt.norm.item())
    for a, b in zip(keep, (*p, *c, opt.m.view(torch.uint8), opt.v.view(torch.uint8))):
        assert torch.equal(a, b)
    g[1][2999] = 0.1  # and the next one is taken
    opt.step(max_norm=1.0)
    assert not torch.equal(keep[0], p[0]) and all(torch.isfinite(t).all() for t in p)


def test_wide_ranges_in_8_bits(cuda_lib):
    """Gradients of 2^-30 … 1 in one block: no step explodes where a small second moment meets a scale of 1."""
    from objectsam_b200.optim import AdamW
    p = [torch.zeros(1024, device=DEV)]
    g = [2.0 ** -(torch.arange(1024, device=DEV) % 31).float()]
    opt = AdamW(p, g, lr=1e-3, weight_decay=0.0, bits=8)
    for _ in range(50):
        opt.step()
        g[0].mul_(-1)
    assert torch.isfinite(p[0]).all() and p[0].abs().max() <= 50 * 1e-3 * 1.1


def test_zero_gradients_and_resume(cuda_lib):
    from objectsam_b200.optim import AdamW
    for bits in (32, 8):
        p, g, _ = tensors([700, 50])
        ref = [t.clone() for t in p]
        a = AdamW(p, g, bits=bits)
        for _ in range(3):
            a.step()
        state = [None if t is None else t.clone() for t in (a.m, a.v, a.m_scale, a.v_scale)]
        mid = [t.clone() for t in p]
        a.step(max_norm=1.0)
        b_p = [t.clone() for t in mid]
        b = AdamW(b_p, g, bits=bits)
        b.load_state(*state, step=3)
        b.step(max_norm=1.0)
        for x, y in zip(p, b_p):
            assert torch.equal(x, y)
        for t in g:
            t.zero_()
        c = AdamW(ref, g, bits=bits, weight_decay=0.0)
        before = [t.clone() for t in ref]
        c.step(max_norm=1.0)
        assert all(torch.equal(x, y) for x, y in zip(ref, before)) and c.norm.item() == 0


def test_same_bits_every_time(cuda_lib):
    from objectsam_b200.optim import AdamW
    got = []
    for _ in range(2):
        p, g, c = tensors([100_003] * 30, packed=True)
        opt = AdamW(p, g, copies=c, bits=8)
        for _ in range(3):
            opt.step(max_norm=0.3)
        got.append([t.clone() for t in (*p, opt.norm, opt.m.view(torch.uint8))])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_states_outlive_steps_on_another_stream(cuda_lib):
    """An optimizer that is let go while its step still waits on another stream than the one it was made on: the allocator
    does not hand its states out before that step is through."""
    from objectsam_b200.optim import AdamW
    p, g, _ = tensors([3_000_001], copy=None)
    opt = AdamW(p, g)
    s, big = torch.cuda.Stream(), torch.randn(8192, 8192, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(200):  # a few hundred milliseconds
            big = big @ big * 1e-2
    opt.step(stream=s)
    held, n = {t.data_ptr() for t in (opt.m, opt.v)}, opt.m.numel()
    del opt
    again = [torch.empty(n, device=DEV) for _ in range(2)]
    busy = not s.query()
    assert not held & {t.data_ptr() for t in again} or not busy
    assert busy, "the step was through too early for this test"
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_capture(cuda_lib, bits):
    """A captured step replays with its capture's step count and rate, over gradients read anew."""
    from objectsam_b200.optim import AdamW
    p, g, c = tensors([5000, 77])
    p2, c2 = [t.clone() for t in p], [t.clone() for t in c]
    a, b = AdamW(p, g, copies=c, bits=bits), AdamW(p2, g, copies=c2, bits=bits)
    for o in (a, b):
        o.step(max_norm=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(max_norm=1.0)
    for by in (1.0, 3.0):
        for t in g:
            t.mul_(by)
        graph.replay()
        b.step(max_norm=1.0)
        b.steps -= 1
    torch.cuda.synchronize()
    for x, y in zip((*p, *c, a.m.view(torch.uint8), a.v.view(torch.uint8), a.norm), (*p2, *c2, b.m.view(torch.uint8), b.v.view(torch.uint8), b.norm)):
        assert torch.equal(x, y)
