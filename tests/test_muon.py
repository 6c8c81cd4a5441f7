"""orthogonalize and muon_step against the formulas in 64 bits, on the CPU path and the HIP kernels.

Tolerances come from the arithmetic, run as a model: `deviation` repeats the steps in float64 and moves every operand
and every sum by random amounts of the full size that its number format allows (below), so it carries the amplification
of early errors (up to 3.4 a step for small singular values) that a formula would have to bound far too widely. The
results may be off by three times what the model is, and by the rounding of their type.

* a pair of fp16 numbers: 2^-21 relative (half a step of either part, and the lo lo product that is left out), and
  2^-25 of a scaled unit (fp16's smallest step);
* one fp16 number, the operands of A and P X where the result is bf16: 2^-11;
* a sum of K products in fp32: sqrt(K) 2^-24 of the sum of absolute products.
"""
import math

import pytest
import torch

from pccl_amd._native import C
from pccl_amd.ops import muon_step, orthogonalize

U = 2.0 ** -24
ABC = (3.4445, -4.7750, 2.0315)
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("hip")
    return torch.device(request.param)


def exact(x, steps=5, abc=ABC, eps=1e-7):
    a, b, c = abc
    x = x.detach().double()
    y = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    flip = y.shape[-2] > y.shape[-1]
    y = y.mT.contiguous() if flip else y
    for _ in range(steps):
        g = y @ y.mT.contiguous()
        y = a * y + (b * g + c * (g @ g)) @ y
    return y.mT.contiguous() if flip else y


def deviation(x, single, steps=5, abc=ABC, eps=1e-7):
    """The model above against `exact`; `single`: one fp16 number per operand of A and P X."""
    a, b, c = abc
    gen = torch.Generator(device=x.device).manual_seed(99)
    x = x.detach().double()
    y = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    y = y.mT.contiguous() if y.shape[-2] > y.shape[-1] else y

    def noise(t):
        return 2 * torch.rand(t.shape, generator=gen, device=t.device, dtype=torch.float64) - 1

    def pair(t, scale, one=False):
        return t * (1 + noise(t) * 2.0 ** (-11 if one else -21)) + noise(t) * 2.0 ** -25 / scale

    def product(s, t):
        r = s @ t
        return r + noise(r) * math.sqrt(s.shape[-1]) * U * (s.abs() @ t.abs())

    want = y
    for _ in range(steps):
        g = product(pair(y, 8192, single), pair(y, 8192, single).mT.contiguous())
        p = b * pair(g, 1024) + c * product(pair(g, 1024), pair(g, 1024))
        y = a * pair(y, 8192) + product(pair(p, 4096, single), pair(y, 8192, single))
        g = want @ want.mT.contiguous()
        want = a * want + (b * g + c * (g @ g)) @ want
    return (y - want).abs().amax((-2, -1), keepdim=True)


def gradient(shape, seed, device, dtype=torch.float32, scale=1e-3):
    """dY^T X of a linear layer, with falling spectra."""
    gen = torch.Generator().manual_seed(seed)
    *batch, m, n = shape
    k = 2 * min(m, n) + 1
    dy = torch.randn(*batch, k, m, generator=gen) * torch.exp(-2.0 * torch.arange(m) / m)
    x = torch.randn(*batch, k, n, generator=gen) * torch.exp(-2.0 * torch.arange(n) / n)
    return ((dy.mT @ x) * scale / k).to(dtype).to(device)


def check(x, got, **kw):
    want = exact(x, **kw)
    dev = deviation(x, x.dtype == torch.bfloat16, **kw)
    half = torch.finfo(x.dtype).eps / 2
    off = (got.double() - want).abs() - want.abs() * half * 1.01
    assert got.dtype == x.dtype and got.shape == x.shape
    assert bool((off <= 3 * dev + torch.finfo(x.dtype).smallest_normal).all()), \
        f"off by up to {float(off.max())}, allowed {float(3 * dev.max())}"


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 5), (64, 64), (65, 63), (100, 300), (517, 130), (2, 3, 40, 96), (5, 256, 192),
          (1, 3001), (700, 64),
          (3, 256, 60), (2, 30, 250), (2, 120, 128), (64, 257)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(device, dtype, shape):
    x = gradient(shape, 1, device, dtype)
    kept = x.clone()
    check(x, orthogonalize(x))
    assert torch.equal(x, kept)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(90, 200, 300), (90, 300, 200), (2, 1030, 2050), (1, 2050, 1030), (3, 640, 640)])
def test_orthogonalize_large(hip, dtype, shape):
    """Sizes that take the larger tiles, with edges inside a tile."""
    gen = torch.Generator(device=hip).manual_seed(4)
    x = (torch.randn(*shape, generator=gen, device=hip) * 1e-3).to(dtype)
    check(x, orthogonalize(x))


def test_singular_values_end_near_one(device):
    x = gradient((96, 200), 2, device)
    s = torch.linalg.svdvals(orthogonalize(x).double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,abc", [(1, ABC), (2, (1.5, -0.5, 0.0)), (8, ABC), (6, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(device, dtype, steps, abc):
    x = gradient((48, 70), 3, device, dtype)
    check(x, orthogonalize(x, steps=steps, coefficients=abc), steps=steps, abc=abc)


def test_sizes_of_the_values(device):
    """The norm's square leaves fp32's range on both sides; eps takes over below it."""
    x = gradient((40, 30), 4, device, scale=1.0)
    want = orthogonalize(x)
    for scale in (2.0 ** 110, 2.0 ** -100):
        check(x * scale, orthogonalize(x * scale, eps=1e-37), eps=1e-37)
        assert torch.equal(orthogonalize(x * scale, eps=1e-37), want)
    check(x * 1e-9, orthogonalize(x * 1e-9, eps=1.0), eps=1.0)
    zero = torch.zeros(3, 40, 30, device=device)
    assert not orthogonalize(zero).any()
    zero[1] = x  # a zero matrix next to another one
    got = orthogonalize(zero)
    assert not got[0].any() and not got[2].any() and torch.equal(got[1], want)
    rank_one = torch.outer(torch.arange(1.0, 41.0), torch.arange(1.0, 31.0)).to(device)
    check(rank_one, orthogonalize(rank_one))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_not_a_number(device, dtype, value):
    x = gradient((3, 70, 90), 5, device, dtype)
    want = orthogonalize(x)
    x[1, 69, 3] = value
    got = orthogonalize(x)
    assert bool(got[1].isnan().all())
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def test_layouts_and_out(device):
    x = gradient((4, 70, 50), 6, device)
    want = orthogonalize(x)
    assert torch.equal(orthogonalize(x.mT.contiguous().mT), want)
    assert torch.equal(orthogonalize(torch.stack([x, x], dim=3)[..., 0]), want)
    assert torch.equal(orthogonalize(x[::2]), want[::2])
    flat = torch.empty(x.numel() + 1, device=device)
    odd = flat[1:].view(x.shape).copy_(x)  # at an odd address
    assert torch.equal(orthogonalize(odd), want)
    out = torch.empty_like(x)
    assert orthogonalize(x, out=out) is out and torch.equal(out, want)
    y = x.clone()
    assert torch.equal(orthogonalize(y, out=y), want) and torch.equal(y, want)
    flat = torch.full((x.numel() + 2,), 7.0, device=device)  # nothing next to the result is touched
    orthogonalize(x, out=flat[1:-1].view(x.shape))
    assert flat[0] == 7.0 and flat[-1] == 7.0 and torch.equal(flat[1:-1].view(x.shape), want)
    for shape in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        assert orthogonalize(torch.empty(shape, device=device)).shape == shape


def test_orthogonalize_refusals(device):
    x = gradient((6, 5), 7, device)
    with pytest.raises(ValueError, match="matrix"):
        orthogonalize(x[0])
    with pytest.raises(TypeError, match="fp32"):
        orthogonalize(x.double())
    with pytest.raises(RuntimeError, match="differentiable"):
        orthogonalize(x.clone().requires_grad_())
    for bad in (torch.empty(5, 6, device=device), x.half(), torch.empty(5, 6, device=device).T):
        with pytest.raises(ValueError, match="out"):
            orthogonalize(x, out=bad)
    with pytest.raises(RuntimeError, match="no_grad"):
        orthogonalize(x, out=torch.empty_like(x, requires_grad=True))
    for eps in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            orthogonalize(x, eps=eps)
    for steps in (0, 101):
        with pytest.raises(ValueError, match="steps"):
            orthogonalize(x, steps=steps)
    for abc in ((1.0, 2.0), (3.4445, -4.775, 20.0), (9.0, 0.0, 0.0), (math.nan, 0.0, 0.0), (1.0, -13.0, 13.0)):
        with pytest.raises(ValueError, match="coefficients"):
            orthogonalize(x, coefficients=abc)


@pytest.mark.gpu
def test_result_may_not_overlap_its_input(hip):
    x = gradient((7, 5, 5), 7, hip)
    with pytest.raises(ValueError, match="shares memory"):
        orthogonalize(x[:5], out=x[1:6])


def test_workspace_is_bounded():
    """Large stacks run in groups: the plan's workspace stays below its budget, or is that of one matrix."""
    import ctypes
    need = lambda *s: C.pcclxMuonWorkspace(len(s) // 3, (ctypes.c_int64 * len(s))(*s))  # noqa: E731
    one = need(1, 64, 512)
    assert one == 2 * (4 * 64 * 512 + 4 * 64 * 64) + 4096
    assert need(3, 512, 64) == 3 * one and need(2, 64, 512, 1, 512, 64) == 3 * one
    assert need(1, 1, 500) == one and need(1, 65, 130) == 2 * (4 * 128 * 192 + 4 * 128 * 128) + 4096
    assert 4 * 2 ** 30 - one < need(10 ** 6, 64, 512) <= 4 * 2 ** 30
    assert need(1, 30000, 60000) > 4 * 2 ** 30
    for small in ((64, 64), (1, 1), (64, 256), (256, 3), (128, 128)):  # one workgroup each, in LDS
        assert need(10 ** 6, *small) == 0
    assert need() == 0 and need(0, 5, 5) == 0
    assert need(1, -1, 5) == -1 and need(1, 2 ** 31, 5) == -1


@pytest.mark.gpu
def test_more_matrices_than_a_group(hip):
    """13100 matrices exceed the workspace's budget, 101 shapes exceed the entries of a launch."""
    x = gradient((50, 100, 130), 8, hip)
    got = orthogonalize(x.repeat(262, 1, 1)).view(262, 50, 100, 130)
    for i in (0, 100, 258, 261):  # the second group starts at 12945
        check(x, got[i])
    x = x[:, :16, :12].contiguous()
    assert torch.equal(orthogonalize(x.repeat(1240, 1, 1)), orthogonalize(x).repeat(1240, 1, 1))
    params = [torch.zeros(5 + i % 7, 3 + i, device=hip) for i in range(101)]
    grads = [gradient(p.shape, i, hip) for i, p in enumerate(params)]
    moms = [torch.zeros_like(p) for p in params]
    muon_step(params, grads, moms, lr=-1.0, weight_decay=0.0, momentum=0.0, adjust_lr="none")
    for p, g in zip(params, grads):
        assert torch.equal(p, orthogonalize(g))


@pytest.mark.gpu
def test_more_matrices_than_a_launch_has(hip):
    """2^22 + 3 matrices of one workgroup each."""
    x = gradient((7, 2, 3), 5, hip)
    n = (1 << 22) + 3
    got = orthogonalize(x.repeat(n // 7 + 1, 1, 1)[:n])
    want = orthogonalize(x)
    assert bool((got[:n // 7 * 7].view(-1, 7, 2, 3) == want).all()) and torch.equal(got[n // 7 * 7:], want[:n % 7])


def model_step(p, g, b, lr, wd, mu, nesterov, factor, steps=5):
    """float64 step, and how far parameter and momentum may be off."""
    p, g, b = p.double(), g.double(), b.double()
    nb = mu * b + (1 - mu) * g
    u = (1 - mu) * g + mu * nb if nesterov else nb
    return p * (1 - lr * wd) - lr * factor * exact(u, steps), nb, u


@pytest.mark.parametrize("wtype,gtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.float16, torch.float16), (torch.float32, torch.bfloat16),
                                         (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", ["original", "match_rms_adamw", "none"])
def test_muon_step(device, wtype, gtype, nesterov, adjust):
    shapes = [(64, 64), (192, 64), (64, 256), (1, 9), (33, 17), (130, 70)]
    gen = torch.Generator().manual_seed(11)
    params = [(torch.randn(s, generator=gen) * 0.02).to(wtype).to(device) for s in shapes]
    moms = [gradient(s, 40 + i, device) for i, s in enumerate(shapes)]
    lr, wd, mu = 0.02, 0.1, 0.95
    for turn in range(2):
        grads = [gradient(s, 50 + 10 * turn + i, device, gtype) for i, s in enumerate(shapes)]
        before = [(p.clone(), b.clone()) for p, b in zip(params, moms)]
        muon_step(params, grads, moms, lr=lr, weight_decay=wd, momentum=mu, nesterov=nesterov, adjust_lr=adjust)
        for p, b, g, (p0, b0) in zip(params, moms, grads, before):
            rows, cols = p.shape
            f = {"original": math.sqrt(max(1, rows / cols)), "match_rms_adamw": 0.2 * math.sqrt(max(rows, cols)),
                 "none": 1.0}[adjust]
            want, nb, u = model_step(p0, g, b0, lr, wd, mu, nesterov, f)
            # three roundings of numbers below |B| + |G|
            assert bool(((b.double() - nb).abs() <= 3 * U * (b0.double().abs() + g.double().abs())).all())
            # u itself carries those roundings into the steps (2^-21 of an entry covers them where |B| + |G| is below
            # four times |u|'s largest entry, hence the factor 4 on the model)
            dev = deviation(u, wtype == torch.bfloat16) * 4 * lr * f
            tol = 3 * dev + want.abs() * torch.finfo(wtype).eps / 2 * 1.01 + 4 * U * (p0.double().abs() + lr * f)
            assert bool(((p.double() - want).abs() <= tol).all())


def test_step_of_zero_gradient(device):
    """No gradient and no momentum: the weights only decay."""
    p = torch.randn(20, 30, device=device)
    want = p * (1 - 0.5 * 0.1)
    b = torch.zeros_like(p)
    muon_step([p], [torch.zeros_like(p)], [b], lr=0.5, weight_decay=0.1)
    assert torch.allclose(p, want, rtol=2 ** -22, atol=0) and not b.any()


def test_muon_step_refusals(device):
    p, g, b = (gradient((6, 5), i, device) for i in range(3))
    kw = dict(lr=0.1)
    muon_step([], [], [], **kw)
    with pytest.raises(ValueError, match="1 parameters"):
        muon_step([p], [], [b], **kw)
    with pytest.raises(ValueError, match="one shape"):
        muon_step([p], [g.T], [b], **kw)
    with pytest.raises(ValueError, match="one shape"):
        muon_step([p[0]], [g[0]], [b[0]], **kw)
    with pytest.raises(TypeError, match="momentum"):
        muon_step([p], [g], [b.bfloat16()], **kw)
    with pytest.raises(TypeError, match="one type"):
        muon_step([p, p.bfloat16()], [g, g], [b, b.clone()], **kw)
    with pytest.raises(TypeError, match="fp32"):
        muon_step([p.double()], [g], [b], **kw)
    with pytest.raises(ValueError, match="contiguous"):
        muon_step([torch.empty(5, 6, device=device).T], [g], [b], **kw)
    with pytest.raises(ValueError, match="shares memory"):
        muon_step([p, p], [g, g], [b, b.clone()], **kw)
    with pytest.raises(ValueError, match="shares memory"):
        muon_step([p, p.clone()], [g, g], [b, b], **kw)
    with pytest.raises(ValueError, match="shares memory"):
        muon_step([p, p.clone()], [g, p], [b, b.clone()], **kw)
    with pytest.raises(ValueError, match="shares memory"):
        muon_step([p], [b], [b], **kw)
    big = torch.zeros(40, device=device)
    with pytest.raises(ValueError, match="shares memory"):
        muon_step([big[:30].view(6, 5), big[10:].view(6, 5)], [g, g], [b, b.clone()], **kw)
    with pytest.raises(ValueError, match="adjust_lr"):
        muon_step([p], [g], [b], adjust_lr="other", **kw)
    for bad in (dict(momentum=1.5), dict(momentum=math.nan), dict(weight_decay=math.inf), dict(eps=0.0)):
        with pytest.raises(ValueError):
            muon_step([p], [g], [b], **kw, **bad)
    with pytest.raises(ValueError, match="finite"):
        muon_step([p], [g], [b], lr=math.nan)
    with pytest.raises(ValueError, match="one device"):
        muon_step([p], [g.to("meta")], [b], **kw)


def test_shared_gradient_and_strided_gradient(device):
    """One gradient tensor for two parameters (a tied layer), and a transposed one."""
    p = [gradient((6, 5), i, device) for i in range(2)]
    g = gradient((6, 5), 7, device)
    b = [torch.zeros_like(g) for _ in p]
    q, c = [x.clone() for x in p], [x.clone() for x in b]
    muon_step(p, [g, g], b, lr=0.1)
    muon_step(q, [g.T.contiguous().T, g.clone()], c, lr=0.1)
    assert all(torch.equal(x, y) for x, y in zip(p + b, q + c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_bits_again(hip, dtype):
    """Equal calls give equal bits, whatever tiles and paths the shapes take; alone, a matrix may take other tiles."""
    shapes = [(128, 64), (64, 64), (300, 500), (17, 900), (100, 128), (1000, 1500), (1100, 4000), (500, 500)]
    grads = [gradient(s, i, hip, dtype) for i, s in enumerate(shapes)]

    def run(pick):
        p = [torch.zeros(shapes[i], device=hip, dtype=dtype) for i in pick]
        b = [torch.zeros(shapes[i], device=hip) for i in pick]
        muon_step(p, [grads[i] for i in pick], b, lr=-1.0, momentum=0.0, weight_decay=0.0, adjust_lr="none")
        return p + b

    whole = run(range(8))
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(whole, run(range(8))))
    for i in range(8):
        p, b = run([i])
        assert torch.equal(b, whole[8 + i])
        check(grads[i], p)
        check(grads[i], whole[i])


@pytest.mark.gpu
def test_side_stream_and_graph(hip):
    """On another stream, and captured once and replayed with new gradients between eager calls and synchronisations."""
    shapes = [(96, 64), (64, 200)]
    p = [torch.zeros(s, device=hip) for s in shapes]
    b = [torch.zeros(s, device=hip) for s in shapes]
    q, c = [x.clone() for x in p], [x.clone() for x in b]
    g = [gradient(s, 3, hip) for s in shapes]
    step = lambda w, m: muon_step(w, g, m, lr=0.1)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(p, b)
    torch.cuda.current_stream().wait_stream(side)
    step(q, c)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(p + b, q + c))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(p, b)
    for turn in range(4):
        for x, s in zip(g, shapes):
            x.copy_(gradient(s, 60 + turn, hip))
        graph.replay()
        torch.cuda.synchronize()
        step(q, c)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(p + b, q + c))


@pytest.mark.gpu
def test_two_calls_at_once(hip):
    """Two streams, each with a workspace of its own."""
    x = [gradient((256, 300), i, hip) for i in range(2)]
    want = [orthogonalize(y) for y in x]
    streams = [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(orthogonalize(x[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for w, ys in zip(want, got) for y in ys)
