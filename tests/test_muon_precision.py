"""Every result has the error of products of 22-bit operands, also a bf16 one, whatever else the call holds.

The model of tests/test_muon.py with pairs everywhere (`deviation(x, False)`): three times its deviation, and the rounding
of the result's type.
"""
import pytest
import torch

from pccl_amd.ops import muon_step, orthogonalize
from test_muon import deviation, exact, gradient

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("hip")
    return torch.device(request.param)


def check_pairs(x, got):
    want = exact(x)
    allowed = 3 * deviation(x, False) + want.abs() * (torch.finfo(got.dtype).eps / 2 * 1.01)
    off = (got.double() - want).abs() - allowed
    assert bool((off <= torch.finfo(got.dtype).smallest_normal).all()), f"off by {float(off.max())} more than allowed"


@pytest.mark.parametrize("shape", [(65, 300), (3, 256, 192), (300, 500), (400, 320)])
def test_bf16_of_few_rows(device, shape):
    x = gradient(shape, 21, device, BF16)
    check_pairs(x, orthogonalize(x))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(320, 1000), (12, 768, 768), (1030, 2050), (2050, 1030), (1, 4096, 1100)])
def test_bf16_of_many_rows(hip, shape):
    """Enough rows for every tile that bf16 matrices take."""
    x = gradient(shape, 22, hip, BF16)
    check_pairs(x, orthogonalize(x))


@pytest.mark.gpu
def test_bf16_beside_a_larger_matrix(hip):
    """A small matrix is as exact next to a large one as it is alone, in either order."""
    shapes = [(17, 900), (100, 300), (1000, 1500), (250, 260), (64, 512), (700, 520)]
    for order in (shapes, shapes[::-1]):
        grads = [gradient(s, 30 + s[0], hip, BF16) for s in order]
        params = [torch.zeros_like(g) for g in grads]
        muon_step(params, grads, [torch.zeros(s, device=hip) for s in order], lr=-1.0, weight_decay=0.0, momentum=0.0,
                  adjust_lr="none")
        for p, g in zip(params, grads):
            check_pairs(g, p)


@pytest.mark.gpu
@pytest.mark.parametrize("wtype,gtype", [(F16, F16), (F32, BF16), (BF16, F32), (F16, F32), (F32, F16)])
def test_types_at_staged_sizes(hip, wtype, gtype):
    """Parameters and gradients of every type, at sizes of several tiles and more entries than a launch takes."""
    shapes = [(1100, 700), (520, 2050), (300, 400), (64, 900), (1030, 1030), (130, 70)] + [(70 + i, 140) for i in range(50)]
    grads = [gradient(s, 40 + i, hip, gtype) for i, s in enumerate(shapes)]
    params = [torch.zeros(s, device=hip, dtype=wtype) for s in shapes]
    moms = [torch.zeros(s, device=hip) for s in shapes]
    muon_step(params, grads, moms, lr=-1.0, weight_decay=0.0, momentum=0.0, adjust_lr="none")
    for p, g, b in zip(params, grads, moms):
        assert torch.equal(b, g.float())
        check_pairs(g, p)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(16, 16), (16, 230), (230, 16), (20, 100), (17, 40), (31, 256), (64, 64), (64, 256),
                                   (128, 128), (70, 300), (16, 1000)])
def test_fp32_of_small_matrices(hip, shape):
    """Few rows leave little for roundings to average out over: root mean square errors of 32 matrices, at most half again
    those of the same steps in fp32 products."""
    x = torch.stack([gradient(shape, 200 + i, hip) for i in range(32)])
    want = exact(x)
    y = (x / x.double().square().sum((-2, -1), keepdim=True).sqrt()).float()
    y = y.mT.contiguous() if shape[0] > shape[1] else y
    for _ in range(5):
        g = y @ y.mT.contiguous()
        y = 3.4445 * y + (-4.7750 * g + 2.0315 * (g @ g)) @ y
    y = y.mT if shape[0] > shape[1] else y
    error = lambda t: float((t.double() - want).square().mean().sqrt())  # noqa: E731
    assert error(orthogonalize(x)) <= 1.5 * error(y), (error(orthogonalize(x)), error(y))


@pytest.mark.gpu
def test_offsets_past_32_bits(hip):
    """More than 2^31 elements in a stack, in one wide and in one tall matrix."""
    y = gradient((4, 1000, 2000), 50, hip, BF16)
    want = orthogonalize(y).float()
    got = orthogonalize(y.repeat(280, 1, 1)).view(280, 4, 1000, 2000)
    # the same products in other tiles: off by their error at most, and then by one step of bf16
    dev = 6 * deviation(y, False).max() + want.abs() * torch.finfo(BF16).eps
    for part in got:
        assert bool(((part.float() - want).abs() <= dev).all())
    del got
    gen = torch.Generator(device=hip).manual_seed(6)
    x = torch.randn(8192, 264000, generator=gen, device=hip, dtype=BF16)
    assert x.numel() > 1 << 31
    abc = (3.4445, -4.7750, 2.0315)
    wide = orthogonalize(x, steps=1, coefficients=abc)
    last = slice(-3000, None)  # far behind 2^31 in the last rows; every row of A depends on the whole of its row of X
    z = x.float() / x.double().square().sum().sqrt().float()
    g = torch.zeros(8192, 8192, device=hip, dtype=torch.float64)
    for k in range(0, 264000, 24000):
        part = z[:, k:k + 24000].double()
        g += part @ part.mT.contiguous()
    p = abc[1] * g + abc[2] * (g @ g)
    for cols in (slice(0, 3000), last):
        want = abc[0] * z[:, cols].double() + p @ z[:, cols].double()
        # an entry is z's 3.4 times and sums of 22-bit products in fp32, far below a tenth of bf16's half step here
        off = (wide[:, cols].double() - want).abs() - want.abs() * (torch.finfo(BF16).eps / 2 * 1.1)
        assert bool((off <= want.abs().max() * 2.0 ** -16).all()), float(off.max())
    tall = orthogonalize(x.mT.contiguous(), steps=1, coefficients=abc)
    assert torch.equal(tall.mT, wide)
