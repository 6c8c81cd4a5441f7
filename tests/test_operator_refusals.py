"""Calls of the training step's operators that the kernels cannot answer: refused before anything is written."""
import pytest
import torch
from torch.autograd import forward_ad

from pccl_amd.ops import muon_step, orthogonalize, token_logprobs
from test_muon import gradient

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("hip")
    return torch.device(request.param)


def test_inference_tensors(device):
    """Outside of inference mode nothing of a call that would write one is carried out; inside, it is."""
    x, p, g, b = (gradient((6, 5), i, device) for i in range(4))
    with torch.inference_mode():
        out, q, c = torch.zeros_like(x), p.clone(), b.clone()
    kept = [v.clone() for v in (p, b, out, q, c)]
    with pytest.raises(RuntimeError, match="inference"):
        orthogonalize(x, out=out)
    for args in (([q], [g], [b]), ([p], [g], [c]), ([p, q], [g, g], [b, c])):
        with pytest.raises(RuntimeError, match="inference"):
            muon_step(*args, lr=0.1)
    assert all(torch.equal(v, k) for v, k in zip((p, b, out, q, c), kept))
    muon_step([p], [g], [b], lr=0.1)
    with torch.inference_mode():
        muon_step([q], [g], [c], lr=0.1)
        assert torch.equal(orthogonalize(x, out=out), orthogonalize(x))
        assert torch.equal(q, p) and torch.equal(c, b)


def test_ignore_index_is_a_token(device):
    """2^64 - 100 is not -100."""
    x, t = gradient((6, 5), 1, device), torch.full((6,), -100, device=device)
    for bad in ((1 << 64) - 100, 1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="ignore_index"):
            token_logprobs(x, t, ignore_index=bad)
    for fine in ((1 << 63) - 1, -(1 << 63)):
        assert bool(token_logprobs(x, t, ignore_index=fine).logprob.isnan().all())
        assert not token_logprobs(x, torch.full_like(t, fine), ignore_index=fine).logprob.any()


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.gpu
def test_forward_mode_is_refused(hip):
    """A dual tensor needs no gradient and has an address: its tangent must not vanish."""
    x, t = gradient((6, 5), 1, hip), torch.arange(5, device=hip).repeat(2)[:6]
    p, g, b = (gradient((6, 5), i, hip) for i in range(3))
    kept = [v.clone() for v in (p, g, b)]
    want = token_logprobs(x, t).logprob, orthogonalize(x)
    with forward_ad.dual_level():
        assert torch.equal(token_logprobs(x, t).logprob, want[0]) and torch.equal(orthogonalize(x), want[1])
        for no_grad in (False, True):
            with torch.set_grad_enabled(not no_grad):
                with pytest.raises(RuntimeError, match="tangent"):
                    token_logprobs(dual(x), t)
                with pytest.raises(RuntimeError, match="tangent"):
                    orthogonalize(dual(x))
                with pytest.raises(RuntimeError, match="tangent"):
                    orthogonalize(x, out=dual(torch.empty_like(x)))
                for k in range(3):
                    with pytest.raises(RuntimeError, match="tangent"):
                        muon_step(*([dual(v) if i == k else v] for i, v in enumerate((p, g, b))), lr=0.1)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: token_logprobs(v, t).logprob, (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v, i: token_logprobs(v, i).logprob)(x, t)
    with pytest.raises(RuntimeError):
        torch.func.vmap(orthogonalize)(gradient((2, 6, 5), 1, hip))
    assert all(torch.equal(v, k) for v, k in zip((p, g, b), kept))


def test_forward_mode_on_the_cpu():
    """There the tangent is the directional derivative."""
    x, t = gradient((6, 5), 1, "cpu", scale=1.0).double().float(), torch.arange(5).repeat(2)[:6]
    v = gradient((6, 5), 2, "cpu", scale=1.0)
    with forward_ad.dual_level():
        r = token_logprobs(forward_ad.make_dual(x, v), t)
        slope = forward_ad.unpack_dual(r.logprob).tangent
    y = x.double()
    want = v.double().gather(1, t[:, None])[:, 0] - (y.softmax(1) * v).sum(1)
    # 5 products of probabilities (each off by at most 8 roundings) and values below |v|, their sum, and a difference
    assert bool(((slope - want).abs() <= 64 * 2.0 ** -24 * v.abs().amax()).all())
