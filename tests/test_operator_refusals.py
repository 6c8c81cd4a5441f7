"""Calls of the training step's operators that the kernels cannot answer: refused before anything is written."""
import pytest
import torch

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
