"""The C entries of the training step's operators refuse what no kernel may see, before they look for a device."""
import ctypes

import pytest

from pccl_amd._native import C

F32, BF16, F16, I32 = 10, 9, 8, 5
BUF = ctypes.create_string_buffer(1 << 14)  # refused calls never reach it
P = (ctypes.addressof(BUF) + 255) // 256 * 256


def forward(logits=P, stride=8, rows=2, vocab=8, dtype=F32, targets=P, top_k=2, logprob=P, entropy=P, stats=P, top=P,
            index=P):
    return C.pcclxTokenLogprobs(logits, stride, rows, vocab, dtype, targets, -100, top_k, logprob, entropy, stats, top,
                                index, None)


def backward(logits=P, rows=2, vocab=8, dtype=F32, targets=P, top_k=2, stats=P, index=P, g_top=P, out=P):
    return C.pcclxTokenLogprobsGrad(logits, 8, rows, vocab, dtype, targets, -100, top_k, stats, index, None, None, g_top,
                                    out, None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(targets=None), dict(logprob=None), dict(entropy=None),
                                 dict(stats=None), dict(top=None), dict(index=None), dict(rows=-1), dict(rows=1 << 31),
                                 dict(vocab=0), dict(vocab=1 << 31), dict(top_k=-1), dict(top_k=9),
                                 dict(vocab=100, top_k=65), dict(dtype=I32), dict(dtype=99), dict(dtype=-1),
                                 dict(dtype=256 + F32)])
def test_token_logprobs(bad):
    assert forward(**bad) == -2


@pytest.mark.parametrize("bad", [dict(logits=None), dict(targets=None), dict(stats=None), dict(out=None),
                                 dict(index=None), dict(rows=-1), dict(vocab=0), dict(top_k=9), dict(dtype=I32),
                                 dict(dtype=256 + F16)])
def test_token_logprobs_grad(bad):
    assert backward(**bad) == -2


def muon(shapes=(1, 4, 300), g=P, w=P + 4864, mom=None, alpha=True, gtype=F32, wtype=F32, coefficients=(1.5, -0.5, 0.0),
         steps=5, work=None, size=None, n=1):
    ptr = lambda v: (ctypes.c_void_p * 1)(v)  # noqa: E731
    s = None if shapes is None else (ctypes.c_int64 * 3)(*shapes)
    return C.pcclxMuon(n, s, g and ptr(g), gtype, w and ptr(w), wtype, mom and ptr(mom),
                       (ctypes.c_float * 1)(0.1) if alpha else None, 1.0, 0.9, 0, steps,
                       coefficients and (ctypes.c_float * 3)(*coefficients), 1e-7, work,
                       C.pcclxMuonWorkspace(1, s) if size is None else size, None)


@pytest.mark.parametrize("bad", [
    dict(), dict(work=P + 8), dict(work=P, size=1), dict(work=P, size=-1),  # no workspace, a crooked or a short one
    dict(work=P, coefficients=None), dict(work=P, g=None), dict(work=P, w=None), dict(work=P, mom=P + 9728, alpha=False),
    dict(work=P, gtype=I32), dict(work=P, wtype=256 + F32), dict(work=P, steps=0), dict(work=P, n=-1),
    dict(work=P, shapes=None, size=1 << 20), dict(work=P, shapes=(-1, 4, 300), size=1 << 20),
    # sizes whose product leaves 64 bits, one of them with a product of 0 there
    dict(work=P, shapes=(1 << 30, 1 << 30, 1 << 30), size=1 << 20),
    dict(work=P, shapes=(1 << 30, 1 << 30, 16), size=1 << 20), dict(work=P, shapes=(16, 1 << 30, 1 << 30), size=1 << 20)])
def test_muon(bad):
    assert muon(**bad) == -2


def test_muon_workspace():
    need = lambda *s: C.pcclxMuonWorkspace(len(s) // 3, (ctypes.c_int64 * len(s))(*s))  # noqa: E731
    assert need(1 << 30, 1 << 30, 1 << 30) == need(16, 1 << 30, 1 << 30) == C.pcclxMuonWorkspace(1, None) == -1
    assert need(1, 1 << 30, 0) == 0
