"""token_logprobs (log probabilities of given tokens, entropy, top alternatives, gradients) against the formulas in
64 bits, on the CPU path and the HIP kernels, at the sizes, masks and strides where it can go wrong.

Tolerances. u = 2^-24 is half a step of fp32. Each of the two sums of a row is built from at most V terms by a thread
(the CPU path: by torch), rescaled a few times and joined by a tree, each term exp(d) with d rounded twice and a
hardware exponential of at most 2 u: relative error below E = (2 V / 64 + 64) u times (1 + |d| averaged over p, which is
below 1 + ln V), for sums whose order puts at most V / 64 terms behind each other.
"""
import math

import pytest
import torch

from pccl_amd.ops import token_logprobs

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("hip")
    return torch.device(request.param)


def reference(logits, targets, top_k, ignore_index=-100):
    """The definition in float64, with the documented values of empty rows and foreign targets."""
    x = logits.detach().cpu().double()
    targets = targets.cpu()
    empty = (x == -math.inf).all(dim=-1)
    top = x.amax(dim=-1, keepdim=True)
    x = x - torch.where(top.isinf(), 0.0, top)  # first: next to the lowest fp32 value even float64 has no room for lse
    lse = torch.logsumexp(x, dim=-1, keepdim=True)
    logp = torch.where(empty[..., None], -math.inf, x - lse)
    p = torch.where(empty[..., None], 0.0, logp.exp())
    entropy = torch.where(empty, 0.0, torch.special.entr(p).sum(dim=-1))
    known = (targets >= 0) & (targets < x.shape[-1])
    lp = logp.gather(-1, torch.where(known, targets, 0)[..., None])[..., 0]
    lp = torch.where(targets == ignore_index, 0.0, torch.where(known, lp, math.nan))
    index = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top_k]
    return lp, entropy, logp.gather(-1, index), index, logp, p


def sum_error(vocab):
    return (2 * vocab / 64 + 64) * U * (1 + math.log(max(vocab, 2)))


def close(got, want, tol):
    got, want = got.detach().cpu().double(), want.double()
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite())
    assert torch.equal(got[~fine].nan_to_num(7.0), want[~fine].nan_to_num(7.0))
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)[fine]
    off = (got[fine] - want[fine]).abs()
    assert bool((off <= tol).all()), f"off by {float((off - tol).max())} more than allowed"


def check(logits, targets, top_k, ignore_index=-100):
    r = token_logprobs(logits, targets, top_k=top_k, ignore_index=ignore_index)
    lp, entropy, top_lp, index, logp, p = reference(logits, targets, top_k, ignore_index)
    err = sum_error(logits.shape[-1])
    assert r.logprob.dtype == r.entropy.dtype == torch.float32 and r.logprob.shape == targets.shape
    close(r.logprob, lp, err + 2 * U * lp.abs().nan_to_num(0, posinf=0, neginf=0))
    close(r.entropy, entropy, err * (2 + math.log(logits.shape[-1])))
    if top_k:
        assert torch.equal(r.top_index.cpu(), index)
        close(r.top_logprob, top_lp, err + 2 * U * top_lp.abs().nan_to_num(0, posinf=0, neginf=0))
    else:
        assert r.top_logprob is None and r.top_index is None
    return r


def gradient_reference(logits, targets, top_k, grads, ignore_index=-100):
    """dx and the absolute sum of its terms' sizes, in float64."""
    lp, entropy, _, index, logp, p = reference(logits, targets, top_k, ignore_index)
    g_lp, g_h, g_top = (None if g is None else g.detach().cpu().double() for g in grads)
    d, size = torch.zeros_like(p), torch.zeros_like(p)
    safe = logp.clamp(min=-1e4)

    def add(g, at):
        for acc, val in ((d, g), (size, g.abs())):
            acc.scatter_add_(-1, at[..., None], val[..., None])
        d.sub_(g[..., None] * p)
        size.add_(g.abs()[..., None] * p * (1 + safe.abs()))

    if g_lp is not None:
        used = targets.cpu() != ignore_index
        add(torch.where(used, g_lp, 0.0), torch.where(used, targets.cpu(), 0))
    if g_top is not None:
        for k in range(top_k):
            add(g_top[..., k], index[..., k])
    if g_h is not None:
        term = g_h[..., None] * p * (safe + entropy[..., None])
        d.sub_(term)
        size.add_(g_h.abs()[..., None] * p * (1 + safe.abs()) * (1 + safe.abs() + entropy[..., None]))
    empty = (logits.detach().cpu() == -math.inf).all(dim=-1, keepdim=True)
    return torch.where(empty, 0.0, d), size


def check_gradient(logits, targets, top_k, which, ignore_index=-100, seed=3):
    gen = torch.Generator().manual_seed(seed)
    x = logits.detach().requires_grad_()
    r = token_logprobs(x, targets, top_k=top_k, ignore_index=ignore_index)
    outs, grads = [], [None, None, None]
    for i, name in enumerate(("logprob", "entropy", "top_logprob")):
        if name in which:
            out = getattr(r, name)
            g = torch.randn(out.shape, generator=gen).to(out.device)
            outs.append(out)
            grads[i] = g
    got, = torch.autograd.grad(outs, x, [g for g in grads if g is not None])
    assert got.dtype == x.dtype and got.shape == x.shape
    want, size = gradient_reference(logits, targets, top_k, grads, ignore_index)
    eps = torch.finfo(x.dtype).eps
    tiny = torch.finfo(x.dtype).smallest_normal * eps  # a step of the subnormal numbers
    close(got, want, want.abs() * eps / 2 * 1.01 + size * sum_error(logits.shape[-1]) * 2 + tiny)


def make(shape, dtype, device, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*shape, generator=g) * scale).to(dtype)
    t = torch.randint(0, shape[-1], shape[:-1], generator=g)
    return x.to(device), t.to(device)


SIZES = [((1, 1), 1), ((3, 2), 2), ((5, 7), 7), ((2, 64), 64), ((9, 257), 5), ((300, 512), 3), ((2, 3, 1000), 20),
         ((4, 8192), 64), ((1, 50304), 5), ((3, 50257), 20), ((261, 3001), 0), ((260, 4099), 17)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,top_k", SIZES)
def test_forward(device, dtype, shape, top_k):
    check(*make(shape, dtype, device), top_k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,top_k,which", [
    ((1, 1), 1, ("logprob", "entropy", "top_logprob")), ((5, 7), 7, ("logprob", "entropy", "top_logprob")),
    ((9, 257), 0, ("logprob",)), ((9, 257), 0, ("entropy",)), ((9, 257), 5, ("top_logprob",)),
    ((2, 3, 1000), 64, ("logprob", "top_logprob")), ((300, 513), 2, ("logprob", "entropy")),
    ((2, 50257), 20, ("logprob", "entropy", "top_logprob")), ((1030, 515), 1, ("logprob", "entropy", "top_logprob"))])
def test_gradient(device, dtype, shape, top_k, which):
    check_gradient(*make(shape, dtype, device), top_k, which)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_is_the_slope(device, dtype):
    """Central differences of a weighted sum of all results, on logits that the type holds exactly."""
    g = torch.Generator().manual_seed(9)
    x = (torch.randint(-16, 17, (4, 6), generator=g) / 8).to(device)
    x[2, 3] = -math.inf
    t = torch.tensor([0, 5, 1, -100], device=device)
    w = [torch.randn(4, generator=g).to(device) for _ in range(2)] + [torch.randn(4, 2, generator=g).to(device)]

    def value(y):
        r = token_logprobs(y, t, top_k=2)
        return sum((a.double() * b.double()).sum() for a, b in zip((r.logprob, r.entropy, r.top_logprob), w))

    # alternatives must not change places within the step
    x += torch.arange(6, device=device) / 64
    leaf = x.to(dtype).requires_grad_()
    assert torch.equal(leaf.detach().float(), x)
    got, = torch.autograd.grad(value(leaf), leaf)
    h = 2.0 ** -8
    for i in range(4):
        for j in range(6):
            d = torch.zeros_like(x)
            d[i, j] = h
            slope = float((value(x + d) - value(x - d)).detach() / (2 * h))
            # third derivatives of log p and H are below 2 + ln 6 with weights below 4: h^2 / 6 * 4 * 5 * 4; the values
            # carry 20 fp32 roundings of numbers below 8
            tol = h * h / 6 * 80 + 20 * 8 * U / h + abs(slope) * torch.finfo(dtype).eps
            assert abs(float(got[i, j]) - slope) <= tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [6, 700, 9001])
def test_masked_tokens(device, dtype, vocab):
    x, t = make((40, vocab), dtype, device, seed=5)
    g = torch.Generator().manual_seed(6)
    ban = (torch.rand(40, vocab, generator=g) < 0.7).to(device)
    ban.scatter_(1, t[:, None], False)
    ban[7] = True                      # a row with nothing left
    ban[8] = True
    ban[8, vocab - 1] = False          # a row with one token, not its target
    x.masked_fill_(ban, -math.inf)
    x[9] = torch.finfo(dtype).min      # a row masked by the type's lowest value alone
    x[10, :vocab // 2] = torch.finfo(dtype).min
    t[11], t[12] = -100, -100
    check(x, t, min(5, vocab))
    check_gradient(x[:8], t[:8], 0, ("logprob", "entropy"))
    check_gradient(x[9:], t[9:], 2, ("logprob", "entropy", "top_logprob"))
    r = token_logprobs(x[7:9], t[7:9], top_k=3)
    assert r.logprob.tolist() == [-math.inf, -math.inf] and r.entropy.tolist() == [0.0, 0.0]
    assert r.top_index[0].tolist() == [0, 1, 2]
    assert r.top_logprob[1].tolist() == [0.0, -math.inf, -math.inf]
    leaf = x[7:8].detach().requires_grad_()
    r = token_logprobs(leaf, t[7:8], top_k=3)
    d, = torch.autograd.grad([r.entropy.sum() + r.logprob.sum() + r.top_logprob.sum()], leaf)
    assert not d.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_not_a_number(device, dtype):
    x, t = make((6, 3000), dtype, device)
    x[1, 17] = math.nan
    x[2, 2999] = math.inf
    x[3] = math.nan
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, t, top_k=4)
    bad = torch.tensor([False, True, True, True, False, False])
    assert torch.equal(r.logprob.isnan().cpu(), bad) and torch.equal(r.entropy.isnan().cpu(), bad)
    assert bool((r.top_index >= 0).all()) and bool((r.top_index < 3000).all())
    assert all(len(set(row)) == 4 for row in r.top_index.tolist())
    assert 17 not in r.top_index[1].tolist() and r.top_index[2, 0] == 2999
    d, = torch.autograd.grad(r.logprob.sum(), leaf)
    assert torch.equal(d.isnan().all(dim=1).cpu(), bad)
    assert torch.equal(d.isnan().any(dim=1).cpu(), bad)


def test_targets_outside_the_vocabulary(device):
    x, _ = make((5, 100), torch.float32, device)
    t = torch.tensor([-1, 100, -100, 2 ** 40, 99], device=device)
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, t)
    assert r.logprob.isnan().tolist() == [True, True, False, True, False] and r.logprob[2] == 0.0
    assert bool(r.entropy.isfinite().all())
    d, = torch.autograd.grad(r.logprob.sum(), leaf)
    assert d.isnan().all(dim=1).tolist() == [True, True, False, True, False]
    assert not d[2].any()
    r = token_logprobs(x, t, ignore_index=-1)
    assert r.logprob[0] == 0.0 and bool(r.logprob[2].isnan())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,rows", [(65, 3), (4000, 300), (50304, 2)])
def test_ties_take_the_lowest_index(device, dtype, vocab, rows):
    """Equal logits everywhere (a zero-initialised head), few distinct values, and the largest values all in the
    elements of one thread, more of them than the candidates' buffer holds."""
    k = 64
    x = torch.zeros(rows, vocab, dtype=dtype, device=device)
    x[0, 5:9] = -0.0
    t = torch.zeros(rows, dtype=torch.int64, device=device)
    check(x, t, k)
    g = torch.Generator().manual_seed(1)
    x = torch.randint(0, 3, (rows, vocab), generator=g).to(dtype).to(device)
    check(x, t, k)
    x = torch.arange(vocab, 0, -1).float().expand(rows, vocab).div(vocab).to(dtype).to(device)
    check(x, t, k)
    x = x.flip(1).contiguous()
    check(x, t, k)


def test_top_values_crowded_in_few_threads(device):
    """64 threads hold 100 large elements each."""
    vocab = 100 * 1024 * 4
    x = torch.zeros(1, vocab)
    pos = torch.arange(vocab)
    x[0, (pos // 4) % 256 < 64] = 1.0
    x[0] += (pos % 977) / 4096.0
    x = x.to(device)
    t = torch.zeros(1, dtype=torch.int64, device=device)
    want = torch.sort(x.cpu(), dim=1, descending=True, stable=True).indices[:, :64]
    r = token_logprobs(x, t, top_k=64)
    assert torch.equal(r.top_index.cpu(), want)
    r = token_logprobs(x.expand(257, -1), t.expand(257), top_k=64)  # the other workgroup size, rows of one memory
    assert torch.equal(r.top_index.cpu(), want.expand(257, -1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(device, dtype):
    full, t = make((6, 1003), dtype, device)
    check(full[:, :1000], t.clamp(max=999), 3)           # padded columns
    check(full[:, 1:], t.clamp(max=1001), 3)             # rows at odd addresses
    check(full[::2], t[::2], 3)
    check(full.T.contiguous().T, t, 3)                   # vocabulary not contiguous
    check(full.view(2, 3, 1003).transpose(0, 1), t.view(2, 3).T, 3)
    check(full[:1].expand(4, -1), t[:4], 3)
    check_gradient(full[:, 1:1000], t.clamp(max=998), 2, ("logprob", "entropy", "top_logprob"))
    leaf = full[0].detach().clone().requires_grad_()     # the gradient of a broadcast row is summed
    r = token_logprobs(leaf.expand(4, -1), t[:4])
    d, = torch.autograd.grad(r.logprob.sum(), leaf)
    want = torch.stack([torch.autograd.grad(token_logprobs(leaf, t[i]).logprob, leaf)[0].float() for i in range(4)])
    size = want.abs().sum(0)
    assert bool(((d.float() - want.sum(0)).abs() <= size * torch.finfo(dtype).eps * 4 + 1e-6).all())
    check(full[0], t[0], 3)                              # no leading dimension
    check(full[:0], t[:0], 3)                            # no rows
    leaf = full[:0].detach().requires_grad_()
    assert torch.autograd.grad(token_logprobs(leaf, t[:0]).logprob.sum(), leaf)[0].shape == (0, 1003)


def test_refusals(device):
    x, t = make((4, 10), torch.float32, device)
    for bad in (-1, 11, 65):
        with pytest.raises(ValueError, match="top_k"):
            token_logprobs(x, t, top_k=bad)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(x.repeat(1, 10), t, top_k=65)
    with pytest.raises(TypeError, match="integer"):
        token_logprobs(x, t, top_k=1.5)
    with pytest.raises(TypeError, match="int64"):
        token_logprobs(x, t.int())
    with pytest.raises(TypeError, match="fp32"):
        token_logprobs(x.double(), t)
    with pytest.raises(ValueError, match="shape"):
        token_logprobs(x, t[:3])
    with pytest.raises(ValueError, match="vocabulary"):
        token_logprobs(x[:, :0], t)
    with pytest.raises(ValueError, match="on"):
        token_logprobs(x, t.to("meta"))
    leaf = x.detach().requires_grad_()
    d, = torch.autograd.grad(token_logprobs(leaf, t).logprob.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)


def test_same_bits_again(device):
    x, t = make((300, 5003), torch.bfloat16, device)
    a, b = (token_logprobs(x, t, top_k=7) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_side_stream_and_graph(hip):
    """Calls on another stream, and forward + backward captured into a graph and replayed with new inputs between
    eager calls."""
    x, t = make((64, 5003), torch.bfloat16, hip)
    want = token_logprobs(x, t, top_k=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(x, t, top_k=3)
        leaf = x.detach().clone().requires_grad_()
        w = torch.randn(64, device=hip)

        def both():
            r = token_logprobs(leaf, t, top_k=3)
            d, = torch.autograd.grad([r.logprob, r.entropy], leaf, [w, w])
            return (*(y.detach() for y in r), d)  # no graph of the leaf outlives the call

        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in range(4):
        y, _ = make((64, 5003), torch.bfloat16, hip, seed=20 + seed)
        with torch.no_grad():
            leaf.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        got = [h.clone() for h in held]
        assert all(torch.equal(p, q) for p, q in zip(got, both()))


@pytest.mark.gpu
def test_offsets_past_32_bits(hip):
    """A row that starts behind 2^32 bytes and 2^31 elements."""
    rows, vocab = 17001, 131072
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=hip)
    g = torch.Generator(device=hip).manual_seed(2)
    x[-3:] = torch.randn(3, vocab, generator=g, device=hip).bfloat16()
    t = torch.randint(0, vocab, (rows,), generator=g, device=hip)
    leaf = x.requires_grad_()
    r = token_logprobs(leaf, t, top_k=2)
    d, = torch.autograd.grad(r.logprob.sum(), leaf)
    few = x.detach()[-3:].clone().requires_grad_()
    s = token_logprobs(few, t[-3:], top_k=2)
    e, = torch.autograd.grad(s.logprob.sum(), few)
    assert torch.equal(r.top_index[-3:], s.top_index)
    close(r.logprob[-3:], s.logprob.cpu(), 2 * sum_error(vocab))
    close(d[-3:], e.cpu(), e.cpu().double().abs() * 2.0 ** -7 + 1e-9)
    assert r.top_index[0].tolist() == [0, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("top_k", [0, 2])
def test_more_rows_than_a_launch_has(hip, top_k):
    """2^26 + 3 short rows: equal rows have equal results, wherever they stand."""
    rows, vocab = (1 << 26) + 3, 5
    few, few_t = make((7, vocab), torch.float16, hip)
    x = few.repeat(rows // 7 + 1, 1)[:rows].requires_grad_()
    t = few_t.repeat(rows // 7 + 1)[:rows]
    r = token_logprobs(x, t, top_k=top_k)
    results = [y for y in r if y is not None]
    d, = torch.autograd.grad([y for y in results if y.requires_grad], x,
                             [torch.ones_like(y) for y in results if y.requires_grad])
    leaf = few.clone().requires_grad_()
    s = [y for y in token_logprobs(leaf, few_t, top_k=top_k) if y is not None]
    e, = torch.autograd.grad([y for y in s if y.requires_grad], leaf,
                             [torch.ones_like(y) for y in s if y.requires_grad])
    n = rows // 7
    for got, want in zip(results + [d], s + [e]):
        got, want = got.detach(), want.detach()
        assert bool((got[:7 * n].view(n, 7, -1) == want.reshape(7, -1)).all())
        assert torch.equal(got[7 * n:], want[:rows - 7 * n])


def edge_positions(vocab, width):
    """Columns where a split of the row over threads, unrolled loads or blocks of `width` elements could lose or double
    one: the ends, and both sides of every multiple of 4 x 64 .. 4 x 512 blocks and of the remainders behind them."""
    at = set(range(min(vocab, 2 * width + 1))) | set(range(max(0, vocab - 3 * width), vocab))
    for threads in (64, 128, 256, 512):
        sweep = 4 * threads * width
        for edge in [*range(sweep, vocab, sweep)][-2:] + [vocab // sweep * sweep + threads * width * k for k in range(4)]:
            at |= {edge - 1, edge, edge + 1, edge + width - 1, edge + width}
    return sorted(i for i in at if 0 <= i < vocab)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,top_k", [(50257, 0), (50304, 2), (50257, 3), (9001, 3), (8191, 0), (4100, 2), (1023, 3),
                                         (255, 0)])
def test_every_element_counts_once(device, dtype, vocab, top_k):
    """Rows of which two or three entries have all the mass, so that losing or doubling one shows. The sums then have
    three terms, each off by at most 4 u and rounded twice."""
    positions = edge_positions(vocab, 16 // dtype.itemsize)
    n = len(positions)
    at = torch.tensor([[p, (7 * p + 13) % vocab, vocab - 1 - p] for p in positions])
    x = torch.full((n, vocab), -1e4)
    x.scatter_(1, at, torch.tensor([1.0, 0.5, 0.0]).expand(n, 3))  # of equal places one counts
    x = x.to(dtype)
    targets = at[:, 0]
    lp, entropy, top_lp, index, logp, p = reference(x, targets, top_k)
    leaf = x.to(device).requires_grad_()
    r = token_logprobs(leaf, targets.to(device), top_k=top_k)
    close(r.logprob, lp, 32 * U)
    close(r.entropy, entropy, 32 * U)
    if top_k:
        assert torch.equal(r.top_index[:, :2].cpu(), index[:, :2])
        close(r.top_logprob[:, :2], top_lp[:, :2], 32 * U)
    d, = torch.autograd.grad(r.logprob.sum(), leaf)
    want = -p
    want.scatter_add_(1, targets[:, None], torch.ones(n, 1, dtype=torch.float64))
    close(d, want, want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + 64 * U)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_masked_targets_and_alternatives(device, dtype):
    """Their log probability is -inf; 1 - p = 1 of their upstream gradient reaches them, and nothing a masked token that
    is neither."""
    x = torch.full((3, 40), -math.inf, dtype=dtype, device=device)
    x[:, :3] = torch.tensor([1.0, 2.0, 0.5], dtype=dtype, device=device)
    t = torch.tensor([1, 7, 4], device=device)
    leaf = x.requires_grad_()
    r = token_logprobs(leaf, t, top_k=5)
    assert r.top_index.tolist() == [[1, 0, 2, 3, 4]] * 3
    assert r.logprob.isneginf().tolist() == [False, True, True] and bool(r.top_logprob[:, 3:].isneginf().all())
    g_lp, g_top = torch.tensor([1.0, 2.0, 4.0], device=device), torch.arange(1.0, 6.0, device=device).repeat(3, 1)
    d, = torch.autograd.grad([r.logprob, r.top_logprob], leaf, [g_lp, g_top])
    want = torch.zeros(3, 40)
    want[:, 3:5] += torch.tensor([4.0, 5.0])  # exact in every type
    want[1, 7] += 2.0
    want[2, 4] += 4.0
    assert torch.equal(d[:, 3:].cpu().float(), want[:, 3:])
    # p is off by at most 64 u; the upstream gradients add up to at most 20
    p = torch.softmax(x[:, :3].detach().cpu().double(), dim=1)
    at = torch.tensor([[2.0, 1.0, 3.0]]).repeat(3, 1).double()  # alternatives' own
    at[0, 1] += 1.0
    close(d[:, :3], at - p * (15.0 + g_lp.cpu()[:, None]),
          64 * U * 20 + torch.finfo(dtype).eps / 2 * (at - p * (15.0 + g_lp.cpu()[:, None])).abs() * 1.01)
