"""Operators of one training step that run as hand-written kernels: Newton-Schulz orthogonalisation, the Muon step
that uses it, and log probabilities of given tokens (with entropy and top alternatives) with their gradient.

``run`` computes them in plain torch operations in 32 bits; with ``own`` set it makes the framework's calls instead.
``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one hidden matrix of the "tiny" preset: the call is latency
        dict(name="orth_tiny", op="orth", batch=1, rows=64, cols=64, dtype="f32"),
        # the attention projections of a 12-layer model of width 768, 16-bit gradients
        dict(name="orth_proj12", op="orth", batch=12, rows=768, cols=768, dtype="bf16"),
        # three tall odd-sized matrices (a cropped or sharded layer)
        dict(name="orth_odd_tall", op="orth", batch=3, rows=1801, cols=517, dtype="f16"),
        # two square matrices of a large model
        dict(name="orth_large", op="orth", batch=2, rows=4096, cols=4096, dtype="bf16"),
        # every matrix of the "tiny" preset (2 layers of width 64) in one step
        dict(name="muon_tiny", op="muon", layers=2, width=64, dtype="f32", nesterov=True),
        # 12 layers of width 640, fp32 parameters (autocast training)
        dict(name="muon_base", op="muon", layers=12, width=640, dtype="f32", nesterov=True),
        # 2 layers of width 2048, 16-bit parameters and gradients
        dict(name="muon_large", op="muon", layers=2, width=2048, dtype="bf16", nesterov=False),
        # one decoded token with five alternatives, GPT vocabulary
        dict(name="logp_token", op="logp", tokens=1, vocab=50304, pad=0, dtype="bf16", top_k=5, masked=False),
        # scoring a batch of prompts, the unpadded vocabulary as a view of padded logits
        dict(name="logp_score", op="logp", tokens=2047, vocab=50257, pad=47, dtype="f32", top_k=20, masked=True),
        # a batch of the GPT training workload: 12 sequences of 1024 tokens, log probabilities alone
        dict(name="logp_eval", op="logp", tokens=12288, vocab=50304, pad=0, dtype="bf16", top_k=0, masked=False),
        # the same batch with its gradient
        dict(name="loss_train", op="loss", tokens=12288, vocab=50304, pad=0, dtype="bf16", top_k=0, masked=False),
        # a small odd batch with gradients of log probability, entropy and alternatives
        dict(name="loss_odd", op="loss", tokens=515, vocab=32003, pad=5, dtype="f16", top_k=4, masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["orth", "muon", "logp", "loss"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "orth":
        rows, cols = _log(rng, 16, 4096), _log(rng, 16, 4096)
        batch = max(1, min(_log(rng, 1, 16), int(1.2e11 / (min(rows, cols) ** 2 * max(rows, cols)))))
        return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=dtype)
    if op == "muon":
        width = _log(rng, 24, 1500)
        return dict(op=op, layers=rng.randint(1, 6 if width > 700 else 12), width=width, dtype=rng.choice(["f32", "bf16"]),
                    nesterov=rng.random() < 0.7)
    tokens, vocab = _log(rng, 1, 12288), _log(rng, 300, 131072)
    tokens = min(tokens, max(1, int(4e8 / vocab)))
    return dict(op=op, tokens=tokens, vocab=vocab, pad=rng.choice([0, 0, 1, 47]), dtype=dtype,
                top_k=rng.choice([0, 1, 5, 20]), masked=rng.random() < 0.5)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _gradients(gen, batch, rows, cols, dtype):
    """Gradients of a linear layer: dY^T X over the tokens, with the decaying spectra that activations and their
    gradients have."""
    tokens = 2 * min(rows, cols)
    fall = lambda n, rate: torch.exp(-rate * torch.arange(n, device="cuda") / n)  # noqa: E731
    d_out = torch.randn(batch, tokens, rows, device="cuda", generator=gen) * fall(rows, 2.0)
    x = torch.randn(batch, tokens, cols, device="cuda", generator=gen) * fall(cols, 2.0)
    return (torch.matmul(d_out.transpose(1, 2).contiguous(), x) * (1e-3 / tokens)).to(dtype)


def prepare(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    if case["op"] == "orth":
        return dict(case=case, x=_gradients(gen, case["batch"], case["rows"], case["cols"], dtype))
    if case["op"] == "muon":
        d, layers = case["width"], case["layers"]
        stacks = {}
        for name, rows, cols in (("qkv", 3 * d, d), ("proj", d, d), ("up", 4 * d, d), ("down", d, 4 * d)):
            grads = _gradients(gen, layers, rows, cols, dtype)
            noise = _gradients(gen, layers, rows, cols, torch.float32)
            weight = torch.randn(layers, rows, cols, device="cuda", generator=gen) * 0.02
            stacks[name] = dict(weight=weight.to(dtype), grad=grads, momentum=grads.float() * 0.5 + noise)
        per = {k: [t for s in stacks.values() for t in s[k].unbind(0)] for k in ("weight", "grad", "momentum")}
        return dict(case=case, stacks=stacks, per=per, lr=0.02, weight_decay=0.1, momentum=0.95)
    tokens, vocab, pad = case["tokens"], case["vocab"], case["pad"]
    full = torch.randn(tokens, vocab + pad, device="cuda", generator=gen) * 2.5
    targets = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen)
    sure = torch.rand(tokens, device="cuda", generator=gen) < 0.5  # a trained model puts its mass on many of the targets
    full[torch.arange(tokens, device="cuda"), targets] += 9.0 * sure
    if case["masked"]:  # forbidden tokens, and padding positions without a target
        banned = torch.rand(vocab + pad, device="cuda", generator=gen) < 0.1
        banned[targets] = False
        full[:, banned] = -float("inf")
        targets[torch.rand(tokens, device="cuda", generator=gen) < 0.1] = -100
    logits = full.to(dtype)[:, :vocab]
    state = dict(case=case, logits=logits, targets=targets)
    if case["op"] == "loss":
        state["logits"] = logits.detach().requires_grad_()
        g = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
        state["grads"] = [-1.0 + 0.1 * g(tokens), 0.1 * g(tokens)] + ([0.1 * g(tokens, case["top_k"])] if case["top_k"] else [])
    return state


def run(state):
    case = state["case"]
    if case["op"] == "orth":
        return _own_orth(state) if own else _orth(state["x"].float()).to(state["x"].dtype)
    if case["op"] == "muon":
        return _own_muon(state) if own else _muon(state)
    return _own_logp(state) if own else _logp(state)


def _result(case, logprob, entropy, top_logprob, top_index, d_logits=None):
    out = dict(logprob=logprob, entropy=entropy)
    if case["top_k"]:
        out.update(top_logprob=top_logprob, top_index=top_index)
    if d_logits is not None:
        out["d_logits"] = d_logits
    return out


# --- the framework's calls ----------------------------------------------------------------------------------------
def _own_orth(state):
    from pccl_amd import ops
    return ops.orthogonalize(state["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)


def _own_muon(state):
    from pccl_amd import ops
    per = state["per"]
    ops.muon_step(per["weight"], per["grad"], per["momentum"], lr=state["lr"], weight_decay=state["weight_decay"],
                  momentum=state["momentum"], nesterov=state["case"]["nesterov"], steps=STEPS,
                  coefficients=COEFFICIENTS, eps=EPS, adjust_lr="match_rms_adamw")
    return {n: (s["weight"], s["momentum"]) for n, s in state["stacks"].items()}


def _own_logp(state):
    from pccl_amd import ops
    case = state["case"]
    r = ops.token_logprobs(state["logits"], state["targets"], top_k=case["top_k"], ignore_index=-100)
    if case["op"] == "logp":
        return _result(case, r.logprob, r.entropy, r.top_logprob, r.top_index)
    outs = [r.logprob, r.entropy] + ([r.top_logprob] if case["top_k"] else [])
    d_logits, = torch.autograd.grad(outs, state["logits"], state["grads"])
    return _result(case, *(t.detach() if t is not None else None for t in r), d_logits)


# --- plain forms --------------------------------------------------------------------------------------------------
def _orth(x):
    a, b, c = COEFFICIENTS
    flip = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if flip else x
    norm = x.double().square().sum(dim=(-2, -1), keepdim=True).sqrt().clamp(min=EPS)
    x = (x / norm).float().contiguous()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-1, -2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-1, -2).contiguous() if flip else x


def _muon(state):
    lr, mu, decay = state["lr"], state["momentum"], state["weight_decay"]
    for s in state["stacks"].values():
        grad, buf = s["grad"].float(), s["momentum"]
        buf.add_(grad - buf, alpha=1 - mu)
        update = _orth(grad + mu * (buf - grad) if state["case"]["nesterov"] else buf)
        scale = lr * 0.2 * math.sqrt(max(grad.shape[-2:]))
        s["weight"].copy_(s["weight"].float() * (1 - lr * decay) - scale * update)
    return {n: (s["weight"], s["momentum"]) for n, s in state["stacks"].items()}


def _top(x, k):
    """The k largest of each row, the lowest index first among equals: one integer key for value and index."""
    bits = x.float().add(0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits)
    key = order * (1 << 32) - torch.arange(x.shape[1], device=x.device)
    index = (-key.topk(k, dim=1, sorted=True).values) & 0xFFFFFFFF
    return index


def _logp(state):
    case = state["case"]
    k, targets = case["top_k"], state["targets"]
    logits = state["logits"].detach()
    x = logits.float()
    top = x.max(dim=1, keepdim=True).values
    shifted = x - top
    e = torch.exp(shifted)
    total = e.sum(dim=1, keepdim=True)
    log_total = total.log()
    logp = shifted - log_total
    p = e / total
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(dim=1)
    valid = targets != -100
    at = torch.where(valid, targets, 0)[:, None]
    logprob = torch.where(valid, logp.gather(1, at)[:, 0], 0.0)
    index = _top(x, k) if k else None
    top_logprob = logp.gather(1, index) if k else None
    if case["op"] == "logp":
        return _result(case, logprob, entropy, top_logprob, index)
    g_logprob, g_entropy, *g_top = state["grads"]
    g_logprob = torch.where(valid, g_logprob, 0.0)
    total_g = g_logprob + (g_top[0].sum(dim=1) if k else 0.0)
    d = -p * (total_g[:, None] + g_entropy[:, None] * torch.where(p > 0, logp + entropy[:, None], 0.0))
    d.scatter_add_(1, at, g_logprob[:, None])
    if k:
        d.scatter_add_(1, index, g_top[0])
    return _result(case, logprob, entropy, top_logprob, index, d.to(logits.dtype))


# --- 64 bits ------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orth":
        return _exact_orth(state["x"].double())
    if case["op"] == "muon":
        return _exact_muon(state)
    return _exact_logp(state)


def _exact_orth(x):
    """The polynomial on the right: X p(X^T X) = p(X X^T) X."""
    a, b, c = COEFFICIENTS
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=EPS)
    wide = x.shape[-1] >= x.shape[-2]
    y = x.mT.contiguous() if wide else x
    one = torch.eye(y.shape[-1], dtype=y.dtype, device=y.device)
    for _ in range(STEPS):
        g = y.mT.contiguous() @ y
        y = y @ (a * one + g @ (b * one + c * g))
    return y.mT.contiguous() if wide else y


def _exact_muon(state):
    lr, mu, decay = state["lr"], state["momentum"], state["weight_decay"]
    out = {}
    for name, s in state["stacks"].items():
        g = s["grad"].double()
        m = mu * s["momentum"].double() + (1 - mu) * g
        u = (1 - mu) * g + mu * m if state["case"]["nesterov"] else m
        step = _exact_orth(u) * (0.2 * max(g.shape[-2], g.shape[-1]) ** 0.5)
        out[name] = ((1 - lr * decay) * s["weight"].double() - lr * step, m)
    return out


def _exact_logp(state):
    case, targets = state["case"], state["targets"]
    x = state["logits"].detach().double()
    logp = x - torch.logsumexp(x, dim=1, keepdim=True)
    p = logp.exp()
    entropy = torch.special.entr(p).sum(dim=1)
    keep = targets >= 0
    rows = torch.arange(len(targets), device=x.device)
    at = targets.clamp(min=0)
    logprob = logp[rows, at].masked_fill(~keep, 0.0)
    k = case["top_k"]
    top_logprob = logp.topk(k, dim=1).values if k else None
    if case["op"] == "logp":
        return _result(case, logprob, entropy, top_logprob, None)
    g = [t.double() for t in state["grads"]]
    g[0] = g[0].masked_fill(~keep, 0.0)
    d = -p * g[0][:, None]
    d -= g[1][:, None] * (p * entropy[:, None] - torch.special.entr(p))
    d[rows, at] += g[0]
    if k:
        index = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        d -= p * g[2].sum(dim=1, keepdim=True)
        d.scatter_add_(1, index, g[2])
    return _result(case, logprob, entropy, top_logprob, None, d)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] in ("orth", "muon"):
        if case["op"] == "orth":
            shapes, moved = [(case["rows"], case["cols"], case["batch"])], 2 * size
        else:
            d, n = case["width"], case["layers"]
            shapes, moved = [(3 * d, d, n), (d, d, n), (4 * d, d, n), (d, 4 * d, n)], 3 * size + 8
        flops = 0
        for r, c, n in shapes:
            lo, hi = min(r, c), max(r, c)
            flops += n * STEPS * (3 * lo * lo * hi + lo ** 3)  # the symmetric products count their half
        return dict(bytes=moved * sum(r * c * n for r, c, n in shapes), flops=flops)
    tokens, vocab, k = case["tokens"], case["vocab"], case["top_k"]
    moved = tokens * (vocab * size + 16 + 12 * k)
    if case["op"] == "loss":
        moved += tokens * (vocab * size + 8 + 4 * k)
    return dict(bytes=moved, flops=tokens * vocab * (5 if case["op"] == "logp" else 11))
