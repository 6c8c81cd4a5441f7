"""The language model's operators as they are used together: GPT's loss, scores and sampled log probabilities on
token_logprobs, and the Muon optimizer on muon_step, against the formulas in 64 bits.

The tolerances of losses and log probabilities are those of tests/test_logprobs.py (a sum over the vocabulary V in fp32:
E = (2 V / 64 + 64) 2^-24 (1 + ln V)), of Muon steps those of tests/test_muon.py.
"""
import copy
import math
import os
import pickle
import subprocess
import sys

import pytest
import torch

from pccl_amd.models import GPT, GPTConfig
from pccl_amd.ops import muon_step, orthogonalize, token_logprobs
from pccl_amd.parallel import Muon, init_optimizer_state, state_tensors
from test_examples import EX, _run
from test_logprobs import close, sum_error
from test_muon import U, deviation, gradient, model_step

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
SIZES = [dict(n_layer=2, n_head=2, n_embd=64, block_size=64, vocab_size=512),  # every matrix in one workgroup
         dict(n_layer=1, n_head=5, n_embd=160, block_size=40, vocab_size=1003, bias=False)]


@pytest.fixture(params=DEVICES)
def device(request):
    if request.param == "cuda":
        request.getfixturevalue("hip")
    return torch.device(request.param)


def make(size, device, **kw):
    torch.manual_seed(5)
    model = GPT(GPTConfig(**size, **kw)).to(device)
    gen = torch.Generator().manual_seed(6)
    idx = torch.randint(size["vocab_size"], (3, 33), generator=gen).to(device)
    targets = idx.roll(-1, dims=1).clone()
    targets[1, 20:] = -1  # a padded sequence
    return model, idx, targets


def autocast(device, on):
    return torch.autocast(device_type=device.type, dtype=torch.bfloat16, enabled=on)


def reference_loss(logits, targets):
    """Mean negative log probability and its gradient, in 64 bits."""
    x, t = logits.detach().double().reshape(-1, logits.shape[-1]), targets.reshape(-1)
    used = t != -1
    logp = torch.log_softmax(x, dim=-1)
    d = logp.exp()
    d[torch.arange(len(t), device=t.device), t.clamp(min=0)] -= 1
    d = d * used[:, None] / used.sum()
    return -logp.gather(1, t.clamp(min=0)[:, None])[used].mean(), d.view(logits.shape), logp.view(logits.shape)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("mixed", [False, True])
def test_fused_loss(device, size, mixed):
    model, idx, targets = make(size, device, fused_loss=True)
    params = list(model.ln_f.parameters())
    with autocast(device, mixed):
        logits, loss = model(idx, targets)
    assert logits.dtype == (torch.bfloat16 if mixed else torch.float32)
    v = size["vocab_size"]
    want, want_d, _ = reference_loss(logits, targets)
    # an error E of every row, and of the mean over N rows: N 2^-24
    tol = sum_error(v) * 2 + targets.numel() * U * float(want)
    close(loss, want.cpu(), tol)
    d, = torch.autograd.grad(loss, logits, retain_graph=True)
    assert d.dtype == logits.dtype
    # p = exp(x - lse) is off by E, its product with the gradient of the mean and its type by their roundings
    tol = want_d.abs() * (torch.finfo(d.dtype).eps / 2 * 1.01) + 3 * sum_error(v) / int((targets != -1).sum())
    assert bool(((d.double() - want_d).abs() <= tol).all())
    # the rest of the backward pass is the model's own
    got = torch.autograd.grad(loss, params, retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(got, torch.autograd.grad(logits, params, grad_outputs=d)))


def test_fused_loss_is_off_by_default(device):
    model, idx, targets = make(SIZES[0], device)
    logits, loss = model(idx, targets)
    assert torch.equal(loss, torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten(),
                                                               ignore_index=-1))
    assert torch.equal(model(idx)[0], logits[:, -1:])


def test_loss_without_targets_is_nan(device):
    model, idx, _ = make(SIZES[0], device, fused_loss=True)
    assert bool(model(idx, torch.full_like(idx, -1))[1].isnan())


@pytest.mark.parametrize("size", SIZES)
def test_score(device, size):
    model, idx, targets = make(size, device)
    got = model.score(idx, targets, top_k=5)
    assert not got.logprob.requires_grad
    _, _, logp = reference_loss(model.logits(idx), targets)
    tol = sum_error(size["vocab_size"]) * 4
    want = torch.where(targets == -1, 0.0, logp.gather(2, targets.clamp(min=0)[..., None])[..., 0])
    close(got.logprob, want.cpu(), tol)
    close(got.entropy, -(logp.exp() * logp).sum(-1).cpu(), tol * 4)
    close(got.top_logprob, logp.topk(5).values.cpu(), tol)
    close(got.top_logprob, logp.gather(2, got.top_index).cpu(), tol)


@pytest.mark.parametrize("top_k", [None, 3])
def test_generate_with_logprobs(device, top_k):
    model, idx, _ = make(SIZES[0], device)
    torch.manual_seed(1)
    plain = model.generate(idx[:, :4], 6, temperature=0.8, top_k=top_k)
    torch.manual_seed(1)
    out, logprobs = model.generate(idx[:, :4], 6, temperature=0.8, top_k=top_k, return_logprobs=True)
    assert torch.equal(plain, out) and logprobs.shape == (3, 6) and logprobs.dtype == torch.float32
    for k in range(6):
        _, _, logp = reference_loss(model(out[:, :4 + k])[0], out[:, 4 + k:5 + k])
        close(logprobs[:, k], logp[:, 0].gather(1, out[:, 4 + k:5 + k])[:, 0].cpu(), sum_error(512) * 4)
    assert model.generate(idx, 0, return_logprobs=True)[1].shape == (3, 0)


def check_step(matrices, others, before, grads, twin, adamw, lr, wd):
    for p, (p0, b0), g in zip(matrices, before, grads):
        factor = 0.2 * math.sqrt(max(p.shape))
        want, _, u = model_step(p0, g, b0, lr, wd, 0.95, True, factor)
        tol = 3 * deviation(u, False) * 4 * lr * factor + want.abs() * U * 1.01
        tol = tol + 4 * U * (p0.double().abs() + lr * factor)
        assert bool(((p.detach().double() - want).abs() <= tol).all())
    for p, q in zip(others, twin):
        q.grad = p.grad.clone()
    adamw.step()
    assert all(torch.equal(p, q) for p, q in zip(others, twin))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("mixed", [False, True])
def test_training_steps(device, size, mixed):
    """Loss, its gradient and the optimizer's step, three times over; then scores by the trained model. Every matrix of
    the blocks follows Muon's formula, everything else AdamW bit for bit."""
    model, idx, targets = make(size, device, fused_loss=True)
    lr, wd = 1e-3, 0.1
    opt = model.configure_optimizers(wd, lr, device_type=device.type, optimizer="muon")
    assert isinstance(opt, Muon)
    init_optimizer_state(opt)
    matrices = [p for p in model.h.parameters() if p.dim() == 2]
    assert {id(p) for g in opt.param_groups if g["muon"] for p in g["params"]} == {id(p) for p in matrices}
    others = [p for g in opt.param_groups if not g["muon"] for p in g["params"]]
    assert len(matrices) == 4 * size["n_layer"] and len(matrices) + len(others) == len(list(model.parameters()))
    twin = [p.detach().clone().requires_grad_() for p in others]
    adamw = torch.optim.AdamW([{"params": [q for q in twin if q.dim() >= 2], "weight_decay": wd},
                               {"params": [q for q in twin if q.dim() < 2], "weight_decay": 0.0}], lr=lr,
                              betas=(0.9, 0.95), fused=device.type == "cuda")
    init_optimizer_state(adamw)
    for turn in range(3):
        opt.zero_grad()
        with autocast(device, mixed):
            logits, loss = model(idx, targets)
        loss.backward()
        want, _, _ = reference_loss(logits, targets)
        close(loss, want.cpu(), sum_error(size["vocab_size"]) * 2 + targets.numel() * U * float(want))
        before = [(p.detach().clone(), opt.state[p]["momentum_buffer"].clone()) for p in matrices]
        grads = [p.grad.clone() for p in matrices]
        assert opt.step() is None
        check_step(matrices, others, before, grads, twin, adamw, lr, wd)
    _, _, logp = reference_loss(model.logits(idx), targets)
    want = torch.where(targets == -1, 0.0, logp.gather(2, targets.clamp(min=0)[..., None])[..., 0])
    close(model.score(idx, targets).logprob, want.cpu(), sum_error(size["vocab_size"]) * 4)


@pytest.mark.gpu
def test_training_step_in_a_graph(hip):
    """Log probabilities, their gradient and the Muon step captured together, replayed with the program's own eager
    work between the replays."""
    gen = torch.Generator().manual_seed(3)
    w0 = (torch.randn(1003, 160, generator=gen) * 0.1).to(hip)
    x, t = torch.empty(96, 160, device=hip), torch.empty(96, dtype=torch.int64, device=hip)
    seed = torch.full((96,), -1 / 96, device=hip)

    def step(w, b):
        leaf = (x @ w.mT).requires_grad_()
        r = token_logprobs(leaf, t)
        d, = torch.autograd.grad(r.logprob, leaf, grad_outputs=seed)
        muon_step([w], [d.mT.contiguous() @ x], [b], lr=0.02)
        return r.logprob.detach()

    def data(turn):
        g = torch.Generator().manual_seed(20 + turn)
        x.copy_(torch.randn(96, 160, generator=g))
        t.copy_(torch.randint(1003, (96,), generator=g))

    w, b = w0.clone(), torch.zeros_like(w0)
    eager = []
    for turn in range(4):
        data(turn)
        eager.append((step(w, b).clone(), w.clone(), b.clone()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(w, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(w, b)
    w.copy_(w0)
    b.zero_()
    for turn in range(4):
        data(turn)
        graph.replay()
        scratch = w.new_empty(1 << 20).fill_(turn) @ w.new_ones(1 << 20)  # eager work that takes the allocator's blocks
        torch.cuda.synchronize()
        assert torch.equal(out, eager[turn][0]) and torch.equal(w, eager[turn][1]) and torch.equal(b, eager[turn][2])
        assert float(scratch) == turn << 20


def small_params(device, dtype=torch.float32):
    gen = torch.Generator().manual_seed(70)
    return [torch.randn(s, generator=gen).to(dtype).to(device).requires_grad_()
            for s in [(40, 24), (24, 40), (24,), (10, 24)]]


def fill_grads(params, turn):
    for i, p in enumerate(params):
        p.grad = gradient(tuple(p.shape) if p.dim() > 1 else (1, *p.shape), 80 + 10 * turn + i, p.device,
                          p.dtype).view(p.shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict(device, dtype, tmp_path):
    """A run that is saved and resumed goes on bit for bit; the momentum of bf16 matrices stays fp32."""
    def optimizer(params):
        return Muon(params[:2], params[2:], lr=0.02, weight_decay=0.1, fused=device.type == "cuda")
    params = small_params(device, dtype)
    opt = optimizer(params)
    for turn in range(2):
        fill_grads(params, turn)
        opt.step()
    torch.save({"p": [p.detach() for p in params], "o": opt.state_dict()}, tmp_path / "ckpt.pt")
    saved = torch.load(tmp_path / "ckpt.pt", map_location="cpu", weights_only=True)
    resumed = [p.to(device).requires_grad_() for p in saved["p"]]
    again = optimizer(resumed)
    again.load_state_dict(saved["o"])
    assert again.state[resumed[0]]["momentum_buffer"].dtype == torch.float32
    for turn in range(2, 4):
        for ps, o in ((params, opt), (resumed, again)):
            fill_grads(ps, turn)
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(params, resumed))
    assert all(torch.equal(opt.state[p]["momentum_buffer"], again.state[q]["momentum_buffer"])
               for p, q in zip(params[:2], resumed[:2]))


def test_state_is_shared(device):
    """init_optimizer_state changes no parameter and leaves every state tensor for the peers' shared state."""
    model, _, _ = make(SIZES[0], device)
    before = [p.detach().clone() for p in model.parameters()]
    opt = model.configure_optimizers(0.1, 1e-3, device_type=device.type, optimizer="muon")
    init_optimizer_state(opt)
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), before))
    names = state_tensors(model, opt)
    for name, p in model.named_parameters():
        state = {k.rsplit(".", 1)[1] for k in names if k.startswith(name + ".")}
        hidden = name.startswith("h.") and p.dim() == 2
        assert state == ({"momentum_buffer"} if hidden else {"step", "exp_avg", "exp_avg_sq"}), name


def test_groups_schedules_and_missing_gradients(device):
    params = small_params(device)
    opt = Muon([{"params": params[:1], "lr": 0.0, "weight_decay": 0.0}, {"params": params[1:2], "adjust_lr": "none"}],
               [{"params": params[2:3]}, {"params": params[3:]}], lr=0.1)
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5 ** k)
    fill_grads(params, 0)
    params[3].grad = None
    before = copy.deepcopy([p.detach() for p in params])
    calls = []

    def closure():
        calls.append(torch.is_grad_enabled())
        return 7.0
    assert opt.step(closure) == 7.0 and calls == [True]
    assert [torch.equal(p, q) for p, q in zip(params, before)] == [True, False, False, True]
    assert params[3] not in opt.state and len(opt.state) == 3
    schedule.step()
    assert [g["lr"] for g in opt.param_groups] == [0.0, 0.05, 0.05, 0.05]
    q, b = before[1].clone(), torch.zeros_like(before[1])
    muon_step([q], [params[1].grad], [b], lr=0.1, adjust_lr="none")
    assert torch.equal(params[1], q)


def test_mixed_types(device):
    """Matrices of two types in one group."""
    params = [gradient((20, 30), i, device, d).requires_grad_() for i, d in enumerate([torch.float32, torch.bfloat16])]
    want = [p.detach().clone() for p in params]
    opt = Muon(params, lr=0.1)
    fill_grads(params, 0)
    opt.step()
    for p, q in zip(params, want):
        muon_step([q], [p.grad], [torch.zeros(20, 30, device=device)], lr=0.1, adjust_lr="match_rms_adamw")
        assert torch.equal(p, q)


def test_refusals(device):
    params = small_params(device)
    with pytest.raises(ValueError, match="two dimensions"):
        Muon(params)
    with pytest.raises(ValueError, match="empty"):
        Muon([])
    with pytest.raises(ValueError, match="more than one|some parameters"):
        Muon(params[:2], params[1:])
    for bad in (dict(lr=math.nan), dict(momentum=2.0), dict(adjust_lr="other"), dict(steps=0), dict(eps=0.0),
                dict(coefficients=(9.0, 9.0, 9.0))):
        with pytest.raises(ValueError):
            Muon(params[:2], **bad)
        with pytest.raises(ValueError):
            Muon([{"params": params[:2], **bad}])
    sharded = gradient((4, 4), 0, device).requires_grad_()
    sharded.placements = ()  # what tells a DTensor
    with pytest.raises(TypeError, match="sharded"):
        Muon([sharded])
    opt = Muon(params[:1])
    with pytest.raises(ValueError, match="constructor"):
        opt.add_param_group({"params": params[2:], "muon": False})
    with pytest.raises(ValueError, match="two dimensions"):
        opt.add_param_group({"params": params[2:3]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": params[1:2]})
    sparse = torch.zeros(40, 24, device=device, requires_grad=True)
    opt = Muon([sparse])
    sparse.grad = torch.zeros(40, 24, device=device).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    with pytest.raises(ValueError, match="adamw"):
        make(SIZES[0], device)[0].configure_optimizers(0.1, 1e-3, device_type=device.type, optimizer="other")


@pytest.mark.parametrize("script,extra,same", [("train_pccl.py", ["--max-iters", "4", "--overlap"], "param_sum"),
                                               ("sync_diloco.py", ["--max-iters", "6", "--inner-steps", "3"],
                                                "outer_sum")])
def test_examples_with_muon(script, extra, same):
    res = _run(script, ["--optimizer", "muon", "--fused-loss", *extra])
    assert all(r["done"] for r in res) and res[0][same] == res[1][same]


@pytest.mark.gpu
def test_example_with_muon_gpu(hip):
    res = _run("train_pccl.py", ["--optimizer", "muon", "--fused-loss", "--max-iters", "4"], device="cuda")
    assert all(r["done"] and r["iter"] == 4 for r in res) and res[0]["param_sum"] == res[1]["param_sum"]


def test_sharded_example_refuses_muon():
    r = subprocess.run([sys.executable, os.path.join(EX, "sync_diloco_fsdp.py"), "--optimizer", "muon"],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 2 and "whole matrices" in r.stderr


def test_added_group_for_adamw_is_refused(device):
    """Parameters that no part of the optimizer would update are not taken, whatever settings come with them."""
    params = small_params(device)
    like_torch = torch.optim.AdamW(params[3:], lr=0.1).param_groups[0]
    for others in ([], params[2:3]):
        opt = Muon(params[:1], others, lr=0.1)
        groups = len(opt.param_groups)
        for settings in (dict(betas=(0.9, 0.95)), {k: v for k, v in like_torch.items() if k != "params"}):
            with pytest.raises(ValueError, match="constructor"):
                opt.add_param_group({"params": params[3:], "muon": False, **settings})
        opt.add_param_group({"params": params[1:2]})
        assert len(opt.param_groups) == groups + 1
        fill_grads(params, 0)
        before = copy.deepcopy([p.detach() for p in params])
        opt.step()
        held = {id(p) for g in opt.param_groups for p in g["params"]}
        assert [torch.equal(p, q) for p, q in zip(params, before)] == [id(p) not in held for p in params]


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "load"])
@pytest.mark.parametrize("with_others", [True, False])
def test_copies_go_on_alike(device, how, with_others):
    """A copied or unpickled optimizer, and one that takes over another's groups with its state, steps to equal bits."""
    params = small_params(device)
    take = params if with_others else params[:2]
    opt = Muon([{"params": params[:1], "lr": 0.05}, {"params": params[1:2], "nesterov": False}],
               [{"params": params[2:3], "weight_decay": 0.0}, {"params": params[3:]}] if with_others else [], lr=0.02,
               betas=(0.8, 0.9), fused=device.type == "cuda")
    for turn in range(2):
        fill_grads(params, turn)
        opt.step()
    if how == "deepcopy":
        copied, again = copy.deepcopy((take, opt))
    elif how == "pickle":
        copied, again = pickle.loads(pickle.dumps((take, opt)))
    else:
        copied = [p.detach().clone().requires_grad_() for p in take]
        # groups of matrices only: which part a group belongs to comes with the state
        again = Muon([{"params": [p.view(-1, 1).detach().requires_grad_()] if p.dim() == 1 else [p]} for p in copied])
        for g, p in zip(again.param_groups, copied):
            g["params"] = [p]
        again.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert [g["muon"] for g in again.param_groups] == [True, True, False, False][:len(take)]
    for turn in range(2, 4):
        for ps, o in ((params, opt), (copied, again)):
            fill_grads(ps, turn)
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(take, copied))
    assert all(p is not q for p, q in zip(take, copied))
    for p, q in zip(take, copied):
        for k, v in opt.state[p].items():
            assert again.state[q][k].dtype == v.dtype and torch.equal(again.state[q][k], v), k


def test_coefficients_of_a_group_and_as_tensors(device):
    """Any sequence of three numbers; what tensors among them hold is read anew by every call."""
    x = gradient((20, 30), 1, device)
    abc = torch.tensor([1.5, -0.5, 0.0], dtype=torch.float64)
    first = orthogonalize(x, coefficients=abc.unbind())
    assert torch.equal(first, orthogonalize(x, coefficients=[1.5, -0.5, 0.0]))
    numbers = abc.unbind()
    orthogonalize(x, coefficients=numbers)
    abc.copy_(torch.tensor([1.875, -1.25, 0.375]))
    assert torch.equal(orthogonalize(x, coefficients=numbers), orthogonalize(x, coefficients=(1.875, -1.25, 0.375)))
    abc[0] = 9.0
    with pytest.raises(ValueError, match="coefficients"):
        orthogonalize(x, coefficients=numbers)
    params = small_params(device)[:2]
    opt = Muon([{"params": params[:1], "coefficients": [1.5, -0.5, 0.0]}, {"params": params[1:]}], lr=0.1,
               coefficients=[1.875, -1.25, 0.375])
    fill_grads(params, 0)
    want = [(p.detach().clone(), torch.zeros_like(p)) for p in params]
    opt.step()
    for p, (q, b), c in zip(params, want, ((1.5, -0.5, 0.0), (1.875, -1.25, 0.375))):
        muon_step([q], [p.grad], [b], lr=0.1, adjust_lr="match_rms_adamw", coefficients=c)
        assert torch.equal(p, q)


def test_no_generated_token_has_fp32_logprobs(device):
    model, idx, _ = make(SIZES[0], device)
    kept = torch.get_default_dtype()
    torch.set_default_dtype(torch.float64)
    try:
        assert model.generate(idx, 0, return_logprobs=True)[1].dtype == torch.float32
    finally:
        torch.set_default_dtype(kept)
