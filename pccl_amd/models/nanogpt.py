"""GPT-2-style decoder (nanoGPT, the workload of the reference's DDP / DiLoCo examples).

Behavioural parity with /root/reference/python/examples/nanogptddp/model.py (GPTConfig defaults = GPT-2 124M,
pre-LN blocks, fused QKV projection, causal SDPA, GELU MLP, tied input/output embeddings, scaled init of residual
projections, AdamW param groups with/without weight decay, 6N+12LHQT FLOP estimate). Written for MI355X:

* attention is ``scaled_dot_product_attention`` (PyTorch-ROCm dispatches it to its CK/AOTriton flash kernels);
* training runs in bf16 autocast (MFU priced against the 2.5 PFLOP/s dense bf16 peak of one MI355X);
* AdamW uses the fused multi-tensor implementation when parameters live on the GPU; Muon, for the matrices of the
  blocks, is :class:`pccl_amd.parallel.Muon`;
* ``fused_loss`` takes the loss from the logits in their own type (:func:`pccl_amd.ops.token_logprobs`): no fp32 copy of
  (tokens, vocabulary), one pass forward and one backward. :meth:`GPT.score` and ``generate``'s log probabilities use
  the same kernel.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.logprobs import TokenLogprobs, token_logprobs
from ..parallel.muon import Muon

MI355X_BF16_DENSE_FLOPS = 2.5e15


@dataclass
class GPTConfig:
    block_size: int = 1024
    vocab_size: int = 50304  # 50257 padded to a multiple of 64
    n_layer: int = 12
    n_head: int = 12
    n_embd: int = 768
    dropout: float = 0.0
    bias: bool = True
    fused_loss: bool = False


class Block(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.n_head = cfg.n_head
        self.dropout = cfg.dropout
        self.ln_1 = nn.LayerNorm(cfg.n_embd, bias=cfg.bias)
        self.c_attn = nn.Linear(cfg.n_embd, 3 * cfg.n_embd, bias=cfg.bias)
        self.c_proj = nn.Linear(cfg.n_embd, cfg.n_embd, bias=cfg.bias)
        self.ln_2 = nn.LayerNorm(cfg.n_embd, bias=cfg.bias)
        self.c_fc = nn.Linear(cfg.n_embd, 4 * cfg.n_embd, bias=cfg.bias)
        self.mlp_proj = nn.Linear(4 * cfg.n_embd, cfg.n_embd, bias=cfg.bias)
        self.drop = nn.Dropout(cfg.dropout)

    def attention(self, x: torch.Tensor) -> torch.Tensor:
        b, t, c = x.shape
        qkv = self.c_attn(x).view(b, t, 3, self.n_head, c // self.n_head)
        q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)  # each (B, nh, T, hs)
        y = F.scaled_dot_product_attention(q, k, v, dropout_p=self.dropout if self.training else 0.0,
                                           is_causal=True)
        return self.drop(self.c_proj(y.transpose(1, 2).reshape(b, t, c)))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = x + self.attention(self.ln_1(x))
        return x + self.drop(self.mlp_proj(F.gelu(self.c_fc(self.ln_2(x)))))


class GPT(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.config = cfg
        self.wte = nn.Embedding(cfg.vocab_size, cfg.n_embd)
        self.wpe = nn.Embedding(cfg.block_size, cfg.n_embd)
        self.drop = nn.Dropout(cfg.dropout)
        self.h = nn.ModuleList(Block(cfg) for _ in range(cfg.n_layer))
        self.ln_f = nn.LayerNorm(cfg.n_embd, bias=cfg.bias)
        self.apply(self._init_weights)
        # GPT-2 scaled init of the residual projections
        for name, p in self.named_parameters():
            if name.endswith("c_proj.weight") or name.endswith("mlp_proj.weight"):
                nn.init.normal_(p, mean=0.0, std=0.02 / math.sqrt(2 * cfg.n_layer))

    @staticmethod
    def _init_weights(m: nn.Module) -> None:
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)
            if m.bias is not None:
                nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)

    def num_params(self, non_embedding: bool = True) -> int:
        n = sum(p.numel() for p in self.parameters())
        return n - self.wpe.weight.numel() if non_embedding else n

    def logits(self, idx: torch.Tensor) -> torch.Tensor:
        b, t = idx.shape
        assert t <= self.config.block_size, f"sequence {t} > block size {self.config.block_size}"
        pos = torch.arange(t, device=idx.device)
        x = self.drop(self.wte(idx) + self.wpe(pos))
        for blk in self.h:
            x = blk(x)
        x = self.ln_f(x)
        return F.linear(x, self.wte.weight)  # tied lm head

    def forward(self, idx: torch.Tensor, targets: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        logits = self.logits(idx)
        if targets is None:
            return logits[:, -1:, :], None
        if self.config.fused_loss:
            logprob = token_logprobs(logits.view(-1, logits.size(-1)), targets.reshape(-1), ignore_index=-1).logprob
            return logits, -logprob.sum() / (targets != -1).sum()
        loss = F.cross_entropy(logits.float().view(-1, logits.size(-1)), targets.view(-1), ignore_index=-1)
        return logits, loss

    def crop_block_size(self, block_size: int) -> None:
        assert block_size <= self.config.block_size
        self.config.block_size = block_size
        self.wpe.weight = nn.Parameter(self.wpe.weight[:block_size].detach().clone())

    def configure_optimizers(self, weight_decay: float, learning_rate: float, betas=(0.9, 0.95),
                             device_type: str = "cuda", optimizer: str = "adamw") -> torch.optim.Optimizer:
        """``optimizer``: "adamw", or "muon" for the matrices of the blocks with AdamW for the embeddings, biases and
        norms; one learning rate and weight decay serve both."""
        params = [p for p in self.parameters() if p.requires_grad]
        if optimizer == "muon":
            matrices = [p for p in self.h.parameters() if p.requires_grad and p.dim() == 2]
            hidden = set(matrices)
            rest = [p for p in params if p not in hidden]
            groups = [{"params": [p for p in rest if p.dim() >= 2], "weight_decay": weight_decay},
                      {"params": [p for p in rest if p.dim() < 2], "weight_decay": 0.0}]
            return Muon(matrices, [g for g in groups if g["params"]], lr=learning_rate, weight_decay=weight_decay,
                        betas=betas, fused=device_type == "cuda")
        if optimizer != "adamw":
            raise ValueError(f"optimizer must be 'adamw' or 'muon', got {optimizer!r}")
        decay = [p for p in params if p.dim() >= 2]
        no_decay = [p for p in params if p.dim() < 2]
        groups = [{"params": decay, "weight_decay": weight_decay}, {"params": no_decay, "weight_decay": 0.0}]
        return torch.optim.AdamW(groups, lr=learning_rate, betas=betas, fused=device_type == "cuda")

    def flops_per_token(self) -> float:
        c = self.config
        return 6 * self.num_params() + 12 * c.n_layer * c.n_head * (c.n_embd // c.n_head) * c.block_size

    def estimate_mfu(self, tokens_per_iter: int, dt: float, peak: float = MI355X_BF16_DENSE_FLOPS) -> float:
        return self.flops_per_token() * tokens_per_iter / dt / peak

    @torch.no_grad()
    def score(self, idx: torch.Tensor, targets: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
        """Log probability of ``targets[b, t]`` after ``idx[b, :t + 1]`` (0 where it is -1), the entropy of the model's
        distribution there and its ``top_k`` alternatives."""
        return token_logprobs(self.logits(idx), targets, top_k=top_k, ignore_index=-1)

    @torch.no_grad()
    def generate(self, idx: torch.Tensor, max_new_tokens: int, temperature: float = 1.0,
                 top_k: Optional[int] = None, return_logprobs: bool = False):
        """``idx`` with ``max_new_tokens`` sampled tokens behind it; with ``return_logprobs`` also their log
        probabilities (fp32, [batch, max_new_tokens]) under the model, before ``temperature`` and ``top_k``."""
        logprobs = []
        for _ in range(max_new_tokens):
            ctx = idx if idx.size(1) <= self.config.block_size else idx[:, -self.config.block_size:]
            raw, _ = self(ctx)
            raw = raw[:, -1, :]
            logits = raw / temperature
            if top_k is not None:
                v, _ = torch.topk(logits, min(top_k, logits.size(-1)))
                logits[logits < v[:, [-1]]] = -float("inf")
            token = torch.multinomial(F.softmax(logits, dim=-1), num_samples=1)
            if return_logprobs:
                logprobs.append(token_logprobs(raw, token[:, 0]).logprob)
            idx = torch.cat((idx, token), dim=1)
        if return_logprobs:
            none = torch.zeros((idx.size(0), 0), dtype=torch.float32, device=idx.device)
            return idx, torch.stack(logprobs, dim=1) if logprobs else none
        return idx
