"""GPT-2 (decoder-only transformer, learned positions, pre-LayerNorm, tied output embedding).

Not part of the reference repository; it is the fifth benchmark configuration (GPT-2 medium:
24 layers, d = 1024, 16 heads, vocabulary 50 257, sequence 1024, bf16 autocast with float32
gradients). Attention uses PyTorch's scaled-dot-product kernel; gradient compression is
independent of the sequence length, so no sequence parallelism is involved.

Documents of different lengths are trained on without padding, packed one behind another: `model.loss(tokens, targets,
offsets)` with the rows of document i from offsets[i] to offsets[i + 1]. Attention then is `packed_attention` and the
loss `token_log_probs`; both keep off the host, so that the lengths may change from step to step of a recorded graph. (A backward pass is recorded
while no earlier loss of the same parameters is alive: PyTorch would run the ends of it on that loss's stream.)
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.attention import packed_attention
from ..ops.tokens import TokenLogProbs, token_log_probs


@dataclass
class GPT2Config:
    vocab_size: int = 50257
    n_positions: int = 1024
    n_embd: int = 1024
    n_layer: int = 24
    n_head: int = 16
    dropout: float = 0.0

    @classmethod
    def medium(cls) -> "GPT2Config":
        return cls()

    @classmethod
    def small(cls) -> "GPT2Config":
        return cls(n_embd=768, n_layer=12, n_head=12)

    @classmethod
    def tiny(cls) -> "GPT2Config":
        return cls(vocab_size=512, n_positions=64, n_embd=64, n_layer=2, n_head=4)


class Block(nn.Module):
    def __init__(self, cfg: GPT2Config):
        super().__init__()
        self.ln_1 = nn.LayerNorm(cfg.n_embd)
        self.attn_qkv = nn.Linear(cfg.n_embd, 3 * cfg.n_embd)
        self.attn_proj = nn.Linear(cfg.n_embd, cfg.n_embd)
        self.ln_2 = nn.LayerNorm(cfg.n_embd)
        self.mlp_fc = nn.Linear(cfg.n_embd, 4 * cfg.n_embd)
        self.mlp_proj = nn.Linear(4 * cfg.n_embd, cfg.n_embd)
        self.n_head, self.dropout = cfg.n_head, cfg.dropout

    def forward(self, x: torch.Tensor, offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        if offsets is not None:
            t, c = x.shape
            q, k, v = self.attn_qkv(self.ln_1(x)).view(t, 3, self.n_head, c // self.n_head).unbind(1)
            x = x + self.attn_proj(packed_attention(q, k, v, offsets).reshape(t, c))
            return x + self.mlp_proj(F.gelu(self.mlp_fc(self.ln_2(x)), approximate="tanh"))
        b, t, c = x.shape
        q, k, v = self.attn_qkv(self.ln_1(x)).split(c, dim=2)
        shape = (b, t, self.n_head, c // self.n_head)
        q, k, v = (z.view(shape).transpose(1, 2) for z in (q, k, v))
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True, dropout_p=self.dropout if self.training else 0.0)
        x = x + self.attn_proj(y.transpose(1, 2).reshape(b, t, c))
        return x + self.mlp_proj(F.gelu(self.mlp_fc(self.ln_2(x)), approximate="tanh"))


class GPT2(nn.Module):
    def __init__(self, cfg: GPT2Config = GPT2Config()):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab_size, cfg.n_embd)
        self.wpe = nn.Embedding(cfg.n_positions, cfg.n_embd)
        self.h = nn.ModuleList(Block(cfg) for _ in range(cfg.n_layer))
        self.ln_f = nn.LayerNorm(cfg.n_embd)
        self.apply(self._init)
        for block in self.h:  # scaled init of the residual projections
            for proj in (block.attn_proj, block.mlp_proj):
                nn.init.normal_(proj.weight, std=0.02 / math.sqrt(2 * cfg.n_layer))

    @staticmethod
    def _init(module: nn.Module) -> None:
        if isinstance(module, (nn.Linear, nn.Embedding)):
            nn.init.normal_(module.weight, std=0.02)
        if isinstance(module, nn.Linear) and module.bias is not None:
            nn.init.zeros_(module.bias)

    def forward(self, tokens: torch.Tensor, offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Logits of [batch, time] tokens, or of [rows] tokens of packed documents (`offsets`: int32, see `packed_attention`; on the GPU
        under bf16 or fp16 autocast). A document's positions begin at zero, and from n_positions on are the
        last one (lengths are not known to the host, which could refuse them); rows that belong to no document give logits of no meaning."""
        if offsets is not None and self.cfg.dropout and self.training:
            raise ValueError("GPT2: packed documents are trained on without dropout")
        if tokens.dim() != (2 if offsets is None else 1):
            raise ValueError(f"GPT2: tokens {tuple(tokens.shape)}; [batch, time] is expected, or [rows] with offsets")
        t = tokens.shape[-1]
        pos = torch.arange(t, device=tokens.device, dtype=torch.int64 if offsets is None else torch.int32)
        if offsets is not None:
            document = torch.searchsorted(offsets[1:].contiguous(), pos, right=True, out_int32=True)
            pos = (pos - offsets[document].clamp_min(0)).clamp(0, self.cfg.n_positions - 1)   # (below zero attention begins at zero too)
        x = self.wte(tokens) + self.wpe(pos)
        for block in self.h:
            x = block(x) if offsets is None else block(x, offsets)
        return F.linear(self.ln_f(x), self.wte.weight)  # tied output embedding

    def loss(self, tokens: torch.Tensor, targets: torch.Tensor, offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Mean negative log probability of the targets; with `offsets`, of those that are not -100 (the end of a document, rows that belong to
        none)."""
        if offsets is not None:
            log_probs = self.score(tokens, targets, offsets).log_probs
            return -log_probs.sum() / (targets != -100).sum().clamp(min=1)
        logits = self(tokens)
        return F.cross_entropy(logits.view(-1, logits.size(-1)).float(), targets.reshape(-1))

    def score(self, tokens: torch.Tensor, targets: torch.Tensor, offsets: Optional[torch.Tensor] = None, **options) -> TokenLogProbs:
        """Log probabilities of the targets; `top`, `entropy` and `temperature` as in `token_log_probs`."""
        return token_log_probs(self(tokens, offsets), targets, **options)
