"""Llama-2-shaped decoder on the native ops (the reference trains HF ``LlamaForCausalLM`` with
eager attention, bench_models/models/train_llama.py:486-520).

Per layer: RMSNorm -> fused QKV GEMM -> (RMS norm of each head of Q and K, in the pass of the
rotation) RoPE on Q and K -> causal flash attention -> output
GEMM with the residual in its epilogue -> RMSNorm -> fused gate|up GEMM -> SwiGLU -> down GEMM
with the residual in its epilogue.  The score matrix is never materialised, which is what lets
the sequence-2048 configuration fit comfortably.  ``tie_embeddings`` shares the token embedding
with the LM head (a parameter used by the first and the last pipeline stage).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn

from .. import ops


@dataclass
class LlamaConfig:
    vocab_size: int = 32000
    hidden_size: int = 4096
    intermediate_size: int = 11008
    num_layers: int = 32
    num_heads: int = 32
    max_seq_len: int = 2048
    rms_eps: float = 1e-5
    rope_theta: float = 10000.0
    tie_embeddings: bool = False
    qk_norm: bool = False                          # RMS norm of each head of the queries and keys
    rope_dim: Optional[int] = None                 # values of a head that rotate (default: all)
    rope_interleaved: bool = False                 # pairs (2i, 2i + 1)
    rope_scaling: Optional[ops.RopeScaling] = None


LLAMA_CONFIGS = {
    "llama2_7b": LlamaConfig(),
    "llama_tiny": LlamaConfig(vocab_size=256, hidden_size=64, intermediate_size=128, num_layers=4,
                              num_heads=4, max_seq_len=32),
}


def llama_config(name: str, **overrides) -> LlamaConfig:
    return LlamaConfig(**{**LLAMA_CONFIGS[name].__dict__, **overrides})


class LlamaBlock(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        d = cfg.hidden_size
        self.num_heads = cfg.num_heads
        self.eps = cfg.rms_eps
        self.input_norm = nn.Parameter(torch.ones(d))
        self.qkv = nn.Linear(d, 3 * d, bias=False)
        self.interleaved = cfg.rope_interleaved
        self.q_norm = self.k_norm = None
        if cfg.qk_norm:
            self.q_norm = nn.Parameter(torch.ones(d // cfg.num_heads))
            self.k_norm = nn.Parameter(torch.ones(d // cfg.num_heads))
        self.o_proj = nn.Linear(d, d, bias=False)
        self.post_norm = nn.Parameter(torch.ones(d))
        self.gate_up = nn.Linear(d, 2 * cfg.intermediate_size, bias=False)
        self.down = nn.Linear(cfg.intermediate_size, d, bias=False)

    def forward(self, x: torch.Tensor, delta, cos: torch.Tensor, sin: torch.Tensor):
        """(x, delta) -> (x', delta'): the residual stream is x + delta, summed inside the next
        RMSNorm launch so that every tensor of the stream has one consumer (its gradient is
        then complete when the norm's backward has added the part arriving through the sum)."""
        B, S, d = x.shape
        H = self.num_heads
        if delta is None:
            y = ops.rms_norm(x, self.input_norm, self.eps)
        else:
            y, x = ops.rms_norm(delta, self.input_norm, self.eps, residual=x)
        qkv = ops.linear(y, self.qkv.weight).view(B, S, 3, H, d // H)
        if self.q_norm is not None:
            qkv = ops.qk_norm_rope_qkv(qkv, self.q_norm, self.k_norm, cos, sin, self.eps,
                                       interleaved=self.interleaved)
            a = ops.attention_qkv(qkv, causal=True)
        elif self.interleaved or 2 * cos.shape[1] < d // H or ops.rope_qkv_in_one(qkv):
            a = ops.attention_qkv(ops.rope_qkv(qkv, cos, sin, interleaved=self.interleaved), causal=True)
        else:
            q, k = ops.rope(qkv[:, :, 0], cos, sin), ops.rope(qkv[:, :, 1], cos, sin)
            a = ops.attention(q, k, qkv[:, :, 2], causal=True)
        a = a.view(B, S, d)
        delta = ops.linear(a, self.o_proj.weight)
        y, x = ops.rms_norm(delta, self.post_norm, self.eps, residual=x)
        g = ops.swiglu(ops.linear(y, self.gate_up.weight))
        return x, ops.linear(g, self.down.weight)


class Llama(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.cfg = cfg
        self.embed = nn.Embedding(cfg.vocab_size, cfg.hidden_size)
        self.layers = nn.ModuleList([LlamaBlock(cfg) for _ in range(cfg.num_layers)])
        self.norm = nn.Parameter(torch.ones(cfg.hidden_size))
        self.lm_head = nn.Linear(cfg.hidden_size, cfg.vocab_size, bias=False)
        if cfg.tie_embeddings:
            self.lm_head.weight = self.embed.weight
        head_dim = cfg.hidden_size // cfg.num_heads
        if cfg.rope_dim is not None and (cfg.rope_dim % 2 or not 0 < cfg.rope_dim <= head_dim):
            raise ValueError(f"rope_dim {cfg.rope_dim} is no even part of a head of {head_dim}")
        cos, sin = ops.rope_tables(cfg.max_seq_len, cfg.rope_dim or head_dim,
                                   cfg.rope_theta, scaling=cfg.rope_scaling)
        self.register_buffer("rope_cos", cos, persistent=False)
        self.register_buffer("rope_sin", sin, persistent=False)
        for m in self.modules():
            if isinstance(m, (nn.Linear, nn.Embedding)):
                nn.init.normal_(m.weight, std=0.02)

    def forward(self, input_ids: torch.Tensor) -> torch.Tensor:
        S = input_ids.shape[1]
        x = ops.embedding(input_ids, self.embed.weight)
        cos, sin = self.rope_cos[:S], self.rope_sin[:S]
        delta = None
        for layer in self.layers:
            x, delta = layer(x, delta, cos, sin)
        if delta is None:
            y = ops.rms_norm(x, self.norm, self.cfg.rms_eps)
        else:
            y, _ = ops.rms_norm(delta, self.norm, self.cfg.rms_eps, residual=x)
        return ops.linear(y, self.lm_head.weight)


def causal_lm_loss(logits: torch.Tensor, input_ids: torch.Tensor) -> torch.Tensor:
    """Next-token cross entropy (shift by one), fused log-softmax + NLL."""
    V = logits.shape[-1]
    return ops.cross_entropy(logits[:, :-1].reshape(-1, V), input_ids[:, 1:].reshape(-1))
