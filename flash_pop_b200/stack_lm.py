"""A token-level language-model wrapper around ``RetNetDecoder``: embedding -> decoder stack -> LayerNorm -> vocabulary
head.  The reference has no such wrapper (its decoders consume embeddings, tests/test_retention_layer.py:97-101);
this is the harness for the full-stack training configuration (12 layers, d_model 1024, 8 heads of 128, FFN 4096,
vocabulary 32000) and for users who want the same."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from flash_pop_b200.layer_ops import norm_in_fp32
from flash_pop_b200.recurrent_state import RecurrentState
from flash_pop_b200.retnet import RetNetDecoder, RetNetDecoderLayer
from flash_pop_b200.token_ops import TokenScores, embedding, token_scores


def _plain_embedding(m: nn.Module) -> bool:
    """An ``nn.Embedding`` whose rows are those of its weight, with nothing attached to it that a call would reach."""
    if type(m) is not nn.Embedding or m.max_norm is not None or m.sparse or m.scale_grad_by_freq or "forward" in m.__dict__:
        return False
    own, every = m.__dict__, nn.modules.module
    return not any(own.get(h, True) for h in ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")) and not (
        every._global_forward_hooks or every._global_forward_pre_hooks or every._global_backward_hooks or every._global_backward_pre_hooks)


class RetNetLM(nn.Module):
    def __init__(self, vocab_size: int = 32000, num_layers: int = 12, num_heads: int = 8, head_dim: int = 128,
                 dim_feedforward: int = 4096, dropout: float = 0.0, device="cuda", dtype=torch.bfloat16, embed_scale: Optional[float] = None,
                 qk_norm: bool = False, counter_dropout: bool = False):
        """embed_scale: the embedding's rows are multiplied by it, an id outside the table has a row of zeros, and the gradient is summed
        in a fixed order (None: a plain ``nn.Embedding``; an embedding with hooks, or another module in its place, is called, and its gradient is
        its own).  qk_norm, counter_dropout: see RetNetDecoderLayer.Config."""
        super().__init__()
        d_model = num_heads * head_dim
        cfg = RetNetDecoderLayer.Config(num_heads=num_heads, head_dim_v=head_dim, head_dim_qk=head_dim,
                                        dim_feedforward=dim_feedforward, dropout=dropout, device=device, dtype=dtype, qk_norm=qk_norm,
                                        counter_dropout=counter_dropout)
        self.embed_scale = embed_scale
        self.embed = nn.Embedding(vocab_size, d_model, device=device, dtype=dtype)
        self.decoder = RetNetDecoder(cfg, num_layers)
        self.norm = nn.LayerNorm(d_model, device=device, dtype=torch.float32)
        self.head = nn.Linear(d_model, vocab_size, bias=False, device=device, dtype=dtype)
        nn.init.normal_(self.embed.weight, std=d_model ** -0.5)
        nn.init.normal_(self.head.weight, std=d_model ** -0.5)

    def _rows(self, tokens: torch.Tensor) -> torch.Tensor:
        m = self.embed
        if self.embed_scale is None:
            return m(tokens)
        if _plain_embedding(m):
            return embedding(tokens, m.weight, self.embed_scale, m.padding_idx)
        inside = (tokens >= 0) & (tokens < getattr(m, "num_embeddings", self.head.out_features))
        return (m(tokens.masked_fill(~inside, 0)) * self.embed_scale).masked_fill(~inside.unsqueeze(-1), 0)

    def forward(self, tokens: torch.Tensor, recurrent_state: Optional[RecurrentState] = None):
        """tokens: (B, T) int64 -> logits (B, T, vocab), new RecurrentState."""
        x, state = self.decoder(self._rows(tokens), recurrent_state)
        return self.head(norm_in_fp32(self.norm, x)), state

    def loss(self, tokens: torch.Tensor) -> torch.Tensor:
        """Next-token cross entropy of `tokens` (B, T)."""
        logits, _ = self(tokens[:, :-1])
        return F.cross_entropy(logits.float().flatten(0, 1), tokens[:, 1:].flatten())

    def score(self, tokens: torch.Tensor, top: int = 0) -> TokenScores:
        """What the model says of `tokens` (B, T): for each of positions 1 to T-1 the log probability of the token that stands there,
        the entropy of the distribution it came from and, with `top`, the most likely tokens with their log probabilities; all
        (B, T-1[, top]), differentiable."""
        if tokens.size(1) < 2:                     # nothing before the first token to say anything of it
            return token_scores(self.head.weight.new_empty((tokens.size(0), 0, self.head.out_features)), tokens[:, 1:], top)
        logits, _ = self(tokens[:, :-1])
        return token_scores(logits, tokens[:, 1:], top)

    def flops_per_token(self, seq_len: int) -> float:
        """Training (forward + backward) FLOPs per token: 6 x matmul parameters + the retention operator."""
        layer = self.decoder.layers[0]
        d = layer.retention.embed_dim
        per_layer = 5 * d * d + 2 * d * layer.linear1.out_features
        matmul = len(self.decoder.layers) * per_layer + d * self.head.out_features
        H, dk, dv = layer.retention.num_heads, layer.retention.head_dim_qk, layer.retention.head_dim_v
        ch = 32.5
        retention = len(self.decoder.layers) * H * ((2 * ch * (dk + dv) + 4 * dk * dv) + (2 * ch * (3 * dk + 2 * dv) + 8 * dk * dv))
        return 6.0 * matmul + retention
