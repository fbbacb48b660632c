"""The operators at both ends of a language model: rows of an embedding table for token ids (scaled, with a dense gradient that is
the same every time), and log probabilities of given tokens under rows of logits, with entropies and the most likely
alternatives.  Over the C ABI (fpb_embedding_*, fpb_token_scores_*)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from flash_pop_b200 import _lib
from flash_pop_b200.layer_ops import _OK_DTYPES, _ptr

MAX_TOP = 32


def _check_ids(tokens: Tensor, like: Tensor) -> None:
    if tokens.dtype not in (torch.int64, torch.int32) or tokens.device != like.device:
        raise ValueError(f"tokens: int64 or int32 ids on {like.device}; got {tokens.dtype} on {tokens.device}")


def _matrix(t: Tensor) -> Tensor:
    """(rows, n) with unit inner stride and rows that do not overlap, copied if that is not what `t` is."""
    ok = (t.stride(1) == 1 or t.size(1) == 1) and (t.size(0) <= 1 or t.stride(0) >= t.size(1))
    return t if ok else t.contiguous()


def _pitch(t: Tensor) -> int:
    return t.stride(0) if t.size(0) > 1 else t.size(1)


class Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        _check_embedding(tokens, weight)
        tokens = tokens.to(torch.int64)
        w, ids = _matrix(weight), tokens.contiguous()
        V, D = w.shape
        N = ids.numel()
        y = torch.empty((*tokens.shape, D), device=w.device, dtype=w.dtype)
        with torch.cuda.device(w.device):
            _lib.check(_lib.lib().fpb_embedding_fwd(N, V, D, _lib.dtype_code(w), _ptr(ids), _ptr(w), _pitch(w), scale, _ptr(y),
                                                    _lib.stream_ptr(w.device)))
        ctx.save_for_backward(ids)
        ctx.of = V, D, w.dtype, scale, padding
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        _lib.native().capturable()
        V, D, dtype, scale, padding = ctx.of
        N = ids.numel()
        dy = _matrix(dy.to(dtype).reshape(N, D))
        dw = torch.empty((V, D), device=dy.device, dtype=dtype)
        need = _lib.lib().fpb_embedding_workspace(N, V, D)
        with torch.cuda.device(dy.device):
            scratch = torch.empty(need, device=dy.device, dtype=torch.uint8)
            _lib.check(_lib.lib().fpb_embedding_bwd(N, V, D, _lib.dtype_code(dy), _ptr(ids), padding, scale, _ptr(dy), _pitch(dy), _ptr(dw),
                                                    _ptr(scratch), need, _lib.stream_ptr(dy.device)))
        return None, dw, None, None


def _check_embedding(tokens: Tensor, weight: Tensor) -> None:
    _lib.require_cuda(tokens, weight)
    if weight.dim() != 2 or weight.size(0) == 0 or weight.size(1) == 0:
        raise ValueError(f"weight: (V, D), neither 0; got {tuple(weight.shape)}")
    if weight.dtype not in _OK_DTYPES:
        raise ValueError(f"weight: bfloat16 or float32; got {weight.dtype}")
    _check_ids(tokens, weight)


def embedding(tokens: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """``weight[tokens] * scale`` for ids of any shape and a (V, D) table, in the table's dtype.  An id outside [0, V) gives a zero
    row and has no part in the gradient.  The gradient of the table is dense; rows are summed in fp32 in the order of the
    ids and rounded once, so it is the same every time.  `padding_idx` (negative: from the end): its row gets no gradient."""
    scale, padding = float(scale), -1
    if padding_idx is not None:
        V = weight.size(0)
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx {padding_idx} outside a table of {V} rows")
        padding = padding_idx % V
    fast = _lib.result(_lib.native().embedding(tokens, weight, scale, padding))
    if fast is not None:
        return fast[0]
    return Embedding.apply(tokens, weight, scale, padding)


class TokenScores(NamedTuple):
    logprob: Tensor                       # of the given tokens, fp32
    entropy: Tensor                       # of each row, in nats, fp32
    top_logprob: Optional[Tensor]         # (..., top) fp32, the most likely first; None without alternatives
    top_tokens: Optional[Tensor]          # (..., top) int64


def _check_scores(logits: Tensor, tokens: Tensor, top: int) -> None:
    _lib.require_cuda(logits, tokens)
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"logits (..., V) and tokens (...): got {tuple(logits.shape)} and {tuple(tokens.shape)}")
    V = logits.size(-1)
    if V == 0:
        raise ValueError("logits over no tokens")
    if logits.dtype not in _OK_DTYPES:
        raise ValueError(f"logits: bfloat16 or float32; got {logits.dtype}")
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top: 0 to {min(MAX_TOP, V)} of {V} tokens; got {top}")
    _check_ids(tokens, logits)


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        _check_scores(logits, tokens, top)
        shape, V = tokens.shape, logits.size(-1)
        tokens, z = tokens.to(torch.int64).reshape(-1).contiguous(), _matrix(logits.reshape(-1, V))
        rows, dev = tokens.numel(), z.device
        new = lambda *extra, dtype=torch.float32: torch.empty((*shape, *extra), device=dev, dtype=dtype)
        logprob, entropy, stats = new(), new(), torch.empty((rows, 2), device=dev, dtype=torch.float32)
        top_logprob, top_tokens = (new(top), new(top, dtype=torch.int64)) if top else (None, None)
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().fpb_token_scores_fwd(rows, V, _lib.dtype_code(z), top, _ptr(z), _pitch(z), _ptr(tokens), _ptr(logprob),
                                                       _ptr(entropy), _ptr(stats), _ptr(top_logprob), _ptr(top_tokens), _lib.stream_ptr(dev)))
        logits = z.view(logits.shape) if z.is_contiguous() else logits
        ctx.save_for_backward(logits, tokens, entropy, stats, top_tokens)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_tokens)
        return logprob, entropy, top_logprob, top_tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_top, _):
        logits, tokens, entropy, stats, top_tokens = ctx.saved_tensors
        _lib.native().capturable()
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None
        V = logits.size(-1)
        z = _matrix(logits.reshape(-1, V))
        rows = z.size(0)
        g_logprob, g_entropy, g_top = (None if g is None else g.to(torch.float32).contiguous() for g in (g_logprob, g_entropy, g_top))
        d = torch.empty(logits.shape, device=z.device, dtype=z.dtype)
        with torch.cuda.device(z.device):
            _lib.check(_lib.lib().fpb_token_scores_bwd(rows, V, _lib.dtype_code(z), 0 if top_tokens is None else top_tokens.size(-1), _ptr(z), _pitch(z),
                                                       _ptr(tokens), _ptr(entropy), _ptr(stats), _ptr(top_tokens), _ptr(g_logprob), _ptr(g_entropy),
                                                       _ptr(g_top), _ptr(d), V, _lib.stream_ptr(z.device)))
        return d, None, None


def token_scores(logits: Tensor, tokens: Tensor, top: int = 0) -> TokenScores:
    """Log probabilities of `tokens` (...) under `logits` (..., V), the entropy of every row, and its `top` (at most 32) most likely
    tokens with their log probabilities, equal logits by index; fp32 arithmetic, one read of the logits.  All but the indices are
    differentiable (one more read and one write).  A token outside [0, V) has the log probability 0 and sends no gradient
    (`cross_entropy`'s rule).  A row of -inf only gives -inf, entropy 0 and no gradient; NaN or +inf in a row make its numbers NaN."""
    fast = _lib.result(_lib.native().token_scores(logits, tokens, top))
    if fast is not None:
        return TokenScores(*fast)
    return TokenScores(*_TokenScores.apply(logits, tokens, top))
