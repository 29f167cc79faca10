"""Log probabilities of given tokens with entropy and the most likely alternatives (CUDA: ``csrc/token_logprobs.cu``, CPU: the oracle in
``ref/logprob.py``)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ..ref import logprob as _ref

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                   # fp32 [T]
    entropy: torch.Tensor                   # fp32 [T]
    top_logprobs: Optional[torch.Tensor]    # fp32 [T, top_k]
    top_ids: Optional[torch.Tensor]         # int64 [T, top_k]


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, top_k):
        from . import logprob_cuda
        lp, ent, stat, top, top_ids = logprob_cuda.forward(logits, ids, top_k)
        ctx.save_for_backward(logits, ids, stat, ent)
        ctx.set_materialize_grads(False)
        if top is None:
            return lp, ent
        ctx.mark_non_differentiable(top, top_ids)
        return lp, ent, top, top_ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_lp, g_ent, *_):
        if g_lp is None and g_ent is None:
            return None, None, None
        from . import logprob_cuda
        logits, ids, stat, ent = ctx.saved_tensors
        return logprob_cuda.backward(logits, ids, stat, ent, g_lp, g_ent), None, None


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Scores of the tokens ``ids`` [T] int64 under ``logits`` [T, V] (bf16, fp16 or fp32; statistics in fp32).

    ``logprob[t]`` = log softmax(logits[t])[ids[t]], and 0 where the id is outside the vocabulary (the -100 of packed batches);
    ``entropy[t]`` = -sum p log p in nats; with ``top_k`` (at most 32) the largest log probabilities and their tokens, descending, the
    lowest token first among equal ones. Impossible tokens (-inf) have log probability -inf and no share in the entropy; a row of
    -inf only has entropy 0 and no gradient; NaN or +inf in a row makes its scores NaN. ``logprob`` and ``entropy`` are
    differentiable (once) in ``logits``."""
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float16, torch.float32) or logits.shape[1] == 0:
        raise ValueError("logits: bf16, fp16 or fp32 [tokens, vocabulary]")
    if ids.dtype != torch.int64 or ids.shape != logits.shape[:1]:
        raise ValueError("ids: int64 [tokens]")
    if ids.device != logits.device:
        raise ValueError(f"tensors on {logits.device} and {ids.device}")
    if not 0 <= top_k <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f"top_k {top_k}: 0 .. {min(MAX_TOP, logits.shape[1])}")
    if not logits.is_cuda:
        return TokenLogprobs(*_ref.token_logprobs(logits, ids, top_k))
    from . import logprob_cuda
    logprob_cuda.check_vocab(logits.shape[1])
    if torch.is_grad_enabled() and logits.requires_grad:
        got = _TokenLogprobs.apply(logits, ids, top_k)
        return TokenLogprobs(*got) if top_k else TokenLogprobs(got[0], got[1], None, None)
    lp, ent, _, top, top_ids = logprob_cuda.forward(logits, ids, top_k)
    return TokenLogprobs(lp, ent, top, top_ids)
