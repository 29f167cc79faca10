"""Log probabilities of given tokens with entropy and the most likely alternatives (CUDA: ``csrc/token_logprobs.cu``, CPU: the oracle in
``ref/logprob.py``)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ..ref import logprob as _ref
from . import logprob_cuda
from .kv8 import FLOAT_TYPES

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                   # fp32 [T]
    entropy: torch.Tensor                   # fp32 [T]
    top_logprobs: Optional[torch.Tensor]    # fp32 [T, top_k]
    top_ids: Optional[torch.Tensor]         # int64 [T, top_k]


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, top_k):
        lp, ent, stat, top, top_ids = logprob_cuda.forward(logits, ids, top_k, True, logits.get_device())
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
        logits, ids, stat, ent = ctx.saved_tensors
        return logprob_cuda.backward(logits, ids, stat, ent, g_lp, g_ent), None, None


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Scores of the tokens ``ids`` [T] int64 under ``logits`` [T, V] (bf16, fp16 or fp32; statistics in fp32).

    ``logprob[t]`` = log softmax(logits[t])[ids[t]], and 0 where the id is outside the vocabulary (the -100 of packed batches);
    ``entropy[t]`` = -sum p log p in nats; with ``top_k`` (at most 32) the largest log probabilities and their tokens, descending, the
    lowest token first among equal ones. Impossible tokens (-inf) have log probability -inf and no share in the entropy; a row of
    -inf only has entropy 0 and no gradient; NaN or +inf in a row makes its scores NaN. ``logprob`` and ``entropy`` are
    differentiable (once) in ``logits``."""
    zs = logits.shape
    if not (len(zs) == 2 and zs[1] > 0 and logits.dtype in FLOAT_TYPES):
        raise ValueError("logits: bf16, fp16 or fp32 [tokens, vocabulary]")
    if not (ids.dtype == torch.int64 and ids.shape == zs[:1]):
        raise ValueError("ids: int64 [tokens]")
    dev = logits.get_device()
    if ids.get_device() != dev:
        raise ValueError(f"tensors on {logits.device} and {ids.device}")
    if not 0 <= top_k <= min(MAX_TOP, zs[1]):
        raise ValueError(f"top_k {top_k}: 0 .. {min(MAX_TOP, zs[1])}")
    if dev < 0:
        return TokenLogprobs(*_ref.token_logprobs(logits, ids, top_k))
    if zs[1] > logprob_cuda.MAX_VOCAB:
        raise ValueError(f"vocabulary {zs[1]}: at most {logprob_cuda.MAX_VOCAB}")
    if logits.requires_grad and torch.is_grad_enabled():
        got = _TokenLogprobs.apply(logits, ids, top_k)
        return TokenLogprobs(*got) if top_k else TokenLogprobs(got[0], got[1], None, None)
    lp, ent, _, top, top_ids = logprob_cuda.forward(logits, ids, top_k, False, dev)
    return TokenLogprobs(lp, ent, top, top_ids)
