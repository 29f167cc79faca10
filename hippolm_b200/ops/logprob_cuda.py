"""CUDA path of the per-token scores (``csrc/token_logprobs.cu``). Arguments are checked in ``ops/logprob.py``."""
from __future__ import annotations

import torch

from ._ext import check, stream_ptr
from .kv8_cuda import _DTYPE, _I, _L, _P, entry, on

MAX_VOCAB = 523_776                                     # 1023 segments of 512 logits


def check_vocab(V: int) -> None:
    if V > MAX_VOCAB:
        raise ValueError(f"vocabulary {V}: at most {MAX_VOCAB}")


def forward(logits, ids, top_k: int):
    T, V = logits.shape
    z = logits if logits.stride(1) == 1 or V == 1 else logits.contiguous()
    ids = ids.contiguous()
    d = z.device
    lp, ent = (torch.empty(T, dtype=torch.float32, device=d) for _ in range(2))
    stat = torch.empty((T, 2), dtype=torch.float32, device=d)                  # maximum, log of the sum behind it
    top = torch.empty((T, top_k), dtype=torch.float32, device=d) if top_k else None
    top_ids = torch.empty((T, top_k), dtype=torch.int64, device=d) if top_k else None
    fn = entry("hippo_token_logprobs", _P, _I, _L, _L, _I, _P, _I, _P, _P, _P, _P, _P, _P)
    with on(z):
        check(fn(z.data_ptr(), _DTYPE[z.dtype], z.stride(0), T, V, ids.data_ptr(), top_k, lp.data_ptr(), ent.data_ptr(),
                 stat.data_ptr(), top.data_ptr() if top_k else None, top_ids.data_ptr() if top_k else None, stream_ptr()),
              "token_logprobs")
    return lp, ent, stat, top, top_ids


def backward(logits, ids, stat, ent, g_lp, g_ent):
    T, V = logits.shape
    z = logits if logits.stride(1) == 1 or V == 1 else logits.contiguous()
    ids = ids.contiguous()
    g_lp = g_lp.float().contiguous() if g_lp is not None else None
    g_ent = g_ent.float().contiguous() if g_ent is not None else None
    dz = torch.empty((T, V), dtype=z.dtype, device=z.device)
    fn = entry("hippo_token_logprobs_grad", _P, _I, _L, _L, _I, _P, _P, _P, _P, _P, _P, _P)
    with on(z):
        check(fn(z.data_ptr(), _DTYPE[z.dtype], z.stride(0), T, V, ids.data_ptr(), stat.data_ptr(), ent.data_ptr(),
                 g_lp.data_ptr() if g_lp is not None else None, g_ent.data_ptr() if g_ent is not None else None, dz.data_ptr(),
                 stream_ptr()), "token_logprobs_grad")
    return dz
