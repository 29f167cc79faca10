"""CUDA path of the per-token scores (``csrc/token_logprobs.cu``). Arguments are checked in ``ops/logprob.py``."""
from __future__ import annotations

import struct as _s

import torch

from .kv8_cuda import DTYPE, _stream, launch

MAX_VOCAB = 523_776                                     # 1023 segments of 512 logits
_FWD = _s.Struct("@8P2q3i")
_BWD = _s.Struct("@8P2q2i")


def _rows(z: torch.Tensor) -> torch.Tensor:
    return z if z.stride(1) == 1 or z.shape[1] == 1 else z.contiguous()


def forward(logits, ids, top_k: int, keep: bool, dev: int):
    """``keep``: also the statistics (maximum, log of the sum behind it) that the backward pass reads."""
    T, V = logits.shape
    z, ids, d = _rows(logits), ids.contiguous(), dev
    lp = torch.empty(T, dtype=torch.float32, device=d)
    ent = torch.empty_like(lp)
    stat = torch.empty((T, 2), dtype=torch.float32, device=d) if keep else None
    top, top_ids = (lp.new_empty((T, top_k)), ids.new_empty((T, top_k))) if top_k else (None, None)
    launch("token_logprobs", dev, _FWD.pack(
        z.data_ptr(), ids.data_ptr(), lp.data_ptr(), ent.data_ptr(), stat.data_ptr() if keep else 0, top.data_ptr() if top_k else 0,
        top_ids.data_ptr() if top_k else 0, _stream(dev), z.stride(0), T, V, top_k, DTYPE[z.dtype]))
    return lp, ent, stat, top, top_ids


def backward(logits, ids, stat, ent, g_lp, g_ent):
    T, V = logits.shape
    z, ids, dev = _rows(logits), ids.contiguous(), logits.get_device()
    g_lp = g_lp.float().contiguous() if g_lp is not None else None
    g_ent = g_ent.float().contiguous() if g_ent is not None else None
    dz = torch.empty((T, V), dtype=z.dtype, device=z.device)
    launch("token_logprobs_grad", dev, _BWD.pack(
        z.data_ptr(), ids.data_ptr(), stat.data_ptr(), ent.data_ptr(), 0 if g_lp is None else g_lp.data_ptr(),
        0 if g_ent is None else g_ent.data_ptr(), dz.data_ptr(), _stream(dev), z.stride(0), T, V, DTYPE[z.dtype]))
    return dz
