"""Pages of the 8-bit key / value caches of a batch that is being decoded (``ops/kv8.py``).

One block table serves all full-attention layers: block b of a request is block b of every layer's cache. The reference keeps no
cache (``src/models/model.py:180-219`` re-runs the forward for every token)."""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from .. import ops
from ..ops.kv8 import CODE_TYPES
from ..ops.kv8_cuda import HEAD_DIMS


def check_cache(dtype, head_dim: Optional[int], device) -> None:
    """Refuses a cache type that there is none of, and a head size that the device's cache does not take. ``dtype`` None: no 8-bit
    cache; ``head_dim`` None: no layer that keeps keys."""
    if dtype is None:
        return
    if dtype not in CODE_TYPES and dtype not in CODE_TYPES.values():
        raise ValueError(f"kv_cache {dtype}: int8 or e4m3")
    if torch.device(device).type == "cuda" and head_dim is not None and head_dim not in HEAD_DIMS:
        raise ValueError(f"kv_cache {dtype}: head_dim {head_dim}, the CUDA cache supports {' and '.join(map(str, HEAD_DIMS))}")


class KV8Pages:
    """Block table, lengths and free blocks of ``len(limits)`` sequences of at most ``limits[n]`` tokens each. The pool has exactly
    the blocks that they can need, so every plan is served; a sequence in ``release`` gives its blocks back and stores nothing.
    (The host keeps the lengths too, to refuse what goes beyond a limit: such a token would have no block.)"""

    def __init__(self, limits: Sequence[int], block_size: int = 64, device=None):
        need = [-(-max(x, 0) // block_size) for x in limits]
        i32 = dict(dtype=torch.int32, device=device)
        self.limits, self.block_size, self.blocks = list(limits), block_size, max(1, sum(need))
        self.table = torch.full((len(need), max([1] + need)), -1, **i32)
        self.lens = torch.zeros(len(need), **i32)
        self.free = torch.arange(self.blocks - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), self.blocks, **i32)
        self.release = None
        self.slots: Optional[torch.Tensor] = None         # of the tokens of the pass that was planned last
        self.passes = 0
        self._held = [0] * len(need)

    @property
    def release(self) -> Optional[torch.Tensor]:
        """bool [sequences], read by the next plan"""
        return self._release

    @release.setter
    def release(self, gone: Optional[torch.Tensor]) -> None:
        self._release, self._gone = gone, [False] * len(self.limits) if gone is None else gone.tolist()

    def plan(self, cu_seqlens: torch.Tensor, num_tokens: int) -> None:
        """Slots for the tokens of the next pass, ``cu_seqlens`` [sequences + 1] packed: the whole prompts first, then one token a
        sequence and pass. Sequences in ``release`` have their rows in the stream like the others."""
        if self.passes and num_tokens != self.table.shape[0]:
            raise ValueError("the cache takes whole prompts first, then one token per sequence and step")
        if cu_seqlens.numel() != len(self.limits) + 1:
            raise ValueError(f"{cu_seqlens.numel() - 1} sequences, the cache has {len(self.limits)}")
        ends = None if self.passes else cu_seqlens.tolist()
        held = []
        for n, (had, gone, limit) in enumerate(zip(self._held, self._gone, self.limits)):
            held.append(0 if gone else had + (1 if self.passes else ends[n + 1] - ends[n]))
            if held[n] > limit and not gone:
                raise ValueError(f"sequence {n}: {held[n]} tokens, its limit is {limit}")
        new = (cu_seqlens[1:] - cu_seqlens[:-1]).to(torch.int32)
        p = ops.kv8_plan(self.table, self.lens, new, self.free, self.free_count, self.block_size, num_tokens, release=self.release)
        self.slots, self.lens, self.free_count = p.slots, p.lens, p.free_count
        self.passes += 1
        self._held = held

    def attend(self, q, k, v, codes, scales, scale: float) -> Optional[torch.Tensor]:
        """Stores the pass's keys and values and, from the second pass on, returns the attention over each sequence's tokens (the
        prompts themselves attend to their unquantised keys: None)."""
        ops.kv8_write(k, v.to(k.dtype), self.slots, codes, scales)
        if self.passes == 1:
            return None
        return ops.attention_decode_kv8(q, codes, scales, self.table, self.lens, scale)


def layer_cache(pages: KV8Pages, heads: int, head_dim: int, dtype: str, device=None) -> dict:
    codes, scales = ops.kv8_empty(pages.blocks, heads, head_dim, pages.block_size, dtype, device)
    return {"pages": pages, "codes": codes, "scales": scales}


def pages_of(caches: Optional[List[dict]]) -> Optional[KV8Pages]:
    return next((c["pages"] for c in caches if "pages" in c), None) if caches is not None else None
