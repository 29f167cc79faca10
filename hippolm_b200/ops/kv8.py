"""The 8-bit paged key / value cache of incremental decoding: planning, the quantising write, and attention over it.

Tensors (all on one device; CUDA tensors run ``csrc/kv8.cu`` / ``csrc/kv8_attention.cu``, CPU tensors the oracle in ``ref/kv8.py``):

* ``codes`` [2, blocks, kv heads, block size, head dim], int8 or float8_e4m3fn, contiguous: keys, then values;
* ``scales`` [2, blocks, kv heads] fp32, powers of two: a cached value is code * scale of its (block, head);
* ``table`` [requests, width] int32: row n lists the blocks of request n in the order of its tokens;
* ``lens`` [requests] int32: tokens cached;
* ``slots`` [tokens] int64: block * block size + offset of every new token, -1 where it is not stored.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ..ref import kv8 as _ref

BLOCK_SIZES = (16, 32, 64)
CODE_TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOAT_TYPES = (torch.bfloat16, torch.float16, torch.float32)


class KV8Plan(NamedTuple):
    slots: torch.Tensor         # int64 [num_tokens]
    lens: torch.Tensor          # int32 [requests]: lengths with the new tokens
    free_count: torch.Tensor    # int32 [1]: blocks left in the free list
    served: torch.Tensor        # bool [requests]: whether the request's new tokens have slots
    cu_seqlens: torch.Tensor    # int32 [requests + 1]: ends of the requests' new tokens in the packed stream


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _same_device(first: torch.Tensor, *rest: torch.Tensor) -> None:
    for t in rest:
        if t.device != first.device:
            raise ValueError(f"tensors on {first.device} and {t.device}")


def kv8_empty(blocks: int, heads: int, head_dim: int, block_size: int = 64, dtype="e4m3", device=None
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of an empty cache. ``dtype``: "e4m3" (relative steps: keys or values of very different sizes in one block)
    or "int8" (even steps: about a third of e4m3's error on values of one size)."""
    dt = CODE_TYPES.get(dtype, dtype)
    _need(dt in CODE_TYPES.values(), f"cache dtype {dtype}: int8 or e4m3")
    _need(block_size in BLOCK_SIZES, f"block_size {block_size}: one of {BLOCK_SIZES}")
    codes = torch.zeros((2, blocks, heads, block_size, head_dim), dtype=torch.int8, device=device).view(dt)
    return codes, torch.ones((2, blocks, heads), dtype=torch.float32, device=device)


def _check_cache(codes: torch.Tensor, scales: torch.Tensor) -> None:
    _need(codes.dim() == 5 and codes.shape[0] == 2 and codes.is_contiguous() and codes.dtype in CODE_TYPES.values(),
          "codes: contiguous int8 or float8_e4m3fn [2, blocks, heads, block_size, head_dim]")
    _need(scales.dtype == torch.float32 and scales.is_contiguous() and scales.shape == codes.shape[:3],
          "scales: contiguous float32 [2, blocks, heads]")
    _need(codes.shape[3] in BLOCK_SIZES, f"block_size {codes.shape[3]}: one of {BLOCK_SIZES}")
    _need(codes.shape[1] > 0 and codes.shape[2] > 0, "an empty cache")
    _need(codes.data_ptr() % 16 == 0, "codes: a start on 16 bytes")


def _check_table(table: torch.Tensor, lens: torch.Tensor) -> None:
    _need(table.dim() == 2 and table.dtype == torch.int32 and table.stride(1) == 1 and table.shape[1] > 0,
          "table: int32 [requests, width > 0], unit stride along the width")
    _need(lens.dtype == torch.int32 and lens.is_contiguous() and lens.shape == table.shape[:1], "lens: contiguous int32 [requests]")


def kv8_plan(table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor, free_list: torch.Tensor, free_count: torch.Tensor,
             block_size: int, num_tokens: int, release: Optional[torch.Tensor] = None) -> KV8Plan:
    """Blocks and slots for the new tokens of a step, without a host read: ``new_lens[n]`` tokens of request n, packed in request order
    into ``num_tokens`` rows.

    ``free_list`` [capacity] int32 is a stack of free blocks, of which the first ``free_count`` entries count. Requests with
    ``release[n]`` (bool) push their blocks back first, in order, and start at length 0; they take no tokens in the same call. Then
    every request pops, in order, the blocks its new tokens need beyond those it has. A request is served (all its tokens, or none)
    if the table is wide enough, its tokens lie within ``num_tokens`` and its blocks are there; the blocks that a request asks for
    but cannot get also stay unavailable to the ones behind it. Tokens of requests that are not served, and rows behind the last
    token, have slot -1.

    ``table`` gets the new blocks and ``free_list`` the released ones, in place; lengths and the stack's height are returned new
    (``plan.lens``, ``plan.free_count``), so a repeated call with the same lengths gives the same plan. Lengths below 0 count as 0,
    lengths beyond the table's width as the width."""
    _check_table(table, lens)
    _need(table.shape[0] <= 1 or table.stride(0) >= table.shape[1], "table: rows that do not overlap")
    _need(new_lens.dtype == torch.int32 and new_lens.is_contiguous() and new_lens.shape == lens.shape,
          "new_lens: contiguous int32 [requests]")
    _need(free_list.dim() == 1 and free_list.dtype == torch.int32 and free_list.is_contiguous() and free_list.numel() > 0,
          "free_list: contiguous int32 [capacity > 0]")
    _need(free_count.dtype == torch.int32 and free_count.numel() == 1, "free_count: int32 [1]")
    _need(block_size in BLOCK_SIZES, f"block_size {block_size}: one of {BLOCK_SIZES}")
    _need(0 <= num_tokens < 1 << 31, "num_tokens: 0 .. 2^31 - 1")
    _need(table.shape[1] * block_size < 1 << 31, "table: at most 2^31 - 1 tokens a row")
    _same_device(table, lens, new_lens, free_list, free_count)
    if release is not None:
        _need(release.dtype == torch.bool and release.is_contiguous() and release.shape == lens.shape,
              "release: contiguous bool [requests]")
        _same_device(table, release)
    if table.shape[0] == 0:
        d = table.device
        return KV8Plan(torch.full((num_tokens,), -1, dtype=torch.int64, device=d), lens.clone(), free_count.reshape(1).clone(),
                       torch.empty(0, dtype=torch.bool, device=d), torch.zeros(1, dtype=torch.int32, device=d))
    if table.is_cuda:
        from . import kv8_cuda
        return KV8Plan(*kv8_cuda.plan(table, lens, new_lens, free_list, free_count, block_size, num_tokens, release))
    return KV8Plan(*_ref.kv8_plan(table, lens, new_lens, free_list, free_count, block_size, num_tokens, release))


@torch.no_grad()
def kv8_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> None:
    """Stores the keys and values [tokens, heads, head_dim] of new tokens at their ``slots``, in place.

    The scale of a (block, head) is the smallest power of two under which its largest value fits the codes. A token at offset o > 0
    of a block joins the o tokens before it: where the new tokens need a larger scale, the older codes are rounded to it. Tokens of
    one block stand next to each other, at ascending slots without gaps (as ``kv8_plan`` lays them out), and no slot appears twice.
    Slots outside the cache are skipped. A key or value that is not finite makes the scale of its (block, head) NaN, so that what
    attends to it is NaN. Not differentiable (the cache belongs to inference)."""
    _check_cache(codes, scales)
    _need(k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype and k.dtype in FLOAT_TYPES,
          "k, v: [tokens, heads, head_dim], both bf16, fp16 or fp32")
    _need(k.shape[1] == codes.shape[2] and k.shape[2] == codes.shape[4], "k, v and codes: heads and head_dim differ")
    _need(slots.dtype == torch.int64 and slots.is_contiguous() and slots.shape == k.shape[:1], "slots: contiguous int64 [tokens]")
    _same_device(codes, scales, k, v, slots)
    if k.shape[0] == 0:
        return
    if k.is_cuda:
        from . import kv8_cuda
        kv8_cuda.write(k, v, slots, codes, scales)
    else:
        _ref.kv8_write(k, v, slots, codes, scales)


@torch.no_grad()
def attention_decode_kv8(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One query token per request against its ``lens[n]`` cached tokens (its own included): q [requests, q heads, head_dim] (bf16,
    fp16 or fp32) -> the same shape and type, contiguous. Query head i reads kv head i // (q heads / kv heads). A request without
    tokens gives zeros; bytes behind the last token are not looked at; a block outside the cache counts as not there. ``scale``
    defaults to head_dim ** -0.5. Inference only (no gradient)."""
    _check_cache(codes, scales)
    _check_table(table, lens)
    _need(q.dim() == 3 and q.dtype in FLOAT_TYPES, "q: bf16, fp16 or fp32 [requests, heads, head_dim]")
    _need(q.shape[0] == table.shape[0] and q.shape[2] == codes.shape[4], "q, table and codes: requests or head_dim differ")
    _need(q.shape[1] > 0 and q.shape[1] % codes.shape[2] == 0, "q heads: a multiple of the kv heads")
    _need(table.shape[1] * codes.shape[3] < 1 << 31, "table: at most 2^31 - 1 tokens a row")
    _same_device(codes, scales, q, table, lens)
    if scale is None:
        scale = q.shape[2] ** -0.5
    if q.shape[0] == 0:
        return torch.empty_like(q)
    if q.is_cuda:
        from . import kv8_cuda
        return kv8_cuda.attention_decode(q, codes, scales, table, lens, float(scale))
    return _ref.attention_decode_kv8(q, codes, scales, table, lens, float(scale))
