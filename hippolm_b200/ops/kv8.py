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
from . import kv8_cuda

BLOCK_SIZES = (16, 32, 64)
CODE_TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOAT_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_CODES = frozenset(CODE_TYPES.values())


class KV8Plan(NamedTuple):
    slots: torch.Tensor         # int64 [num_tokens]
    lens: torch.Tensor          # int32 [requests]: lengths with the new tokens
    free_count: torch.Tensor    # int32 [1]: blocks left in the free list
    served: torch.Tensor        # bool [requests]: whether the request's new tokens have slots


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def kv8_empty(blocks: int, heads: int, head_dim: int, block_size: int = 64, dtype="e4m3", device=None
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of an empty cache. ``dtype``: "e4m3" (relative steps: keys or values of very different sizes in one block)
    or "int8" (even steps: about a third of e4m3's error on values of one size)."""
    dt = CODE_TYPES.get(dtype, dtype)
    _need(dt in CODE_TYPES.values(), f"cache dtype {dtype}: int8 or e4m3")
    _need(block_size in BLOCK_SIZES, f"block_size {block_size}: one of {BLOCK_SIZES}")
    codes = torch.zeros((2, blocks, heads, block_size, head_dim), dtype=torch.int8, device=device).view(dt)
    return codes, torch.ones((2, blocks, heads), dtype=torch.float32, device=device)


# The operators check their arguments in one expression and call these only to say what is wrong: a decoding step makes these
# calls for every layer, and its time is the host's.
def _cache_ok(codes, c, scales) -> bool:
    return (len(c) == 5 and c[0] == 2 and c[1] > 0 and c[2] > 0 and c[3] in BLOCK_SIZES and codes.dtype in _CODES
            and codes.is_contiguous() and codes.data_ptr() % 16 == 0 and scales.dtype == torch.float32 and scales.is_contiguous()
            and scales.shape == c[:3])


def _refuse_cache(codes, scales) -> None:
    _need(codes.dim() == 5 and codes.shape[0] == 2 and codes.is_contiguous() and codes.dtype in CODE_TYPES.values(),
          "codes: contiguous int8 or float8_e4m3fn [2, blocks, heads, block_size, head_dim]")
    _need(scales.dtype == torch.float32 and scales.is_contiguous() and scales.shape == codes.shape[:3],
          "scales: contiguous float32 [2, blocks, heads]")
    _need(codes.shape[3] in BLOCK_SIZES, f"block_size {codes.shape[3]}: one of {BLOCK_SIZES}")
    _need(codes.shape[1] > 0 and codes.shape[2] > 0, "an empty cache")
    _need(codes.data_ptr() % 16 == 0, "codes: a start on 16 bytes")


def _refuse_table(table, lens) -> None:
    _need(table.dim() == 2 and table.dtype == torch.int32 and table.stride(1) == 1 and table.shape[1] > 0,
          "table: int32 [requests, width > 0], unit stride along the width")
    _need(lens.dtype == torch.int32 and lens.is_contiguous() and lens.shape == table.shape[:1], "lens: contiguous int32 [requests]")


def _refuse_devices(*tensors) -> None:
    raise ValueError("tensors on different devices: " + ", ".join(str(t.device) for t in tensors))


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
    ts, ls = table.shape, lens.shape
    if not (len(ts) == 2 and ts[1] > 0 and table.dtype == lens.dtype == new_lens.dtype == free_list.dtype == free_count.dtype == torch.int32
            and ls == ts[:1] == new_lens.shape and lens.is_contiguous() and new_lens.is_contiguous() and table.stride(1) == 1
            and (ts[0] <= 1 or table.stride(0) >= ts[1]) and free_list.is_contiguous() and free_list.dim() == 1
            and free_list.numel() > 0 and free_count.numel() == 1 and block_size in BLOCK_SIZES and 0 <= num_tokens < 1 << 31
            and ts[1] * block_size < 1 << 31
            and (release is None or (release.dtype == torch.bool and release.is_contiguous() and release.shape == ls))):
        _refuse_table(table, lens)
        _need(table.shape[0] <= 1 or table.stride(0) >= table.shape[1], "table: rows that do not overlap")
        _need(new_lens.dtype == torch.int32 and new_lens.is_contiguous() and new_lens.shape == lens.shape,
              "new_lens: contiguous int32 [requests]")
        _need(free_list.dim() == 1 and free_list.dtype == torch.int32 and free_list.is_contiguous() and free_list.numel() > 0,
              "free_list: contiguous int32 [capacity > 0]")
        _need(free_count.dtype == torch.int32 and free_count.numel() == 1, "free_count: int32 [1]")
        _need(block_size in BLOCK_SIZES, f"block_size {block_size}: one of {BLOCK_SIZES}")
        _need(0 <= num_tokens < 1 << 31, "num_tokens: 0 .. 2^31 - 1")
        _need(table.shape[1] * block_size < 1 << 31, "table: at most 2^31 - 1 tokens a row")
        _need(False, "release: contiguous bool [requests]")
    dev = table.get_device()
    if not (dev == lens.get_device() == new_lens.get_device() == free_list.get_device() == free_count.get_device()) or (
            release is not None and release.get_device() != dev):
        _refuse_devices(table, lens, new_lens, free_list, free_count, *([] if release is None else [release]))
    if ts[0] == 0:
        d = table.device
        return KV8Plan(torch.full((num_tokens,), -1, dtype=torch.int64, device=d), lens.clone(), free_count.clone(),
                       torch.empty(0, dtype=torch.bool, device=d))
    if dev >= 0:
        return KV8Plan._make(kv8_cuda.plan(table, lens, new_lens, free_list, free_count, block_size, num_tokens, release, dev, ts))
    return KV8Plan(*_ref.kv8_plan(table, lens, new_lens, free_list, free_count, block_size, num_tokens, release))


def kv8_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> None:
    """Stores the keys and values [tokens, heads, head_dim] of new tokens at their ``slots``, in place.

    The scale of a (block, head) is the smallest power of two under which its largest value fits the codes. A token at offset o > 0
    of a block joins the o tokens before it: where the new tokens need a larger scale, the older codes are rounded to it. Tokens of
    one block stand next to each other, at ascending slots without gaps (as ``kv8_plan`` lays them out), and no slot appears twice.
    Slots outside the cache are skipped. A key or value that is not finite makes the scale of its (block, head) NaN, so that what
    attends to it is NaN. Not differentiable (the cache belongs to inference)."""
    ks, c = k.shape, codes.shape
    if not (_cache_ok(codes, c, scales) and len(ks) == 3 and ks == v.shape and k.dtype == v.dtype and k.dtype in FLOAT_TYPES
            and ks[1] == c[2] and ks[2] == c[4] and slots.dtype == torch.int64 and slots.is_contiguous() and slots.shape == ks[:1]):
        _refuse_cache(codes, scales)
        _need(k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype and k.dtype in FLOAT_TYPES,
              "k, v: [tokens, heads, head_dim], both bf16, fp16 or fp32")
        _need(ks[1] == c[2] and ks[2] == c[4], "k, v and codes: heads and head_dim differ")
        _need(False, "slots: contiguous int64 [tokens]")
    dev = codes.get_device()
    if not (dev == scales.get_device() == k.get_device() == v.get_device() == slots.get_device()):
        _refuse_devices(codes, scales, k, v, slots)
    if ks[0] == 0:
        return
    if dev >= 0:
        kv8_cuda.write(k, v, slots, codes, scales, dev, ks, c)
    else:
        with torch.no_grad():
            _ref.kv8_write(k, v, slots, codes, scales)


def attention_decode_kv8(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One query token per request against its ``lens[n]`` cached tokens (its own included): q [requests, q heads, head_dim] (bf16,
    fp16 or fp32) -> the same shape and type, contiguous. Query head i reads kv head i // (q heads / kv heads). A request without
    tokens gives zeros; bytes behind the last token are not looked at; a block outside the cache counts as not there. ``scale``
    defaults to head_dim ** -0.5. Inference only (no gradient)."""
    qs, c, ts = q.shape, codes.shape, table.shape
    if not (_cache_ok(codes, c, scales) and len(qs) == 3 and len(ts) == 2 and q.dtype in FLOAT_TYPES and qs[0] == ts[0] and ts[1] > 0
            and table.dtype == lens.dtype == torch.int32 and table.stride(1) == 1 and lens.is_contiguous() and lens.shape == ts[:1]
            and qs[2] == c[4] and qs[1] > 0 and qs[1] % c[2] == 0 and ts[1] * c[3] < 1 << 31):
        _refuse_cache(codes, scales)
        _refuse_table(table, lens)
        _need(q.dim() == 3 and q.dtype in FLOAT_TYPES, "q: bf16, fp16 or fp32 [requests, heads, head_dim]")
        _need(qs[0] == table.shape[0] and qs[2] == c[4], "q, table and codes: requests or head_dim differ")
        _need(qs[1] > 0 and qs[1] % c[2] == 0, "q heads: a multiple of the kv heads")
        _need(False, "table: at most 2^31 - 1 tokens a row")
    dev = codes.get_device()
    if not (dev == scales.get_device() == q.get_device() == table.get_device() == lens.get_device()):
        _refuse_devices(codes, scales, q, table, lens)
    if scale is None:
        scale = qs[2] ** -0.5
    if qs[0] == 0:
        return torch.empty_like(q)
    if dev >= 0:
        return kv8_cuda.attention_decode(q, codes, scales, table, lens, scale, dev, qs, c, ts[1])
    with torch.no_grad():
        return _ref.attention_decode_kv8(q, codes, scales, table, lens, scale)
