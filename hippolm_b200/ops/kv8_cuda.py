"""CUDA path of the 8-bit paged key / value cache (``csrc/kv8.cu``, ``csrc/kv8_attention.cu``). Arguments are checked in ``ops/kv8.py``.

These calls run once a layer and decoding step, where the host is the bound: arguments go to the library as one packed block."""
from __future__ import annotations

import ctypes as _c
import struct as _s

import torch

from ._ext import check, lib

DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_stream = torch._C._cuda_getCurrentRawStream            # the handle of a device's current stream
_current = torch._C._cuda_getDevice                     # (the tensors of a call have initialised CUDA)
ONE_BLOCK_TOKENS = 16384
HEAD_DIMS = (64, 128)
_FNS: dict = {}
_SMS: dict = {}

_PLAN = _s.Struct("@12P2q4i")
_WRITE = _s.Struct("@6P6q6i")
_ATTEND = _s.Struct("@8P4q9if")


def launch(name: str, dev: int, block: bytes) -> None:
    """Calls entry point ``name`` with its argument block, with ``dev`` as the current device (launches need it)."""
    fn = _FNS.get(name)
    if fn is None:
        fn = getattr(lib(), "hippo_" + name)
        fn.argtypes, fn.restype = (_c.c_char_p,), _c.c_int
        _FNS[name] = fn
    if dev == _current():
        check(fn(block), name)
        return
    with torch.cuda.device(dev):
        check(fn(block), name)


def plan(table, lens, new_lens, free_list, free_count, block_size, num_tokens, release, dev: int, shape):
    N, M = shape
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    lens_out, count = torch.empty_like(lens), torch.empty_like(free_count)
    served = torch.empty(N, dtype=torch.bool, device=dev) if release is None else torch.empty_like(release)
    # prompts: the slots are laid out by a kernel of their own, which looks requests up by the ends of their tokens
    cu = torch.empty(N + 1, dtype=torch.int32, device=dev) if num_tokens > ONE_BLOCK_TOKENS else None
    launch("kv8_plan", dev, _PLAN.pack(
        table.data_ptr(), lens.data_ptr(), new_lens.data_ptr(), free_list.data_ptr(), free_count.data_ptr(),
        0 if release is None else release.data_ptr(), slots.data_ptr(), lens_out.data_ptr(), count.data_ptr(), served.data_ptr(),
        0 if cu is None else cu.data_ptr(), _stream(dev), table.stride(0), num_tokens, M, N, free_list.numel(), block_size))
    return slots, lens_out, count, served


def _rows(x: torch.Tensor) -> torch.Tensor:
    """Rows of 16-byte aligned, contiguous heads (any token and head stride that keeps them so)."""
    n = 16 // x.element_size()
    t, h, d = x.stride()
    if d != 1 or t % n or h % n or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format)                  # contiguous() would keep an unaligned start
    return x


def write(k, v, slots, codes, scales, dev: int, ks, cs, window: int = 0):
    """``window``: tokens that a block looks through, 0 by size (tests give it)."""
    T, H, D = ks
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim {D}: the CUDA cache supports 64 and 128")
    k, v = _rows(k), _rows(v)
    (kt, kh, _), (vt, vh, _) = k.stride(), v.stride()
    _, blocks, _, bs, _ = cs
    launch("kv8_write", dev, _WRITE.pack(
        k.data_ptr(), v.data_ptr(), slots.data_ptr(), codes.data_ptr(), scales.data_ptr(), _stream(dev), kt, kh, vt, vh, T, blocks,
        H, D, bs, DTYPE[k.dtype], codes.dtype != torch.int8, window))


def attention_decode(q, codes, scales, table, lens, scale: float, dev: int, qs, cs, M: int):
    N, Hq, D = qs
    _, blocks, H, bs, _ = cs
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim {D}: the CUDA cache supports 64 and 128")
    if 2 * blocks * H * bs >= 1 << 31:
        raise ValueError("the cache has 2^31 rows or more")
    q = _rows(q)
    qn, qh, _ = q.stride()
    G = Hq // H
    groups, tiles = N * H * (-(-G // 8)), -(-M * bs * D // 4096)
    if groups * (tiles + 1) >= 1 << 31:
        raise ValueError(f"{N} requests of up to {M * bs} tokens and {H} heads: 2^31 tiles of 4096 / {D} tokens or more")
    sms = _SMS.get(dev)
    if sms is None:
        sms = _SMS[dev] = torch.cuda.get_device_properties(dev).multi_processor_count
    # a warp takes tiles of 4096 / D tokens; twelve of them (eight where they need more registers) fill a multiprocessor
    workers = 4 * min((2 if D == 128 or G > 4 else 3) * sms, -(-(groups * tiles) // 4))
    ws = torch.empty(workers * (2 * min(G, 8) * (D + 2) + 4), dtype=torch.float32, device=dev)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    launch("kv8_attention", dev, _ATTEND.pack(
        q.data_ptr(), out.data_ptr(), codes.data_ptr(), scales.data_ptr(), table.data_ptr(), lens.data_ptr(), ws.data_ptr(),
        _stream(dev), qn, qh, table.stride(0), blocks, N, H, Hq, D, bs, M, DTYPE[q.dtype], codes.dtype != torch.int8, workers, scale))
    return out
