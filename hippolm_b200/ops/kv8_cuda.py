"""CUDA path of the 8-bit paged key / value cache (``csrc/kv8.cu``, ``csrc/kv8_attention.cu``). Arguments are checked in ``ops/kv8.py``."""
from __future__ import annotations

import contextlib
import ctypes as _c

import torch

from ._ext import check, lib, stream_ptr

_P, _I, _L, _F = _c.c_void_p, _c.c_int, _c.c_longlong, _c.c_float
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NO_SWITCH = contextlib.nullcontext()


def on(t: torch.Tensor):
    """Context in which launches go to ``t``'s device (its current stream), whatever the current device is."""
    return _NO_SWITCH if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


_FNS: dict = {}


def entry(name: str, *argtypes):
    """Entry point of the kernel library with its argument types set."""
    fn = _FNS.get(name)
    if fn is None:
        fn = getattr(lib(), name)
        fn.argtypes, fn.restype = argtypes, _c.c_int
        _FNS[name] = fn
    return fn


def plan(table, lens, new_lens, free_list, free_count, block_size, num_tokens, release):
    N, M = table.shape
    d = table.device
    slots = torch.empty(num_tokens, dtype=torch.int64, device=d)
    out = torch.empty(2 * N + 2, dtype=torch.int32, device=d)                  # lens [N], count [1], cu_seqlens [N + 1]
    served = torch.empty(N, dtype=torch.bool, device=d)
    fn = entry("hippo_kv8_plan", _P, _L, _I, _P, _P, _I, _P, _I, _P, _P, _I, _L, _P, _P, _P, _P, _P, _P)
    o = out.data_ptr()
    with on(table):
        check(fn(table.data_ptr(), table.stride(0), M, lens.data_ptr(), new_lens.data_ptr(), N, free_list.data_ptr(),
                 free_list.numel(), free_count.data_ptr(), release.data_ptr() if release is not None else None, block_size,
                 num_tokens, slots.data_ptr(), o, o + 4 * N, served.data_ptr(), o + 4 * N + 4, stream_ptr()), "kv8_plan")
    lens_out, count, cu = out.split((N, 1, N + 1))
    return slots, lens_out, count, served, cu


def _rows(x: torch.Tensor) -> torch.Tensor:
    """Rows of 16-byte aligned, contiguous heads (any token and head stride that keeps them so)."""
    n = 16 // x.element_size()
    if x.stride(2) != 1 or x.stride(0) % n or x.stride(1) % n or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format)                  # contiguous() would keep an unaligned start
    return x


def write(k, v, slots, codes, scales, form: int = 0):
    """``form``: 0 by size, 1 a warp for each run of tokens, 2 a block for each window of tokens (tests)."""
    T, H, D = k.shape
    if D not in (64, 128):
        raise ValueError(f"head_dim {D}: the CUDA cache supports 64 and 128")
    k, v = _rows(k), _rows(v)
    fn = entry("hippo_kv8_write", _P, _P, _I, _L, _L, _L, _L, _P, _L, _I, _I, _I, _L, _I, _P, _P, _I, _P)
    with on(k):
        check(fn(k.data_ptr(), v.data_ptr(), _DTYPE[k.dtype], k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(),
                 T, H, D, codes.shape[3], codes.shape[1], codes.dtype != torch.int8, codes.data_ptr(), scales.data_ptr(), form,
                 stream_ptr()), "kv8_write")


def attention_decode(q, codes, scales, table, lens, scale: float):
    N, Hq, D = q.shape
    _, blocks, H, bs, _ = codes.shape
    M = table.shape[1]
    if D not in (64, 128):
        raise ValueError(f"head_dim {D}: the CUDA cache supports 64 and 128")
    if 2 * blocks * H * bs >= 1 << 31:
        raise ValueError("the cache has 2^31 rows or more")
    if q.stride(2) != 1:
        q = q.contiguous()
    G = Hq // H
    with on(q):
        workers = entry("hippo_kv8_attention_workers", _L)(N * H * (-(-G // 8)) * (-(-M * bs // 32)))
        rows = min(G, 8)
        ws = torch.empty(workers * (2 * rows * (D + 2) + 4), dtype=torch.float32, device=q.device)
        out = torch.empty((N, Hq, D), dtype=q.dtype, device=q.device)
        fn = entry("hippo_kv8_attention", _P, _I, _L, _L, _P, _P, _P, _I, _L, _I, _I, _I, _I, _P, _L, _I, _P, _I, _F, _I, _P, _P)
        check(fn(q.data_ptr(), _DTYPE[q.dtype], q.stride(0), q.stride(1), out.data_ptr(), codes.data_ptr(), scales.data_ptr(),
                 codes.dtype != torch.int8, blocks, H, Hq, D, bs, table.data_ptr(), table.stride(0), M, lens.data_ptr(), N, scale,
                 workers, ws.data_ptr(), stream_ptr()), "kv8_attention")
    return out
