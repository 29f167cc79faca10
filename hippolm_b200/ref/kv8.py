"""Pure-PyTorch oracles of the 8-bit paged key / value cache (CPU execution path + test references).

A cache is ``codes`` [2, blocks, kv heads, block size, head dim] (int8 or float8_e4m3fn; keys, then values) and ``scales``
[2, blocks, kv heads] fp32; a cached value is code * scale. Scales are powers of two: a scaled value is rounded once, and where a
block's scale grows its older codes are only shifted (exact in e4m3 above the subnormal range). A scale of NaN marks a block and
head that took a key or value that is not finite. The reference has no cache (``src/models/model.py:180-219`` re-runs the forward).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

MIN_EXP = -100      # exponent of the scale of a block whose values are all zero (or below 2^-100 of the largest code)


def pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32, exactly, for integer -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def scale_exponent(amax: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Smallest e >= MIN_EXP with amax <= largest code * 2^e (448 = 0.875 * 2^9 for e4m3, 127 = 0.9921875 * 2^7 for int8)."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).int() if dtype == torch.float8_e4m3fn else x - 7 + (m > 0.9921875).int()
    return torch.where(amax > 0, e.clamp(min=MIN_EXP), MIN_EXP)


def encode(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """fp32 values within the range of the codes -> codes, rounded to nearest, ties to even."""
    return x.to(dtype) if dtype == torch.float8_e4m3fn else torch.round(x).to(torch.int8)


def kv8_plan(table, lens, new_lens, free_list, free_count, block_size: int, num_tokens: int, release=None):
    N, M = table.shape
    cap = free_list.numel()
    count = min(max(int(free_count), 0), cap)
    old = [min(max(x, 0), M * block_size) for x in lens.tolist()]
    new = [max(x, 0) for x in new_lens.tolist()]
    gone = [bool(x) for x in release.tolist()] if release is not None else [False] * N
    up = lambda a: -(-a // block_size)                                              # noqa: E731
    for n in range(N):
        if gone[n]:
            for j in range(up(old[n])):
                if count < cap:
                    free_list[count] = table[n, j]
                    count += 1
            old[n] = 0
    slots = torch.full((num_tokens,), -1, dtype=torch.int64)
    served, out, cu, top, used = [], [], [0], 0, 0
    for n in range(N):
        start = cu[-1]
        cu.append(start + new[n])
        fits = not gone[n] and old[n] + new[n] <= M * block_size and cu[-1] <= num_tokens
        need = up(old[n] + new[n]) - up(old[n]) if fits else 0
        top += need
        ok = new[n] == 0 or (fits and (need == 0 or top <= count))
        served.append(ok)
        out.append(old[n] + new[n] if ok else old[n])
        if not ok or new[n] == 0:
            continue
        for j in range(need):
            table[n, up(old[n]) + j] = free_list[count - 1 - (top - need) - j]
        used += need
        for i in range(new[n]):
            p = old[n] + i
            b = int(table[n, p // block_size])
            slots[start + i] = b * block_size + p % block_size if b >= 0 else -1
    i32 = dict(dtype=torch.int32)
    return slots, torch.tensor(out, **i32), torch.tensor([count - used], **i32), torch.tensor(served, dtype=torch.bool)


def _write_run(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, off: int) -> None:
    """x [L, H, D] at offsets off .. off + L - 1 of one block: codes [H, bs, D], scales [H]."""
    xf = x.float()
    amax = xf.abs().amax((0, 2))
    e = scale_exponent(torch.nan_to_num(amax, nan=0.0, posinf=0.0), codes.dtype)
    bad = ~torch.isfinite(amax)
    if off > 0:
        bad = bad | torch.isnan(scales)
        e_old = torch.frexp(torch.nan_to_num(scales, nan=1.0))[1] - 1
        e_old = torch.where(bad, 0, e_old).clamp(MIN_EXP, 127)
        e = torch.maximum(e, e_old)
        down = torch.where(bad, 0, e_old - e).clamp(min=-126)
        kept = encode(codes[:, :off].float() * pow2(down)[:, None, None], codes.dtype)
        codes[:, :off] = torch.where(bad[:, None, None], codes[:, :off].float(), kept.float()).to(codes.dtype)
    val = encode(torch.where(bad[None, :, None], 0.0, xf * pow2(-e)[None, :, None]), codes.dtype)
    codes[:, off:off + x.shape[0]] = val.transpose(0, 1)
    scales.copy_(torch.where(bad, float("nan"), pow2(e)))


def kv8_write(k, v, slots, codes, scales) -> None:
    _, blocks, H, bs, D = codes.shape
    sl = slots.tolist()
    t = 0
    while t < len(sl):
        s = sl[t]
        if s < 0 or s >= blocks * bs:
            t += 1
            continue
        L = 1
        while t + L < len(sl) and sl[t + L] == s + L and (s + L) % bs:
            L += 1
        for i, x in enumerate((k, v)):
            _write_run(x[t:t + L], codes[i, s // bs], scales[i, s // bs], s % bs)
        t += L


def gather(codes, scales, blocks: torch.Tensor, length: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [length, H, D] (fp32) of the tokens held by ``blocks`` in order; a block outside the pool gives NaN rows,
    which the callers mask."""
    got = []
    ok = (blocks >= 0) & (blocks < codes.shape[1])
    at = blocks.clamp(0, codes.shape[1] - 1).long()
    for i in range(2):
        x = codes[i].view(torch.int8)[at].view(codes.dtype).float() * scales[i][at][..., None, None]     # [B, H, bs, D]
        x = torch.where(ok[:, None, None, None], x, float("nan"))
        got.append(x.transpose(1, 2).reshape(-1, codes.shape[2], codes.shape[4])[:length])
    return got[0], got[1]


def attention_decode_kv8(q, codes, scales, table, lens, scale: Optional[float] = None) -> torch.Tensor:
    N, Hq, D = q.shape
    _, nb, H, bs, _ = codes.shape
    if scale is None:
        scale = D ** -0.5
    out = torch.zeros((N, Hq, D), dtype=torch.float32, device=q.device)
    for n in range(N):
        length = min(max(int(lens[n]), 0), table.shape[1] * bs)
        if length == 0:
            continue
        row = table[n, :-(-length // bs)]
        k, v = gather(codes, scales, row, length)
        there = ((row >= 0) & (row < nb)).repeat_interleave(bs)[:length]            # tokens of a bad block are not attended to
        if not bool(there.any()):
            continue
        k, v = k[there].repeat_interleave(Hq // H, 1), v[there].repeat_interleave(Hq // H, 1)
        p = torch.softmax(torch.einsum("hd,lhd->hl", q[n].float(), k) * scale, -1)
        out[n] = torch.einsum("hl,lhd->hd", p, v)
    return out.to(q.dtype)
