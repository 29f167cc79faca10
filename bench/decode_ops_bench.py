#!/usr/bin/env python
"""Device time of the operators of a decoding step over the 8-bit paged cache (plan, quantising write, attention) and of the
per-token scores. ``--only PART`` runs the lines whose name contains PART, ``--iters N`` timed iterations of each (0: one call)."""
import argparse
import json

import torch

from common import time_ms
from hippolm_b200 import ops


def cache(N, lens, H, D, bs, kind):
    need = [-(-x // bs) for x in lens]
    blocks = sum(need) + 1
    codes, scales = ops.kv8_empty(blocks, H, D, bs, kind, "cuda")
    codes.view(torch.int8).random_(-100, 100)
    scales.fill_(2.0 ** -6)
    perm = torch.randperm(blocks, device="cuda").to(torch.int32)
    table, at = torch.full((N, max(need)), -1, dtype=torch.int32, device="cuda"), 0
    for n, c in enumerate(need):
        table[n, :c] = perm[at:at + c]
        at += c
    return codes, scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def attention(N, L, Hq, H, D, bs, kind):
    codes, scales, table, lens = cache(N, [L] * N, H, D, bs, kind)
    q = torch.randn(N, Hq, D, device="cuda").bfloat16()
    return (f"attention {N} x {L}, {Hq} / {H} heads of {D}, blocks of {bs}, {kind}",
            lambda: ops.attention_decode_kv8(q, codes, scales, table, lens), 2 * N * L * H * D)


def write(N, L, H, D, bs, kind):
    codes, scales, table, _ = cache(N, [L] * N, H, D, bs, kind)
    k, v = (torch.randn(N * L, H, D, device="cuda").bfloat16() for _ in range(2))
    pos = torch.arange(L, device="cuda")
    slots = (table.long()[:, pos // bs] * bs + pos % bs).reshape(-1)
    return f"write {N} x {L}, {H} heads of {D}, blocks of {bs}, {kind}", lambda: ops.kv8_write(k, v, slots, codes, scales), 6 * N * L * H * D


def plan(N, L, bs):
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, new = torch.full((N, -(-2 * L // bs)), -1, **i32), torch.zeros(N, **i32), torch.full((N,), L, **i32)
    free = torch.arange(N * -(-2 * L // bs), **i32)
    count = torch.full((1,), free.numel(), **i32)
    return f"plan {N} x {L} new tokens, blocks of {bs}", lambda: ops.kv8_plan(table, lens, new, free, count, bs, N * L), 8 * N * L


def scores(T, V, top, dt):
    z, ids = (torch.randn(T, V, device="cuda") * 2).to(dt), torch.randint(0, V, (T,), device="cuda")
    return f"scores {T} x {V} {str(dt)[6:]}, {top} alternatives", lambda: ops.token_logprobs(z, ids, top_k=top), z.numel() * z.element_size()


def score_gradient(T, V, dt):
    z, ids = (torch.randn(T, V, device="cuda") * 2).to(dt).requires_grad_(True), torch.randint(0, V, (T,), device="cuda")
    g = torch.randn(T, device="cuda")
    got = ops.token_logprobs(z, ids)
    return (f"score gradient {T} x {V} {str(dt)[6:]}",
            lambda: torch.autograd.grad((got.logprob, got.entropy), z, (g, g), retain_graph=True), 2 * z.numel() * z.element_size())


CASES = [(plan, 16, 1, 64), (plan, 64, 7600, 64), (write, 32, 1, 32, 128, 64, "e4m3"), (write, 24, 1040, 16, 128, 32, "e4m3"),
         (attention, 1, 500, 16, 16, 128, 16, "e4m3"), (attention, 8, 4096, 32, 32, 128, 64, "e4m3"),
         (attention, 8, 4096, 32, 32, 128, 64, "int8"), (attention, 16, 4096, 32, 32, 64, 64, "int8"),
         (attention, 16, 4096, 64, 8, 128, 64, "e4m3"), (attention, 2, 131072, 4, 4, 128, 64, "int8"),
         (attention, 32, 7000, 32, 32, 128, 64, "e4m3"), (scores, 8, 128256, 5, torch.bfloat16),
         (scores, 2048, 128256, 0, torch.bfloat16), (scores, 2048, 128256, 20, torch.bfloat16), (scores, 3001, 32000, 0, torch.float32),
         (score_gradient, 3001, 32000, torch.float32)]


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--only", default=""); ap.add_argument("--iters", type=int, default=10)
    a = ap.parse_args()
    for make, *args in CASES:
        name, fn, nbytes = make(*args)
        if a.only not in name:
            continue
        if a.iters == 0:
            fn()
            torch.cuda.synchronize()
            continue
        us = time_ms(fn, iters=a.iters) * 1e3
        print(json.dumps({"case": name, "us": round(us, 2), "gb_s": round(nbytes / us / 1e3, 1)}), flush=True)


if __name__ == "__main__":
    main()
