"""The operators of a decoding step over an 8-bit paged key / value cache, and of scoring tokens: what is measured.

A decoding step of the server plans where its new tokens go (``kv8_plan``), stores their keys and values in 8 bits
(``kv8_write``), attends over the cache (``attention_decode_kv8``) and reads log probabilities off the logits
(``token_logprobs``, which training objectives on log probabilities and entropies also differentiate).

Layouts: ``codes`` [2, blocks, kv heads, block size, head dim] (int8 or float8_e4m3fn; keys first, then values), ``scales``
[2, blocks, kv heads] fp32 powers of two, ``table`` [requests, width] int32 (row n lists the blocks of request n in order),
``lens`` [requests] int32 tokens cached, ``slots`` [tokens] int64 = block * block size + offset (-1: not stored).
A cached value is code * scale of its (block, head).
"""
import math
import random

import torch

own = False

IGNORED = -100        # a target that is not scored (padding of packed batches)
MIN_EXP = -100        # exponent of the scale of a block of zeros


# ----------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # 16 requests, one token each: what every decoding step of a small batch pays before its first layer
        {"name": "plan_decode_16", "op": "plan", "n": 16, "lo": 30, "hi": 2000, "new_lo": 1, "new_hi": 1, "bs": 64,
         "release": False},
        # a continuous batch: 300 slots of a server, some requests just ended and give their blocks back
        {"name": "plan_mixed_300", "op": "plan", "n": 300, "lo": 0, "hi": 8192, "new_lo": 0, "new_hi": 37, "bs": 16,
         "release": True},
        # packed prompts of an offline evaluation: the slots of half a million tokens
        {"name": "plan_prompts_64", "op": "plan", "n": 64, "lo": 0, "hi": 0, "new_lo": 7000, "new_hi": 8192, "bs": 64,
         "release": False},
        # one layer's keys and values of one token for each of 32 requests (32 heads of 128, the 7B hybrid)
        {"name": "write_decode_32", "op": "write", "n": 32, "lo": 1, "hi": 8000, "new_lo": 1, "new_hi": 1, "heads": 32,
         "dim": 128, "bs": 64, "codes": "e4m3", "dtype": "bf16"},
        # packed prompts of uneven lengths, a tensor-parallel shard of 16 heads
        {"name": "write_prompts_24", "op": "write", "n": 24, "lo": 0, "hi": 0, "new_lo": 17, "new_hi": 4099, "heads": 16,
         "dim": 128, "bs": 32, "codes": "e4m3", "dtype": "bf16"},
        # a single request in the middle of its answer: latency of one layer's attention
        {"name": "attend_1x500", "op": "attend", "n": 1, "lo": 500, "hi": 500, "q_heads": 16, "kv_heads": 16, "dim": 128,
         "bs": 16, "codes": "e4m3", "dtype": "bf16"},
        # one rank of eight at a long context: few heads, so the work has to be split along the sequence
        {"name": "attend_long_2x4", "op": "attend", "n": 2, "lo": 100003, "hi": 131072, "q_heads": 4, "kv_heads": 4,
         "dim": 128, "bs": 64, "codes": "int8", "dtype": "bf16"},
        # a ragged batch with shared key / value heads and heads of 64
        {"name": "attend_ragged_48", "op": "attend", "n": 48, "lo": 1, "hi": 8192, "q_heads": 32, "kv_heads": 8, "dim": 64,
         "bs": 32, "codes": "int8", "dtype": "bf16"},
        # a full batch of the 7B hybrid near its training length
        {"name": "attend_batch_32", "op": "attend", "n": 32, "lo": 6001, "hi": 8192, "q_heads": 32, "kv_heads": 32,
         "dim": 128, "bs": 64, "codes": "e4m3", "dtype": "bf16"},
        # the sampled tokens of a decoding step, with five alternatives each
        {"name": "logprob_decode_8", "op": "logprob", "rows": 8, "vocab": 128256, "top": 5, "dtype": "bf16",
         "backward": False},
        # prompt tokens of an evaluation, with the twenty alternatives a completion request may ask for
        {"name": "logprob_score_4096", "op": "logprob", "rows": 4096, "vocab": 128256, "top": 20, "dtype": "bf16",
         "backward": False},
        # a training objective on log probabilities with an entropy term, small vocabulary, fp32 logits
        {"name": "logprob_train_3001", "op": "logprob", "rows": 3001, "vocab": 32000, "top": 0, "dtype": "fp32",
         "backward": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "logprob", "logprob"])
    bs = rng.choice([16, 32, 64])
    if op == "plan":
        n = _log_int(rng, 1, 512)
        if rng.random() < 0.5:
            return {"op": op, "n": n, "lo": 0, "hi": _log_int(rng, 1, 8192), "new_lo": 0, "new_hi": rng.choice([1, 1, 5, 40]),
                    "bs": bs, "release": rng.random() < 0.5}
        top = _log_int(rng, 1, min(8192, (1 << 19) // n))
        return {"op": op, "n": n, "lo": 0, "hi": rng.choice([0, 100]), "new_lo": max(1, top // 4), "new_hi": top, "bs": bs,
                "release": False}
    codes, dtype = rng.choice(["e4m3", "int8"]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = rng.choice([64, 128])
    if op == "write":
        heads = rng.choice([1, 4, 8, 16, 32])
        if rng.random() < 0.5:
            return {"op": op, "n": _log_int(rng, 1, 256), "lo": 0, "hi": _log_int(rng, 1, 2048), "new_lo": 1, "new_hi": 1,
                    "heads": heads, "dim": dim, "bs": bs, "codes": codes, "dtype": dtype}
        n = _log_int(rng, 1, 32)
        top = _log_int(rng, 2, max(2, 40000 * 16 // (n * heads)))
        top = min(top, 8192)
        return {"op": op, "n": n, "lo": 0, "hi": rng.choice([0, 77]), "new_lo": 1, "new_hi": top, "heads": heads, "dim": dim,
                "bs": bs, "codes": codes, "dtype": dtype}
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8, 16, 32])
        q = kv * rng.choice([1, 1, 1, 2, 4, 8, 12])
        n = _log_int(rng, 1, 128)
        most = max(2, min(131072, (32 * 32 * 8192 // 2) // (n * kv)))
        hi = _log_int(rng, 1, most)
        if dtype == "fp32":
            dtype = "bf16"
        return {"op": op, "n": n, "lo": rng.choice([0, 1, (hi + 1) // 2]), "hi": hi, "q_heads": q, "kv_heads": kv, "dim": dim,
                "bs": bs, "codes": codes, "dtype": dtype}
    backward = rng.random() < 0.4
    vocab = rng.choice([512, 4096, 32000, 128256, _log_int(rng, 64, 160000)])
    rows = _log_int(rng, 1, max(1, min(8192, 200_000_000 // vocab)))
    return {"op": op, "rows": rows, "vocab": vocab, "top": 0 if backward else rng.choice([0, 1, 5, 20]), "dtype": dtype,
            "backward": backward}


# ----------------------------------------------------------------------------------------------------- inputs
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8,
          "e4m3": torch.float8_e4m3fn}


def _lengths(case, lo, hi, salt):
    """Lengths of a case's requests: even over the logarithm where the range is wide. They belong to the case, not to the seed
    (a case has one amount of work)."""
    rng = random.Random("%s %d %d %d" % (salt, case["n"], lo, hi))
    if lo >= 1 and hi > 8 * lo:
        got = [_log_int(rng, lo, hi) for _ in range(case["n"])]
    else:
        got = [rng.randint(lo, hi) for _ in range(case["n"])]
    if salt == "cached" and case["n"] > 1 and hi > lo:
        got[0] = hi
    return got


def _cached(case):
    return _lengths(case, case["lo"], case["hi"], "cached")


def _new(case):
    return _lengths(case, case["new_lo"], case["new_hi"], "new")


def _released(case):
    rng = random.Random("released %d" % case["n"])
    return [bool(case.get("release")) and rng.random() < 0.1 for _ in range(case["n"])]


def _up(a, b):
    return -(-a // b)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _table(counts, width, gen, spare):
    """A block table whose row n has counts[n] blocks out of a shuffled pool, -1 behind them; the shuffled pool; the blocks in use."""
    used = sum(counts)
    pool = torch.randperm(used + spare, generator=gen, device="cuda").to(torch.int32)
    cnt = _ints(counts, torch.int64)
    j = torch.arange(width, device="cuda")
    at = (cnt.cumsum(0) - cnt)[:, None] + j
    table = torch.where(j < cnt[:, None], pool[at.clamp(max=used + spare - 1)], -1)
    return table.to(torch.int32).contiguous(), pool, used


def _pool_values(shape, dtype, gen):
    """Codes and scales of a filled cache: normal values, a few strong channels, quantised by block and head."""
    codes = torch.empty(shape, dtype=_TYPES[dtype], device="cuda")
    scales = torch.empty(shape[:3], dtype=torch.float32, device="cuda")
    strong = 1 + 5 * (torch.rand((shape[2], 1, shape[4]), generator=gen, device="cuda") < 0.03).float()
    for i in range(2):
        step = max(1, (1 << 28) // (shape[2] * shape[3] * shape[4]))
        for b in range(0, shape[1], step):
            x = torch.randn((min(step, shape[1] - b),) + tuple(shape[2:]), generator=gen, device="cuda")
            x *= strong if i == 0 else 1.0
            e = _exponent(x.abs().amax((-1, -2)), dtype)
            codes[i, b:b + step] = _encode(x * _pow2(-e)[..., None, None], dtype)
            scales[i, b:b + step] = _pow2(e)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "plan":
        lens, new = _cached(case), _new(case)
        width = max(1, _up(max(a + b for a, b in zip(lens, new)), case["bs"]))
        spare = sum(_up(a + b, case["bs"]) - _up(a, case["bs"]) for a, b in zip(lens, new)) + 8
        s["table"], pool, used = _table([_up(a, case["bs"]) for a in lens], width, gen, spare)
        s["free"] = torch.cat([pool[used:], torch.full((used,), -1, dtype=torch.int32, device="cuda")])
        s["count"] = _ints([spare])
        s["lens"], s["new"], s["tokens"] = _ints(lens), _ints(new), sum(new)
        s["released"] = _ints(_released(case), torch.bool) if case["release"] else None
    elif case["op"] == "write":
        lens, new = _cached(case), _new(case)
        counts = [_up(a + b, case["bs"]) for a, b in zip(lens, new)]
        table, pool, _ = _table(counts, max(counts), gen, 4)
        blocks = pool.numel()
        s["codes"], s["scales"] = _pool_values((2, blocks, case["heads"], case["bs"], case["dim"]), case["codes"], gen)
        s["slots"] = _slots(table, _ints(lens, torch.int64), _ints(new, torch.int64), sum(new), case["bs"])
        shape = (sum(new), case["heads"], case["dim"])
        s["k"], s["v"] = ((torch.randn(shape, generator=gen, device="cuda") * 1.2).to(_TYPES[case["dtype"]]) for _ in range(2))
    elif case["op"] == "attend":
        lens = _cached(case)
        counts = [_up(a, case["bs"]) for a in lens]
        s["table"], pool, _ = _table(counts, max(1, max(counts)), gen, 1)
        s["codes"], s["scales"] = _pool_values((2, pool.numel(), case["kv_heads"], case["bs"], case["dim"]), case["codes"], gen)
        s["lens"] = _ints(lens)
        s["q"] = torch.randn((case["n"], case["q_heads"], case["dim"]), generator=gen, device="cuda").to(_TYPES[case["dtype"]])
    else:
        rows, vocab = case["rows"], case["vocab"]
        z = torch.randn((rows, vocab), generator=gen, device="cuda") * 2
        ids = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        z[torch.arange(rows, device="cuda"), ids] += 6 * torch.rand((rows,), generator=gen, device="cuda")
        ids[torch.rand((rows,), generator=gen, device="cuda") < 0.02] = IGNORED
        s["logits"], s["ids"] = z.to(_TYPES[case["dtype"]]), ids
        if case["backward"]:
            s["logits"].requires_grad_(True)
            s["d_logprob"] = torch.randn((rows,), generator=gen, device="cuda") / rows
            s["d_entropy"] = 0.1 * torch.randn((rows,), generator=gen, device="cuda") / rows
    return s


# ----------------------------------------------------------------------------------------------------- plain forms
def _pow2(e):
    """2^e as fp32, exactly (-126 <= e <= 127)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax, dtype):
    """The smallest e with amax <= largest code * 2^e (448 = 0.875 * 2^9 in e4m3, 127 = 0.9921875 * 2^7 in int8)."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).int() if dtype == "e4m3" else x - 7 + (m > 0.9921875).int()
    return torch.where(amax > 0, e.clamp(min=MIN_EXP), MIN_EXP)


def _encode(x, dtype):
    return torch.round(x).to(torch.int8) if dtype == "int8" else x.to(torch.float8_e4m3fn)


def _slots(table, lens, new, tokens, bs):
    cu = new.cumsum(0)
    t = torch.arange(tokens, device="cuda")
    n = torch.searchsorted(cu, t, right=True).clamp(max=new.numel() - 1)
    pos = (lens + new - cu)[n] + t
    return table[n, pos // bs].long() * bs + pos % bs


def _plan(s):
    """Released requests push their blocks on the stack of free blocks; then each request, in order, pops what its new tokens need
    beyond the blocks it has. A request whose blocks do not fit any more gets nothing. Lengths and the stack's height come back new."""
    table, free, bs = s["table"], s["free"], s["bs"]
    lens, new, count = s["lens"].long(), s["new"].long(), s["count"].long()
    have = (lens + bs - 1) // bs
    j = torch.arange(table.shape[1], device="cuda")
    may = torch.ones_like(lens, dtype=torch.bool)
    if s["released"] is not None:
        back = torch.where(s["released"], have, 0)
        at = (count + back.cumsum(0) - back)[:, None] + j
        at = torch.where(j < back[:, None], at, free.numel())
        more = torch.cat([free, free[:1]])
        more.scatter_(0, at.reshape(-1), table.reshape(-1))
        free.copy_(more[:-1])
        count = count + back.sum()
        lens, have, may = torch.where(s["released"], 0, lens), torch.where(s["released"], 0, have), ~s["released"]
    need = torch.where(may, (lens + new + bs - 1) // bs - have, 0)
    top = need.cumsum(0)
    served = (new == 0) | (may & ((need == 0) | (top <= count)))
    need, top = torch.where(served, need, 0), torch.where(served, top, 0)
    k = j - have[:, None]
    fresh = (k >= 0) & (k < need[:, None])
    at = (count - 1 - (top - need)[:, None] - k).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[at], table))
    slots = _slots(table, lens, new, s["tokens"], bs)
    cu = new.cumsum(0)
    n = torch.searchsorted(cu, torch.arange(s["tokens"], device="cuda"), right=True)
    slots = torch.where(served[n], slots, -1)
    return [slots, torch.where(served, lens + new, lens).int(), (count - need.sum()).int(), served, table, free]


def _write_one(x, slots, codes, scales, dtype):
    """One of the two halves: x [tokens, heads, dim] into codes [blocks, heads, bs, dim], scales [blocks, heads]. The first new offset
    of a block tells how many tokens it holds already; where the new ones need a larger scale those are quantised anew."""
    blocks, heads, bs, dim = codes.shape
    b, off = slots // bs, slots % bs
    x = x.float()
    amax = torch.zeros((blocks, heads), device="cuda").index_reduce_(0, b, x.abs().amax(-1), "amax")
    start = torch.full((blocks,), bs, device="cuda").scatter_reduce_(0, b, off, "amin")
    touched = (start < bs)[:, None]
    old = torch.where((start > 0)[:, None], torch.frexp(scales)[1] - 1, MIN_EXP)
    e = torch.maximum(_exponent(amax, dtype), old)
    down = torch.where(touched & (start > 0)[:, None], old - e, 0).clamp(min=-126)
    kept = _encode(codes.float() * _pow2(down)[..., None, None], dtype)
    again = (down < 0)[..., None, None] & (torch.arange(bs, device="cuda")[:, None] < start[:, None, None, None])
    codes.copy_(torch.where(again, kept.float(), codes.float()))
    scales.copy_(torch.where(touched, _pow2(e), scales))
    codes.view(torch.int8)[b, :, off] = _encode(x * _pow2(-e)[b][..., None], dtype).view(torch.int8)


def _write(s):
    _write_one(s["k"], s["slots"], s["codes"][0], s["scales"][0], s["codes_type"])
    _write_one(s["v"], s["slots"], s["codes"][1], s["scales"][1], s["codes_type"])


def _attend(s):
    q, codes, scales, table, lens = s["q"], s["codes"], s["scales"], s["table"].long().clamp(min=0), s["lens"]
    n, heads, dim = q.shape
    _, _, kv, bs, _ = codes.shape
    span = table.shape[1] * bs

    def cached(i):                                                                   # [n, kv, span, dim]
        x = codes[i].view(torch.int8)[table].view(codes.dtype).float() * scales[i][table][..., None, None]
        return x.transpose(1, 2).reshape(n, kv, span, dim)

    score = (q.float().view(n, kv, heads // kv, dim) * dim ** -0.5) @ cached(0).transpose(2, 3)
    seen = (torch.arange(span, device="cuda") < lens[:, None])[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    o = (p @ cached(1)) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.view(n, heads, dim).to(q.dtype)


def _logprob(s):
    z, ids, top = s["logits"].detach().float(), s["ids"], s["top"]
    scored = ids >= 0
    peak = z.amax(-1, keepdim=True)
    e = torch.exp(z - peak)
    total = e.sum(-1, keepdim=True)
    lse = peak + torch.log(total)
    own_z = z.gather(1, ids.clamp(min=0)[:, None])
    logprob = torch.where(scored, (own_z - lse)[:, 0], 0.0)
    p = e / total
    entropy = -(p * (z - lse)).sum(-1)
    if s["backward"]:
        d = -p * (s["d_logprob"] * scored)[:, None] - p * ((z - lse) + entropy[:, None]) * s["d_entropy"][:, None]
        d.scatter_add_(1, ids.clamp(min=0)[:, None], (s["d_logprob"] * scored)[:, None])
        return [logprob, entropy, d.to(s["logits"].dtype)]
    if top == 0:
        return [logprob, entropy]
    # descending values, the lowest index first among equal ones: one whole number that orders both
    bits = (z + 0.0).view(torch.int32).long()                                        # -0.0 equals 0.0
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 20) + (z.shape[1] - 1 - torch.arange(z.shape[1], device="cuda"))
    best = z.shape[1] - 1 - (key.topk(top, -1).values & 0xFFFFF)
    return [logprob, entropy, z.gather(1, best) - lse, best]


# ----------------------------------------------------------------------------------------------------- one pass
def run(s):
    """The cache's codes are exactly defined (the scales are powers of two, so a scaled value is rounded once), and come back as
    they are held, with their scales."""
    op = s["op"]
    if own:
        from hippolm_b200 import ops
        if op == "plan":
            p = ops.kv8_plan(s["table"], s["lens"], s["new"], s["free"], s["count"], s["bs"], s["tokens"], release=s["released"])
            return [p.slots, p.lens, p.free_count, p.served, s["table"], s["free"]]
        if op == "write":
            ops.kv8_write(s["k"], s["v"], s["slots"], s["codes"], s["scales"])
            return [s["codes"], s["scales"]]
        if op == "attend":
            return [ops.attention_decode_kv8(s["q"], s["codes"], s["scales"], s["table"], s["lens"])]
        if s["backward"]:
            lp, ent = ops.token_logprobs(s["logits"], s["ids"])[:2]
            return [lp, ent, torch.autograd.grad((lp, ent), s["logits"], (s["d_logprob"], s["d_entropy"]))[0]]
        got = ops.token_logprobs(s["logits"], s["ids"], top_k=s["top"])
        return list(got) if s["top"] else list(got[:2])
    if op == "plan":
        return _plan(s)
    if op == "write":
        _write(dict(s, codes_type="int8" if s["codes"].dtype == torch.int8 else "e4m3"))
        return [s["codes"], s["scales"]]
    if op == "attend":
        return [_attend(s)]
    return _logprob(s)


# ----------------------------------------------------------------------------------------------------- work
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def work(case):
    if case["op"] == "plan":
        lens, new, bs = _cached(case), _new(case), case["bs"]
        gone = _released(case)
        fresh = sum(_up(a + b, bs) - _up(a, bs) for a, b, g in zip(lens, new, gone) if not g)
        back = sum(_up(a, bs) for a, g in zip(lens, gone) if g)
        # lengths read and written, a block popped or pushed is read and written once, one slot written for each token
        return {"bytes": 13 * case["n"] + 8 * (fresh + back) + 8 * sum(new), "flops": 4 * sum(new) + 8 * case["n"]}
    if case["op"] == "write":
        lens, new, bs = _cached(case), _new(case), case["bs"]
        tokens, row = sum(new), case["heads"] * case["dim"]
        blocks = sum(_up(a + b, bs) - a // bs for a, b in zip(lens, new) if b)
        return {"bytes": 2 * tokens * row * (_BYTES[case["dtype"]] + 1) + 8 * tokens + 2 * 8 * blocks * case["heads"],
                "flops": 2 * 3 * tokens * row}
    if case["op"] == "attend":
        lens = _cached(case)
        blocks = sum(_up(a, case["bs"]) for a in lens)
        rows = 2 * case["n"] * case["q_heads"] * case["dim"] * _BYTES[case["dtype"]]
        return {"bytes": 2 * sum(lens) * case["kv_heads"] * case["dim"] + blocks * (8 * case["kv_heads"] + 4) + rows,
                "flops": 4 * sum(lens) * case["q_heads"] * case["dim"]}
    size = case["rows"] * case["vocab"]
    if case["backward"]:
        return {"bytes": 2 * size * _BYTES[case["dtype"]] + case["rows"] * 24, "flops": 12 * size}
    return {"bytes": size * _BYTES[case["dtype"]] + case["rows"] * (16 + 12 * case["top"]), "flops": 6 * size}


# ----------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None                                       # whole numbers only: there is nothing to compute in 64 bits
    if case["op"] == "write":
        return _exact_write(case, s)
    if case["op"] == "attend":
        codes, scales, bs = s["codes"], s["scales"], case["bs"]
        group = case["q_heads"] // case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for n, length in enumerate(_cached(case)):
            if length == 0:
                continue
            blocks = s["table"][n, :_up(length, bs)].long()
            for h in range(case["kv_heads"]):
                k, v = ((codes[i].view(torch.int8)[blocks, h].view(codes.dtype).double() * scales[i][blocks, h].double()[:, None, None])
                        .reshape(-1, case["dim"])[:length] for i in range(2))
                q = s["q"][n, h * group:(h + 1) * group].double()
                out[n, h * group:(h + 1) * group] = torch.softmax(q @ k.T / math.sqrt(case["dim"]), -1) @ v
        return [out]
    z, ids = s["logits"].detach(), s["ids"]
    scored = ids >= 0
    got = [[], [], [], []]
    for a in range(0, case["rows"], 512):
        x = z[a:a + 512].double()
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        h = torch.special.entr(p).sum(-1)
        hit = torch.zeros_like(x)
        i = ids[a:a + 512]
        hit[scored[a:a + 512], i[scored[a:a + 512]]] = 1.0
        got[0].append((lp * hit).sum(-1))
        got[1].append(h)
        if case["backward"]:
            d_lp = s["d_logprob"][a:a + 512].double()[:, None] * hit.sum(-1, keepdim=True)
            d_h = s["d_entropy"][a:a + 512].double()[:, None]
            got[2].append(d_lp * (hit - p) - d_h * p * (lp + h[:, None]))
        elif case["top"]:
            got[2].append(lp.sort(-1, descending=True).values[:, :case["top"]])
    out = [torch.cat(got[0]), torch.cat(got[1])]
    if case["backward"]:
        return out + [torch.cat(got[2])]
    return out + [torch.cat(got[2]), None] if case["top"] else out


def _exact_write(case, s):
    """Codes and scales from the definition, one (block, head) at a time over the whole pool, in 64 bits."""
    codes, scales, bs = s["codes"].double(), s["scales"].double(), case["bs"]
    blocks, offs = s["slots"] // bs, s["slots"] % bs
    largest = 127.0 if case["codes"] == "int8" else 448.0

    def nearest(x):
        if case["codes"] == "int8":
            return torch.round(x)
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)     # 3 bits behind the leading one
        return torch.round(x / step) * step

    for i, x in enumerate((s["k"].double(), s["v"].double())):
        for b in range(0, codes.shape[1], 64):                                       # 64 blocks of the pool at a time
            mine = ((blocks >= b) & (blocks < b + 64)).nonzero()[:, 0]
            if mine.numel() == 0:
                continue
            new = torch.zeros_like(codes[i, b:b + 64])
            there = torch.zeros(new.shape[0], bs, dtype=torch.bool, device="cuda")
            new[blocks[mine] - b, :, offs[mine]] = x[mine]
            there[blocks[mine] - b, offs[mine]] = True
            first = torch.where(there.any(1), there.int().argmax(1), bs)
            past = (torch.arange(bs, device="cuda") < first[:, None]) & there.any(1)[:, None]
            value = torch.where(past[:, None, :, None], codes[i, b:b + 64], new / scales[i, b:b + 64, :, None, None])
            peak = new.abs().amax((2, 3)) / largest
            scale = torch.exp2(torch.ceil(torch.log2(peak.clamp(min=2.0 ** MIN_EXP))))
            scale = torch.where(past.any(1)[:, None], torch.maximum(scale, scales[i, b:b + 64]), scale)
            held = nearest(value * (scales[i, b:b + 64] / scale)[..., None, None])
            use = (past | there)[:, None, :, None]
            codes[i, b:b + 64] = torch.where(use, held, codes[i, b:b + 64])
            scales[i, b:b + 64] = torch.where(there.any(1)[:, None], scale, scales[i, b:b + 64])
    return [codes, scales]
