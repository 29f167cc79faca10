"""8-bit paged key / value cache and per-token scores: the CUDA kernels against plain 64-bit statements."""
import math

import numpy as np
import pytest
import torch

import kv8_plain as plain
from hippolm_b200 import ops
from hippolm_b200.ops import _ext
from hippolm_b200.ops.kv8 import kv8_empty
from test_kv8 import PLAN_CASES, WRITE_RUNS, cache_case, check_plan, check_special, check_write, make_plan_case, runs_to_slots

pytestmark = pytest.mark.gpu
DEV = "cuda"


def to(device, *xs):
    return [x.to(device) for x in xs]


# ------------------------------------------------------------------------------------------------ plan
@pytest.mark.parametrize("n,bs,M,hi,new_hi,spare,release",
                         PLAN_CASES + [(1500, 16, 5, 70, 3, 900, True), (1025, 32, 3, 96, 2, 2000, False), (130, 64, 9, 500, 80, 90, True)])
def test_plan_matches_lists(n, bs, M, hi, new_hi, spare, release):
    for seed in range(2):
        check_plan(make_plan_case(seed, n, bs, M, hi, new_hi, spare, release, DEV))


@pytest.mark.parametrize("n,new_hi", [(3, 9000), (40, 1200), (2000, 30)])
def test_plan_of_prompts(n, new_hi):
    c = make_plan_case(n, n, 64, new_hi // 64 + 3, 100, new_hi, n * (new_hi // 64 + 2), False, DEV)
    assert c["num_tokens"] > 12000                                            # both sides of the size rule
    check_plan(c)
    check_plan(dict(c, num_tokens=c["num_tokens"] + 70000, table=c["table"].clone(), free_list=c["free_list"].clone()))
    check_plan(dict(c, num_tokens=c["num_tokens"] - 1, table=c["table"].clone(), free_list=c["free_list"].clone()))


def test_plan_of_a_strided_table():
    c = make_plan_case(1, 6, 16, 8, 100, 20, 30, False, DEV)
    wide = torch.full((6, 20), -3, dtype=torch.int32, device=DEV)
    wide[:, 4:12] = c["table"]
    c["table"] = wide[:, 4:12]
    check_plan(c)
    assert (wide[:, :4] == -3).all() and (wide[:, 12:] == -3).all()


# ------------------------------------------------------------------------------------------------ write
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bs", [16, 32, 64])
@pytest.mark.parametrize("window", [0, 5, 16])
def test_write_matches_64_bits(kind, D, bs, window):
    from hippolm_b200.ops import kv8_cuda
    dtypes = [torch.bfloat16, torch.float16, torch.float32]
    for runs in range(len(WRITE_RUNS)):
        codes, scales, g = cache_case(runs, kind, 3, D, bs, 8)
        codes, scales = codes.to(DEV), scales.to(DEV)
        slots = runs_to_slots(WRITE_RUNS[runs](bs), bs)
        dt = dtypes[(runs + bs // 16) % 3]
        k, v = ((torch.randn(slots.numel(), 3, D, generator=g) * 20 ** float(i)).to(dt) for i in range(2))
        k, v, slots = to(DEV, k, v, slots)
        check_write(k, v, slots, codes, scales, kind, write=lambda *a: kv8_cuda.write(*a, 0, a[0].shape, a[3].shape, window=window))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("window", [0, 2, 16])
def test_write_poison_zeros_far_slots_and_strides(kind, window):
    from hippolm_b200.ops import kv8_cuda
    codes, scales, g = cache_case(0, kind, 2, 64, 16, 4)
    codes, scales = codes.to(DEV), scales.to(DEV)
    qkv = torch.randn(7, 2, 3 * 64, generator=g)
    qkv[0, 1, 3], qkv[2, 0, 64], qkv[4, :, :64], qkv[6] = math.nan, math.inf, 0.0, 1e-38
    qkv = qkv.to(DEV)
    k, v = qkv[..., :64], qkv[..., 64:128]                                    # strided heads
    slots = torch.tensor([5, 16, 17, 4 * 16, 2 * 16, 1 << 40, 3 * 16], device=DEV)
    write = lambda *a: kv8_cuda.write(*a, 0, a[0].shape, a[3].shape, window=window)                         # noqa: E731
    check_write(k, v, slots, codes, scales, kind, write=write)
    check_write(k[5:6], v[5:6], torch.tensor([18], device=DEV), codes, scales, kind, write=write)
    check_write(k[5:6], v[5:6], torch.tensor([16], device=DEV), codes, scales, kind, write=write)
    odd = torch.randn(2 * 2 * 64 + 1, device=DEV)[1:].view(2, 2, 64)          # 4-byte alignment
    check_write(odd, odd, torch.tensor([32, 33], device=DEV), codes, scales, kind, write=write)


@pytest.mark.parametrize("kind,bs", [("e4m3", 64), ("int8", 16)])
def test_write_of_many_runs_equals_a_few(kind, bs):
    """One call with thousands of short and long runs against calls with a few of them each (other windows)."""
    g = torch.Generator().manual_seed(bs)
    runs, block = [], 0
    while sum(r[2] for r in runs) < 6000:
        off = int(torch.randint(0, bs, (1,), generator=g)) if torch.rand(1, generator=g) < 0.7 else 0
        ln = 1 if torch.rand(1, generator=g) < 0.5 else int(torch.randint(1, bs - off + 1, (1,), generator=g))
        runs.append((block, off, ln))
        block += 1
    codes, scales = kv8_empty(block, 3, 64, bs, kind, DEV)
    codes.view(torch.int8).copy_(torch.randint(-100, 100, codes.shape, generator=g).to(torch.int8))
    scales.mul_(0.01).copy_(torch.exp2(torch.randint(-9, 2, scales.shape, generator=g).float()))
    slots = runs_to_slots(runs, bs)
    k, v = (torch.randn(slots.numel(), 3, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    other_c, other_s = codes.clone(), scales.clone()
    ops.kv8_write(k, v, slots.to(DEV), codes, scales)
    at = 0
    for i in range(0, len(runs), 9):
        n = sum(r[2] for r in runs[i:i + 9])
        ops.kv8_write(k[at:at + n], v[at:at + n], slots[at:at + n].to(DEV), other_c, other_s)
        at += n
    assert torch.equal(codes.view(torch.int8), other_c.view(torch.int8)) and torch.equal(scales, other_s)
    few = slots[:300]
    c0, s0 = kv8_empty(block, 3, 64, bs, kind, DEV)
    check_write(k[:300], v[:300], few.to(DEV), c0, s0, kind)


@pytest.mark.parametrize("kind,dtype", [("e4m3", torch.bfloat16), ("int8", torch.float32), ("int8", torch.float16)])
@pytest.mark.parametrize("D,bs", [(64, 32), (128, 32), (128, 16)])
def test_write_of_runs_of_every_short_length(kind, dtype, D, bs):
    """Runs of 1 to 16 tokens, alone and behind older ones, the largest value in their first, middle or last row; one is poisoned."""
    runs = [(b, 0 if b % 2 == 0 else min(b, bs - 1 - b // 2), b // 2 + 1) for b in range(32)]
    runs = [(b, min(off, bs - ln), ln) for b, off, ln in runs]
    codes, scales, g = cache_case(7, kind, 3, D, bs, 32)
    slots = runs_to_slots(runs, bs)
    k, v = (torch.randn(slots.numel(), 3, D, generator=g) for _ in range(2))
    at = 0
    for b, _, ln in runs:
        k[at + (b * 5) % ln, b % 3, b % D] = 300.0
        if b == 21:
            v[at + ln - 1, 1, 5] = math.inf
        at += ln
    check_write(*to(DEV, k.to(dtype), v.to(dtype), slots, codes, scales), kind, write=ops.kv8_write)


def test_write_leaves_the_rest_of_the_cache():
    codes, scales = kv8_empty(60, 2, 64, 64, "int8", DEV)
    codes.fill_(77); scales.fill_(0.5)
    T = 3000                                                                  # windows of whole blocks
    slots = torch.arange(T, device=DEV) + 64
    k = torch.randn(T, 2, 64, device=DEV)
    c0, s0 = codes.clone(), scales.clone()
    check_write(k[:100], k[:100] * 3, slots[:100], codes.clone(), scales.clone(), "int8")
    ops.kv8_write(k, k, slots, codes, scales)
    last = (64 + T) // 64
    assert torch.equal(codes[:, 0], c0[:, 0]) and torch.equal(codes[:, last + 1:], c0[:, last + 1:])
    assert torch.equal(codes[:, last, :, (64 + T) % 64:], c0[:, last, :, (64 + T) % 64:])
    assert torch.equal(scales[:, 0], s0[:, 0]) and torch.equal(scales[:, last + 1:], s0[:, last + 1:])


# ------------------------------------------------------------------------------------------------ attention
def attend_case(seed, kind, Hq, H, D, bs, lens, dtype, spare=2, tail=None):
    counts = [-(-x // bs) for x in lens]
    nb = sum(counts) + spare
    codes, scales, g = cache_case(seed, kind, H, D, bs, nb)
    M = max(counts + [1])
    table = torch.full((len(lens), M), -1, dtype=torch.int32)
    perm = torch.randperm(nb, generator=g).to(torch.int32)
    at = 0
    for n, c in enumerate(counts):
        table[n, :c] = perm[at:at + c]
        at += c
    if tail is not None:                                                      # bytes behind the last token
        raw = codes.view(torch.int8)
        for n, x in enumerate(lens):
            if x % bs:
                raw[:, int(table[n, x // bs]), :, x % bs:] = tail
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype)
    return to(DEV, q, codes, scales, table, torch.tensor(lens, dtype=torch.int32))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bs", [16, 32, 64])
@pytest.mark.parametrize("Hq,H", [(2, 2), (6, 2), (12, 1)])
def test_attention_matches_64_bits(kind, D, bs, Hq, H):
    dt = {16: torch.bfloat16, 32: torch.float16, 64: torch.float32}[bs]
    for i, lens in enumerate(([1], [0, 33, 0, 15, 64, 0], [200, 16, 31, 32, 65, 7, 129])):
        c = attend_case(i, kind, Hq, H, D, bs, lens, dt, tail=127)            # 0x7f: NaN in e4m3
        plain.check_attend(ops.attention_decode_kv8(*c), *c, D ** -0.5)
    assert _ext.device_status()[0] == 0


@pytest.mark.parametrize("kind,D,bs,Hq,H,lens", [
    ("e4m3", 128, 64, 2, 2, [5003, 1, 2000]), ("int8", 64, 16, 4, 1, [9001]), ("int8", 128, 32, 8, 1, [3001, 2999, 64, 1]),
    ("e4m3", 64, 64, 3, 3, [1] * 200 + [700] + [0] * 30 + [2] * 40)])
def test_attention_of_long_and_many_sequences(kind, D, bs, Hq, H, lens):
    c = attend_case(3, kind, Hq, H, D, bs, lens, torch.float32, tail=-1)
    plain.check_attend(ops.attention_decode_kv8(*c), *c, D ** -0.5)
    a, b = ops.attention_decode_kv8(*c), ops.attention_decode_kv8(*c)
    assert torch.equal(a, b)


def test_attention_scales_of_any_size_and_poison():
    q, codes, scales, table, lens = attend_case(5, "int8", 4, 2, 64, 16, [100, 47, 33], torch.float32)
    scales[1] *= torch.exp2(torch.randint(-40, 40, scales[1].shape, device=DEV).float())
    plain.check_attend(ops.attention_decode_kv8(q, codes, scales, table, lens), q, codes, scales, table, lens, 64 ** -0.5)
    scales[1, 3:] *= 1.37                                                     # not a power of two: still code * scale
    plain.check_attend(ops.attention_decode_kv8(q, codes, scales, table, lens, scale=0.01), q, codes, scales, table, lens, 0.01)
    scales[0, int(table[1, 1]), 0] = math.nan
    scales[1, int(table[2, 0]), 1] = math.nan
    got = ops.attention_decode_kv8(q, codes, scales, table, lens)
    assert torch.isnan(got[1, :2]).all() and torch.isnan(got[2, 2:]).all()
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1, 2:]).all() and torch.isfinite(got[2, :2]).all()
    q[0, 0, 5] = math.nan
    got = ops.attention_decode_kv8(q, codes, scales, table, lens)
    assert torch.isnan(got[0, 0]).all() and torch.isfinite(got[0, 1:]).all()


def test_attention_bad_blocks_long_lengths_and_strides():
    q, codes, scales, table, lens = attend_case(6, "e4m3", 4, 2, 128, 16, [90, 64, 17, 40], torch.bfloat16)
    table[0, 2], table[1, 0], table[2, :2], table[3, 1] = -1, 1 << 30, -5, codes.shape[1]
    lens[1] = 1 << 30                                                         # counts as the table's width
    table[1, 4:] = table[0, 0]
    wide = torch.randn(4, 9, 128 * 3, device=DEV, dtype=torch.bfloat16)
    wide[:, 1:5, 128:256] = q
    qs = wide[:, 1:5, 128:256]
    got = ops.attention_decode_kv8(qs, codes, scales, table, lens)
    plain.check_attend(got, q, codes, scales, table, lens, 128 ** -0.5)
    assert not got[2].any()
    cols = torch.empty(4, 128, 4, device=DEV, dtype=torch.bfloat16).transpose(1, 2)
    cols.copy_(q)
    assert torch.equal(ops.attention_decode_kv8(cols, codes, scales, table, lens), got)
    shared = table[:1].expand(4, -1)
    lens[1] = 70
    plain.check_attend(ops.attention_decode_kv8(q, codes, scales, shared, lens), q, codes, scales, shared, lens, 128 ** -0.5)


def test_attention_behind_four_gigabytes():
    """Blocks whose codes lie beyond 2^32 bytes and 2^31 elements of the cache."""
    nb = 700_000
    codes = torch.zeros((2, nb, 1, 64, 128), dtype=torch.int8, device=DEV)    # 11.5 GB
    scales = torch.ones((2, nb, 1), device=DEV)
    k = torch.randn(130, 1, 128, device=DEV)
    v = torch.randn(130, 1, 128, device=DEV)
    blocks = [nb - 1, 5, nb - 2]
    slots = torch.tensor([blocks[i // 64] * 64 + i % 64 for i in range(130)], device=DEV)
    ops.kv8_write(k, v, slots, codes, scales)
    table = torch.tensor([blocks], dtype=torch.int32, device=DEV)
    lens = torch.tensor([130], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 2, 128, device=DEV)
    got = ops.attention_decode_kv8(q, codes, scales, table, lens)
    small_c, small_s = codes[:, blocks].contiguous(), scales[:, blocks].contiguous()
    plain.check_attend(got, q, small_c, small_s, torch.tensor([[0, 1, 2]], dtype=torch.int32), lens, 128 ** -0.5)
    want_c, want_s = plain.write(k, v, torch.arange(130), torch.zeros_like(small_c), torch.ones_like(small_s), "int8")
    assert np.array_equal(plain.value_of(small_c), want_c) and np.array_equal(small_s.cpu().double().numpy(), want_s)


# ------------------------------------------------------------------------------------------------ scores
def score_bound(z, dtype):
    """Sums of V fp32 terms in up to 16 partial sums of V / 512 each, exponentials off by 2^-21 or so of their arguments' size: the
    logarithm moves by that much, plus a few half steps of the largest logit."""
    V = z.shape[1]
    zmax = float(z.float().abs().nan_to_num(0, 0, 0).max())
    return (V / 512 + 64) * 2.0 ** -24 + 2.0 ** -20 + 8 * 2.0 ** -24 * max(zmax, 1.0)


@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (3, 2, 2), (5, 33, 20), (2, 600, 5), (4, 1031, 32), (1, 9000, 20), (3, 32000, 1),
                                     (2, 128256, 20), (700, 515, 3), (1, 523776, 32),
                                     (1300, 9001, 20), (5000, 700, 3), (9500, 130, 8), (1000, 1024, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_scores_match_64_bits(T, V, top, dtype):
    g = torch.Generator().manual_seed(V)
    z = (torch.randn(T, V, generator=g) * 3).to(dtype)
    ids = torch.randint(0, V, (T,), generator=g)
    ids[T // 2] = -100
    if T > 2:
        ids[2] = V
    zd, idd = to(DEV, z, ids)
    got = ops.token_logprobs(zd, idd, top_k=top)
    x = z.double()
    lp = torch.log_softmax(x, -1)
    inside = (ids >= 0) & (ids < V)
    want = torch.where(inside, lp.gather(1, ids.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    b = score_bound(z, dtype)
    assert float((got.logprob.cpu() - want).abs().max()) <= b
    # the entropy weighs every error by the distance from the maximum, up to 2 max|z|
    assert float((got.entropy.cpu() - torch.special.entr(lp.exp()).sum(-1)).abs().max()) <= b * (1 + 2 * float(z.abs().max()))
    order = torch.sort(z.float(), dim=-1, descending=True, stable=True)
    assert torch.equal(got.top_ids.cpu(), order.indices[:, :top])
    assert float((got.top_logprobs.cpu() - lp.gather(1, order.indices[:, :top])).abs().max()) <= b
    plain_call = ops.token_logprobs(zd, idd)
    assert plain_call.top_ids is None and torch.equal(plain_call.logprob, got.logprob) and torch.equal(plain_call.entropy, got.entropy)


@pytest.mark.parametrize("T,V,top", [(5000, 4099, 20), (5000, 2047, 0), (4800, 9001, 3), (2500, 4097, 32), (600, 20011, 5), (150, 66001, 20)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_scores_of_many_rows(T, V, top, dtype):
    """More rows than the card holds at once (blocks of one warp and of few), rows at odd addresses, equal logits among the largest."""
    g = torch.Generator(device=DEV).manual_seed(V)
    z = (torch.randn(T, V + 3, device=DEV, generator=g) * 3).to(dtype)[:, 1:V + 1]
    z[::7] = z[::7].round()
    z[5, :] = -math.inf
    z[5, V - 1] = 1.0
    ids = torch.randint(0, V, (T,), device=DEV, generator=g)
    ids[5] = V - 1
    got = ops.token_logprobs(z, ids, top_k=top)
    b = score_bound(z[6:], dtype)
    for s in range(0, T, 500):
        lp = torch.log_softmax(z[s:s + 500].double(), -1)
        assert float((got.logprob[s:s + 500] - lp.gather(1, ids[s:s + 500, None])[:, 0]).abs().max()) <= b
        assert float((got.entropy[s:s + 500] - torch.special.entr(lp.exp()).sum(-1)).abs().max()) <= b * (1 + 2 * float(z[6:].abs().max()))
        if top:
            order = torch.sort(z[s:s + 500].float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
            assert torch.equal(got.top_ids[s:s + 500], order)
            want, have = lp.gather(1, order), got.top_logprobs[s:s + 500]
            assert torch.equal(torch.isneginf(want), torch.isneginf(have))
            assert float((have - want).nan_to_num(0.0).abs().max()) <= b


def test_scores_of_masked_and_broken_rows():
    check_special(DEV)


@pytest.mark.parametrize("V,top", [(4096, 20), (20000, 32), (128256, 7), (1000, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_alternatives_among_equal_logits(V, top, dtype):
    z = torch.zeros(10, V, device=DEV, dtype=dtype)
    z[1, V - 5:] = 1.0
    z[2, ::3] = 2.0
    z[3] = -math.inf
    z[4, V // 2:] = math.nan
    z[5, 5:] = -math.inf
    z[6] = torch.finfo(dtype).min
    z[6, V // 3] = -3.0
    z[7] = -1.5 - torch.arange(V, device=DEV) % 7
    z[8, 100:900:90] = math.inf
    z[9, ::2] = -0.0
    got = ops.token_logprobs(z, torch.zeros(10, dtype=torch.int64, device=DEV), top_k=top)
    order = torch.sort(z.float().cpu() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids.cpu(), order)
    want = torch.log_softmax(z.double().cpu(), -1).gather(1, order)
    for t in (0, 1, 2, 5, 6, 7, 9):
        w = want[t].clamp(min=torch.finfo(torch.float32).min)
        g = got.top_logprobs[t].cpu().double().clamp(min=torch.finfo(torch.float32).min)
        assert bool(((g - w).abs() <= 1e-5 + 1e-6 * w.abs()).all()), t
    assert torch.isneginf(got.top_logprobs[3]).all() and torch.isnan(got.top_logprobs[[4, 8]]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,off,ld", [(5, 13, 0, 13), (7, 1001, 3, 1024), (3, 4096, 1, 4099), (2, 32000, 0, 32000)])
def test_score_gradient(dtype, T, V, off, ld):
    g = torch.Generator().manual_seed(V)
    store = torch.full((T, ld + 16), float("nan"), dtype=dtype)
    store[:, off:off + V] = (torch.randn(T, V, generator=g) * 2).to(dtype)
    store[0, off + V // 2] = -math.inf
    z = store.to(DEV)[:, off:off + V].detach().requires_grad_(True)             # rows that start anywhere
    ids = torch.randint(0, V, (T,), generator=g)
    ids[T - 1] = -100
    a, b = torch.randn(T, generator=g), torch.randn(T, generator=g)
    x = z.detach().cpu().double()
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    h = torch.special.entr(p).sum(-1, keepdim=True)
    hit = torch.nn.functional.one_hot(ids.clamp(min=0), V).double() * (ids >= 0)[:, None]
    want_lp = a[:, None].double() * (hit - p * (ids >= 0)[:, None])
    want_h = -b[:, None].double() * p * torch.where(p > 0, lp + h, 0.0)
    ad, bd, idd = to(DEV, a, b, ids)
    for g_lp, g_h in ((ad, bd), (ad, None), (None, bd)):
        got = ops.token_logprobs(z, idd, top_k=min(V, 3) if g_h is None else 0)
        outs = [o for o, gr in ((got.logprob, g_lp), (got.entropy, g_h)) if gr is not None]
        (d,) = torch.autograd.grad(outs, z, [gr for gr in (g_lp, g_h) if gr is not None])
        assert d.dtype == dtype and d.shape == z.shape
        want = (want_lp if g_lp is not None else 0) + (want_h if g_h is not None else 0)
        size = a.abs().max() * (p + hit) + b.abs().max() * p * (lp.clamp(min=-100).abs() + h + 1)     # terms before they cancel
        # p and H off by the bound of the scores and by fp32 arguments of the exponential (2^-19 for |z - lse| < 32), one rounding
        tol = size * (2.0 ** -17 + score_bound(x, dtype) * (2 + 2 * 8.0)) + want.abs() * plain.half_step(dtype)
        if dtype == torch.float16:
            tol = tol + 2.0 ** -25
        assert bool(((d.cpu().double() - want).abs() <= tol + 1e-38).all())
    with pytest.raises(RuntimeError):
        got = ops.token_logprobs(z, idd)
        (d,) = torch.autograd.grad(got.logprob.sum(), z, create_graph=True)
        torch.autograd.grad(d.sum(), z)


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def test_refusals():
    codes, scales = kv8_empty(4, 2, 96, 16, "int8", DEV)
    table, lens = torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV)
    x, sl = torch.zeros(3, 2, 96, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for f in (lambda: ops.kv8_write(x, x, sl, codes, scales), lambda: ops.attention_decode_kv8(x, codes, scales, table, lens),
              lambda: ops.attention_decode_kv8(x, codes.cpu(), scales, table, lens),
              lambda: ops.token_logprobs(torch.zeros(1, 523777, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)),
              lambda: ops.token_logprobs(x[:, 0], sl.cpu())):
        with pytest.raises(ValueError):
            f()


def test_empty_calls():
    codes, scales = kv8_empty(4, 2, 64, 16, "int8", DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    ops.kv8_write(torch.zeros(0, 2, 64, device=DEV), torch.zeros(0, 2, 64, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), codes, scales)
    assert ops.attention_decode_kv8(torch.zeros(0, 2, 64, device=DEV), codes, scales, torch.zeros(0, 3, **i32), torch.zeros(0, **i32)).shape == (0, 2, 64)
    p = ops.kv8_plan(torch.zeros(0, 3, **i32), torch.zeros(0, **i32), torch.zeros(0, **i32), torch.arange(4, **i32), torch.full((1,), 4, **i32), 16, 3)
    assert p.slots.tolist() == [-1] * 3 and int(p.free_count) == 4
    z = torch.zeros(0, 9, device=DEV, requires_grad=True)
    got = ops.token_logprobs(z, torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    got.logprob.sum().backward()
    assert got.top_ids.shape == (0, 2) and z.grad.shape == (0, 9)


def step(s):
    """One decoding step of one layer: plan, write, attend, score."""
    p = ops.kv8_plan(s["table"], s["lens"], s["new"], s["free"], s["count"], 16, s["k"].shape[0])
    ops.kv8_write(s["k"], s["v"], p.slots, s["codes"], s["scales"])
    o = ops.attention_decode_kv8(s["q"], s["codes"], s["scales"], s["table"], p.lens)
    got = ops.token_logprobs(o.flatten(1), s["ids"], top_k=4)
    s["lens"].copy_(p.lens)
    s["count"].copy_(p.free_count)
    return [p.slots, o, got.logprob, got.entropy, got.top_ids]


def step_state(seed, n=5):
    g = torch.Generator().manual_seed(seed)
    codes, scales = kv8_empty(60, 2, 64, 16, "e4m3", DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    return dict(table=torch.full((n, 12), -1, **i32), lens=torch.zeros(n, **i32), new=torch.ones(n, **i32),
                free=torch.randperm(60, generator=g).to(**i32), count=torch.full((1,), 60, **i32), codes=codes, scales=scales,
                q=torch.randn(n, 4, 64, generator=g).to(DEV), k=torch.randn(n, 2, 64, generator=g).to(DEV),
                v=torch.randn(n, 2, 64, generator=g).to(DEV), ids=torch.randint(0, 256, (n,), generator=g).to(DEV))


def test_steps_captured_in_two_graphs_equal_eager_steps():
    """Two captured decoding steps replayed in turn on two streams (their workspaces are their own), against eager steps."""
    eager, graphed = [step_state(i) for i in range(2)], [step_state(i) for i in range(2)]
    side = [torch.cuda.Stream() for _ in range(2)]
    for st in graphed:                                                        # warm-up on copies of the state
        step({k: x.clone() for k, x in st.items()})
    torch.cuda.synchronize()
    graphs = []
    for st in graphed:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(st)
        graphs.append((gr, out))
    for i in range(40):
        for st in graphed + eager:
            st["k"].mul_(1.01)
        torch.cuda.synchronize()
        for (gr, _), s in zip(graphs, side):
            with torch.cuda.stream(s):
                gr.replay()
        want = [step(st) for st in eager]
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b), i
    for a, b in zip(graphed, eager):
        assert torch.equal(a["codes"].view(torch.int8), b["codes"].view(torch.int8)) and torch.equal(a["scales"], b["scales"])
        assert a["lens"].tolist() == [40] * 5 and a["count"].tolist() == b["count"].tolist()


def test_steps_of_a_batch_follow_exact_attention():
    """Steps through plan, write and attention with requests that come and go, against attention on the cached values."""
    torch.manual_seed(2)
    bs, H, D, N, M = 16, 2, 64, 4, 8
    codes, scales = kv8_empty(20, H, D, bs, "int8", DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    table, lens = torch.full((N, M), -1, **i32), torch.zeros(N, **i32)
    free, count = torch.arange(20, **i32), torch.full((1,), 20, **i32)
    steps = [([40, 3, 0, 17], None), ([1, 1, 1, 1], None), ([1, 1, 1, 1], [False, False, False, True]), ([1, 1, 0, 60], None),
             ([1, 1, 1, 1], [True, False, False, False]), ([90, 1, 1, 1], None), ([1, 1, 1, 1], None)]
    for new, gone in steps:
        p = ops.kv8_plan(table, lens, torch.tensor(new, **i32), free, count, bs, sum(new),
                         release=torch.tensor(gone, device=DEV) if gone else None)
        lens, count = p.lens, p.free_count
        k, v = torch.randn(sum(new), H, D, device=DEV), torch.randn(sum(new), H, D, device=DEV)
        ops.kv8_write(k, v, p.slots, codes, scales)
        q = torch.randn(N, 2 * H, D, device=DEV)
        plain.check_attend(ops.attention_decode_kv8(q, codes, scales, table, lens), q, codes, scales, table, lens, D ** -0.5)
        used = [b for n in range(N) for b in table[n, :-(-int(lens[n]) // bs)].tolist()]
        left = free[:int(count)].tolist()
        assert sorted(used + left) == list(range(20))                         # every block has one owner


def test_tensors_used_on_a_side_stream():
    c = attend_case(9, "e4m3", 4, 2, 64, 16, [300, 20], torch.bfloat16)
    want = ops.attention_decode_kv8(*c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(50):
            got = ops.attention_decode_kv8(*c)
            junk = torch.full((1 << 20,), float("nan"), device=DEV)           # takes freed workspaces
            del junk
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_tensors_on_another_device_than_the_current_one():
    c = [x.to("cuda:1") for x in attend_case(9, "int8", 4, 2, 64, 16, [300, 20], torch.bfloat16)]
    got = ops.attention_decode_kv8(*c)
    assert got.device.index == 1
    plain.check_attend(got, *c, 64 ** -0.5)


def test_captured_gradient():
    """A forward and backward pass in a CUDA graph, replayed on new values. (No eager graph of the same leaf lives during the capture:
    torch would tie the leaf's gradient to that graph's stream and refuse the capture, for any operator.)"""
    z = torch.randn(6, 500, device=DEV, requires_grad=True)
    ids = torch.arange(6, device=DEV)

    def grad():
        got = ops.token_logprobs(z, ids)
        return torch.autograd.grad(got.logprob.sum() + got.entropy.sum(), z)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        grad()
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        d = grad()
    for _ in range(3):
        with torch.no_grad():
            z.mul_(-1.5)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(d, grad())


def _in_a_thread(fn):
    import threading
    got = []

    def run():
        try:
            got.append(fn())
        except BaseException as e:                                            # noqa: BLE001
            got.append(e)
    t = threading.Thread(target=run)
    t.start()
    t.join(timeout=120)
    assert got, "the thread did not come back"
    if isinstance(got[0], BaseException):
        raise got[0]
    return got[0]


def test_first_call_of_a_thread_may_be_captured():
    """A thread whose first calls stand inside a capture (nothing of the thread has touched the device before)."""
    c = attend_case(11, "int8", 4, 2, 64, 16, [90, 5], torch.bfloat16)
    z, ids = torch.randn(3, 900, device=DEV), torch.arange(3, device=DEV)
    st = step_state(5)
    want, lp = ops.attention_decode_kv8(*c), ops.token_logprobs(z, ids, top_k=2)
    ref = step({k: x.clone() for k, x in st.items()})
    torch.cuda.synchronize()

    def run():
        s, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            a, b = ops.attention_decode_kv8(*c), ops.token_logprobs(z, ids, top_k=2)
            d = step(st)
        gr.replay()
        torch.cuda.synchronize()
        return a, b, d
    a, b, d = _in_a_thread(run)
    assert torch.equal(a, want) and torch.equal(b.logprob, lp.logprob) and torch.equal(b.top_ids, lp.top_ids)
    for x, y in zip(d, ref):
        assert torch.equal(x, y)


def test_two_threads_on_two_streams():
    import threading
    cases = [attend_case(20 + i, "e4m3", 4, 2, 128, 64, [700 + i, 3, 0, 250], torch.bfloat16) for i in range(2)]
    want = [ops.attention_decode_kv8(*c) for c in cases]
    zs = [torch.randn(5, 40000, device=DEV) for _ in range(2)]
    ids = torch.zeros(5, dtype=torch.int64, device=DEV)
    scores = [ops.token_logprobs(z, ids, top_k=4) for z in zs]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(60):
                a, b = ops.attention_decode_kv8(*cases[i]), ops.token_logprobs(zs[i], ids, top_k=4)
                if not (torch.equal(a, want[i]) and torch.equal(b.logprob, scores[i].logprob) and torch.equal(b.top_ids, scores[i].top_ids)):
                    bad.append(i)
    ts = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(timeout=120)
    assert not bad


def test_more_requests_than_workers_and_a_wide_table():
    lens = [(i * 7) % 23 for i in range(5000)]
    q, codes, scales, table, ln = attend_case(30, "int8", 2, 1, 64, 16, [1], torch.float32)
    codes, scales, _ = cache_case(31, "int8", 1, 64, 16, 40)
    codes, scales = codes.to(DEV), scales.to(DEV)
    g = torch.Generator().manual_seed(1)
    table = torch.randint(0, 40, (5000, 300), generator=g).to(torch.int32).to(DEV)      # shared blocks, width far beyond the lengths
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn(5000, 2, 64, generator=g).to(DEV)
    got = ops.attention_decode_kv8(q, codes, scales, table, ln)
    pick = [0, 1, 2, 3, 1776, 2500, 4998, 4999]
    plain.check_attend(got[pick], q[pick], codes, scales, table[pick], ln[pick], 64 ** -0.5)
    assert not got[ln == 0].any()
    one = torch.cat([ops.attention_decode_kv8(q[i:i + 50], codes, scales, table[i:i + 50], ln[i:i + 50]) for i in range(0, 5000, 50)])
    assert float((one - got).abs().max()) < 1e-5 * float(got.abs().max())


def test_a_block_of_zeros_beside_large_values():
    """Scales from 2^-100 (zeros) to 2^90 in one sequence, in one warp and joined over many."""
    for lens in ([40], [6000]):
        q, codes, scales, table, ln = attend_case(40, "e4m3", 1, 1, 64, 16, lens, torch.float32)
        codes[1, int(table[0, 1])] = 0
        scales[1, int(table[0, 1])] = 2.0 ** -100
        scales[1, int(table[0, 0])] = 2.0 ** 90
        plain.check_attend(ops.attention_decode_kv8(q, codes, scales, table, ln), q, codes, scales, table, ln, 64 ** -0.5)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,heads", [(64, 4), (128, 4), (64, 8), (128, 8)])
@pytest.mark.parametrize("sink_scale", [0, 4])
def test_attention_of_a_sink_and_a_flat_tail(kind, D, heads, sink_scale):
    """One strong token whose value is zero before thousands of equal weak ones: the output is the tail's share, from 2^-8 to 2^-38 of
    the strong token's weight each. Far more units than warps (one table row for all), so that a warp holds whole units; queries of
    one channel, positive values, so that every bound is relative. ``sink_scale``: the strong token's block has a value scale of
    2^4 times the others'."""
    L, bs, N = 8192, 64, 4 * 12 * 148
    g = torch.Generator().manual_seed(D + heads)
    codes, scales = kv8_empty(L // bs, 1, D, bs, kind, DEV)
    keys, values = torch.zeros(L, D), torch.randint(1, 15, (L, D), generator=g).float()
    keys[0, 0], values[0] = 64.0, 0.0                                          # whole numbers below 16 and 64 are codes of both types
    values[1:bs] = 0.0                                                         # (the strong token's block holds no other value)
    for i, x in enumerate((keys, values)):
        codes[i, :, 0] = x.view(-1, bs, D).to(codes.dtype).to(DEV)
    scales.fill_(2.0 ** -6)
    scales[1, 0] *= 2.0 ** sink_scale
    offsets = torch.tensor([8.0, 17.0, 21.0, 25.05, 12.0, 19.5, 30.0, 38.0])[:heads]
    q = torch.zeros(heads, D)
    q[:, 0] = offsets / (math.log2(math.e) * D ** -0.5)                        # the strong token's score: key 64 * 2^-6 = 1
    table = torch.arange(L // bs, dtype=torch.int32, device=DEV)[None].expand(N, -1)
    got = ops.attention_decode_kv8(q.to(DEV).expand(N, -1, -1), codes, scales, table, torch.full((N,), L, dtype=torch.int32, device=DEV))
    s = q.double()[:, :1] * (keys.double()[:, 0] * 2.0 ** -6) * D ** -0.5
    p = torch.exp(s - s.amax(1, keepdim=True))
    want = (p / p.sum(1, keepdim=True)) @ (values.double() * 2.0 ** -6)
    A = float(offsets.max())
    # a score: the query's two terms 2^-23, its sum and the factors of the scale eight roundings, the exponential's argument and value;
    # then the split of the probabilities (2^-21), sums of the tokens, the division. All terms are positive: relative.
    rel = 2 * math.log(2) * (A * 16 * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -20 + (L / 8 + 64) * 2.0 ** -24
    # and half the last step of a probability's two terms, 2^-40 of the largest p * value scale, for every token's code
    tol = want * rel + L * 2.0 ** -40 * 2.0 ** (sink_scale - 6) * 14
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), ((off / want).amax((0, 2)), (off / tol).amax((0, 2)))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,heads", [(64, 2), (128, 6)])
@pytest.mark.parametrize("outlier", [2.0 ** 8, 2.0 ** 14, 2.0 ** 20, 2.0 ** 127])
def test_attention_of_queries_with_an_outlier_channel(kind, D, heads, outlier):
    """A channel of the query that is larger than the others by far, where the keys have nothing."""
    q, codes, scales, table, lens = attend_case(41, kind, heads, 1, D, 16, [300, 33], torch.float32)
    codes[0, ..., 3] = 0
    if outlier == 2.0 ** 127:
        q *= 2.0 ** 108                                                       # (the largest exponent; keys to match)
        scales[0] *= 2.0 ** -108
    q[..., 3] = 1.9 * outlier
    got = ops.attention_decode_kv8(q, codes, scales, table, lens)
    ref, bound = plain.attend(q, codes, scales, table.cpu(), lens.cpu(), D ** -0.5)
    used = [table[n, j] for n in range(2) for j in range(-(-int(lens[n]) // 16))]
    keys = (codes[0].float() * scales[0][..., None, None])[torch.stack(used).long()]
    # a query's element is off by 2^-39 of the row's largest at most: so much for every key channel; both ways in the exponent
    extra = float(keys.abs().sum(-1).max()) * 1.9 * outlier * 2.0 ** -39 * D ** -0.5
    values = (codes[1].float() * scales[1][..., None, None]).abs().max()
    tol = bound * (1 + 2.0 ** -24) + 2 * extra * float(values) + np.abs(ref) * 2.0 ** -24
    assert (np.abs(got.cpu().double().numpy() - ref) <= tol).all(), float((np.abs(got.cpu().double().numpy() - ref) / tol).max())
