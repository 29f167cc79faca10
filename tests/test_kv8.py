"""8-bit paged key / value cache and per-token scores on the CPU: the oracles against plain 64-bit statements, and the refusals."""
import math
import random

import numpy as np
import pytest
import torch

import kv8_plain as plain
from hippolm_b200 import ops
from hippolm_b200.ops.kv8 import kv8_empty


def make_plan_case(seed, n, bs, M, hi, new_hi, spare, release, device="cpu"):
    r = random.Random(seed)
    lens = [r.randint(0, min(hi, M * bs)) for _ in range(n)]
    new = [r.randint(0, new_hi) for _ in range(n)]
    counts = [-(-a // bs) for a in lens]
    pool = list(range(sum(counts) + spare))
    r.shuffle(pool)
    table = [[-1] * M for _ in range(n)]
    at = 0
    for i, c in enumerate(counts):
        table[i][:c] = pool[at:at + c]
        at += c
    free = pool[at:] + [-7] * at
    i32 = dict(dtype=torch.int32, device=device)
    rel = torch.tensor([r.random() < 0.3 for _ in range(n)], device=device) if release else None
    return dict(table=torch.tensor(table, **i32), lens=torch.tensor(lens, **i32), new_lens=torch.tensor(new, **i32),
                free_list=torch.tensor(free or [-7], **i32), free_count=torch.tensor([spare], **i32), block_size=bs,
                num_tokens=sum(new), release=rel)


def check_plan(c):
    want = plain.plan(c["table"], c["lens"], c["new_lens"], c["free_list"], c["free_count"], c["block_size"], c["num_tokens"], c["release"])
    before = {k: c[k].clone() for k in ("lens", "new_lens", "free_count")}
    for _ in range(2):                                          # a second call with the same lengths gives the same plan
        p = ops.kv8_plan(**c)
        got = [p.slots, p.lens, p.free_count, p.served, c["table"], c["free_list"]]
        for name, g, w in zip(("slots", "lens", "count", "served", "table", "free"), got, want):
            assert g.tolist() == w, name
    for k, x in before.items():
        assert torch.equal(c[k], x), k


PLAN_CASES = [(1, 16, 4, 60, 3, 1, False), (5, 16, 8, 100, 20, 12, False), (9, 32, 5, 160, 40, 6, True), (33, 64, 3, 192, 70, 50, True),
              (7, 16, 6, 96, 9, 0, False), (40, 16, 12, 190, 1, 7, True), (3, 64, 1, 0, 64, 2, False)]


@pytest.mark.parametrize("n,bs,M,hi,new_hi,spare,release", PLAN_CASES)
def test_plan_matches_lists(n, bs, M, hi, new_hi, spare, release):
    for seed in range(4):
        check_plan(make_plan_case(seed, n, bs, M, hi, new_hi, spare, release))


def test_plan_rows_behind_the_tokens_and_short_buffers():
    c = make_plan_case(3, 4, 16, 8, 50, 9, 20, False)
    total = c["num_tokens"]
    for tokens in (total + 5, max(total - 3, 0), 0):
        check_plan(dict(c, num_tokens=tokens, table=c["table"].clone(), free_list=c["free_list"].clone()))


def cache_case(seed, kind, H, D, bs, nb, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    codes, scales = kv8_empty(nb, H, D, bs, kind, device)
    x = torch.randn(codes.shape, generator=g) * torch.exp2(torch.randint(-3, 4, codes.shape[:3], generator=g).float())[..., None, None]
    amax = x.abs().amax((-1, -2))
    s = torch.tensor([plain.scale_for(float(a), kind) for a in amax.flatten()]).view(amax.shape)
    scales.copy_(s)
    codes.copy_(torch.tensor(plain.round_code((x / s[..., None, None]).double().numpy(), kind)).float().to(plain.DT[kind]))
    return codes, scales, g


def runs_to_slots(runs, bs):
    """[(block, offset, length)] -> packed slots; block None: rows that are not stored."""
    out = []
    for b, off, ln in runs:
        out += [-1] * ln if b is None else [b * bs + off + i for i in range(ln)]
    return torch.tensor(out, dtype=torch.int64)


WRITE_RUNS = [
    lambda bs: [(2, 0, 1)],
    lambda bs: [(0, bs - 1, 1), (3, 5, 1), (None, 0, 2), (4, 0, 1), (1, 1, 1)],
    lambda bs: [(0, 3, bs - 3), (1, 0, bs), (5, 0, 7), (2, 9, 4)],
    lambda bs: [(5, 0, bs), (6, 0, bs), (7, 0, bs), (3, 1, bs - 1), (None, 0, 3), (0, 0, 1), (1, 2, 3), (2, 0, bs)],
]


def check_write(k, v, slots, codes, scales, kind, write=None):
    want_c, want_s = plain.write(k, v, slots, codes, scales, kind)
    (write or ops.kv8_write)(k, v, slots, codes, scales)
    assert np.array_equal(scales.cpu().double().numpy(), want_s, equal_nan=True)
    assert np.array_equal(plain.value_of(codes), want_c)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("runs", range(len(WRITE_RUNS)))
def test_write_matches_64_bits(kind, bs, runs):
    codes, scales, g = cache_case(runs, kind, 3, 8, bs, 8)
    slots = runs_to_slots(WRITE_RUNS[runs](bs), bs)
    k, v = (torch.randn(slots.numel(), 3, 8, generator=g) * 20 ** float(i) for i in range(2))
    check_write(k, v, slots, codes, scales, kind)


def test_write_poison_zeros_and_far_slots():
    for kind in ("int8", "e4m3"):
        codes, scales, g = cache_case(0, kind, 2, 8, 16, 4)
        k, v = torch.randn(6, 2, 8, generator=g), torch.randn(6, 2, 8, generator=g)
        k[0, 1, 3], v[2, 0, 0], k[4] = math.nan, math.inf, 0.0
        slots = torch.tensor([5, 16, 17, 4 * 16, 2 * 16, 1 << 40])
        check_write(k, v, slots, codes, scales, kind)
        assert torch.isnan(scales[0, 0, 1]) and torch.isnan(scales[1, 1, 0]) and scales[0, 2, 0] == 2.0 ** -100
        # a poisoned block stays poisoned while tokens join it, and is clean again once it is filled from its start
        check_write(k[5:], v[5:], torch.tensor([18]), codes, scales, kind)
        assert torch.isnan(scales[1, 1, 0])
        check_write(k[5:], v[5:], torch.tensor([16]), codes, scales, kind)
        assert not torch.isnan(scales[1, 1, 0])


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("Hq,H,lens", [(2, 2, [1, 0, 17, 40]), (6, 2, [48, 3, 5, 16]), (9, 1, [30, 31, 32, 33])])
def test_attention_matches_64_bits(kind, Hq, H, lens):
    codes, scales, g = cache_case(7, kind, H, 8, 16, 16)
    table = torch.randperm(16, generator=g)[:12].view(4, 3).to(torch.int32)
    lens = torch.tensor(lens, dtype=torch.int32)
    q = torch.randn(4, Hq, 8, generator=g)
    plain.check_attend(ops.attention_decode_kv8(q, codes, scales, table, lens), q, codes, scales, table, lens, 8 ** -0.5)
    table[2, 1], table[3, 0] = -1, 99                           # blocks outside the cache count as not there
    got = ops.attention_decode_kv8(q, codes, scales, table, lens, scale=0.3)
    plain.check_attend(got, q, codes, scales, table, lens, 0.3)


def test_cached_step_follows_attention_on_exact_values():
    """plan -> write -> attend, several steps, against attention on the unquantised values: within the codes' step."""
    torch.manual_seed(0)
    N, H, D, bs, M = 3, 2, 16, 16, 4
    for kind, rel in (("int8", 2.0 ** -6), ("e4m3", 2.0 ** -4)):          # int8: the scale may be twice the largest value / 127
        codes, scales = kv8_empty(N * M, H, D, bs, kind)
        table = torch.full((N, M), -1, dtype=torch.int32)
        lens = torch.zeros(N, dtype=torch.int32)
        free, count = torch.arange(N * M, dtype=torch.int32), torch.tensor([N * M], dtype=torch.int32)
        hist = [[] for _ in range(N)]
        for new in ([17, 1, 30], [1, 1, 1], [1, 1, 1], [3, 0, 1]):
            new_t = torch.tensor(new, dtype=torch.int32)
            p = ops.kv8_plan(table, lens, new_t, free, count, bs, sum(new))
            assert p.served.all()
            lens, count = p.lens, p.free_count
            k, v = torch.randn(sum(new), H, D), torch.randn(sum(new), H, D)
            ops.kv8_write(k, v, p.slots, codes, scales)
            for n in range(N):
                hist[n] += [(k[i], v[i]) for i in range(sum(new[:n]), sum(new[:n + 1]))]
            q = torch.randn(N, H, D)
            o = ops.attention_decode_kv8(q, codes, scales, table, lens)
            for n in range(N):
                kk, vv = torch.stack([a for a, _ in hist[n]]), torch.stack([b for _, b in hist[n]])
                ref = ops.attention_decode(q[n:n + 1], kk, vv)[0]
                # keys off by rel of the largest: scores by rel * |q|_1 max|k| / 4 (the softmax scale); values by rel of the largest
                ds = rel * float(q[n].abs().sum(-1).max() * kk.abs().max()) * D ** -0.5
                assert float((o[n] - ref).abs().max()) <= (2 * math.expm1(min(ds, 3.0)) + rel) * float(vv.abs().max())


SCORE_ROWS = [(1, 1, 1), (3, 2, 2), (5, 33, 20), (2, 600, 5), (4, 1031, 32)]


@pytest.mark.parametrize("T,V,top", SCORE_ROWS)
def test_scores_match_64_bits(T, V, top):
    g = torch.Generator().manual_seed(V)
    z = (torch.randn(T, V, generator=g) * 3).bfloat16().float()           # rounded: many equal logits
    ids = torch.randint(0, V, (T,), generator=g)
    ids[T // 2] = -100
    got = ops.token_logprobs(z, ids, top_k=top)
    lp, ent, tv, ti = plain.scores(z, ids, top)
    assert np.allclose(got.logprob.numpy(), lp, rtol=2e-6, atol=4e-6) and np.allclose(got.entropy.numpy(), ent, rtol=2e-6, atol=4e-6)
    assert got.top_ids.numpy().tolist() == ti.tolist() and np.allclose(got.top_logprobs.numpy(), tv, rtol=2e-6, atol=4e-6)


def special_rows(V):
    lo = torch.finfo(torch.float32).min
    z = torch.zeros(8, V)
    z[0] = -math.inf
    z[1, 1:] = -math.inf
    z[2] = lo
    z[3] = lo; z[3, V // 2] = 5.0
    z[4, 3] = math.nan
    z[5, 2] = math.inf
    z[6] = -0.0; z[6, 5] = 0.0
    z[7] = torch.linspace(-50, 50, V)
    return z, torch.tensor([0, 0, 3, V // 2, 1, 2, V, V - 1])


def check_special(device="cpu"):
    V = 40
    z, ids = special_rows(V)
    got = ops.token_logprobs(z.to(device), ids.to(device), top_k=6)
    lp, ent, tv, ti = plain.scores(z, ids, 6)
    assert np.allclose(got.logprob.cpu().numpy(), lp, rtol=1e-5, atol=1e-5, equal_nan=True)
    assert np.allclose(got.entropy.cpu().numpy(), ent, rtol=1e-5, atol=1e-5, equal_nan=True)
    assert got.top_ids.cpu().tolist() == ti.tolist()
    assert np.allclose(got.top_logprobs.cpu().numpy(), tv, rtol=1e-5, atol=1e-5, equal_nan=True)


def test_scores_of_masked_and_broken_rows():
    check_special()


def test_score_gradient_formula_and_differences():
    g = torch.Generator().manual_seed(1)
    z = torch.randn(5, 13, generator=g, dtype=torch.float32)
    z[1, 4], z[2] = -math.inf, -math.inf
    ids = torch.tensor([3, 0, 1, -100, 12])
    a, b = torch.randn(5, generator=g), torch.randn(5, generator=g)
    z.requires_grad_(True)
    got = ops.token_logprobs(z, ids)
    (d,) = torch.autograd.grad((got.logprob, got.entropy), z, (a, b))
    assert torch.isfinite(d).all() and not d[2].any()
    base = z.detach().double()
    for t, v in ((0, 3), (0, 7), (3, 2), (4, 12), (1, 5)):
        num = 0.0
        for sgn in (1, -1):
            zz = base.clone()
            zz[t, v] += sgn * 1e-5
            lp, ent, _, _ = plain.scores(zz, ids, 0)
            num += sgn * (float(a[t]) * lp[t] + float(b[t]) * ent[t])
        assert abs(num / 2e-5 - float(d[t, v])) < 1e-5


def test_rows_of_any_alignment_are_copied_to_16_bytes():
    from hippolm_b200.ops.kv8_cuda import _rows
    flat = torch.randn(4 * 2 * 64 + 8, dtype=torch.float32)
    for dt in (torch.float32, torch.bfloat16):
        for off in range(8):
            x = flat.to(dt)[off:off + 512].view(4, 2, 64)
            for y in (x, x.transpose(0, 1), x[:, :, ::2], flat.to(dt)[off:off + 4 * 2 * 63].view(4, 2, 63)[..., :62]):
                r = _rows(y)
                assert r.data_ptr() % 16 == 0 and torch.equal(r, y) and r.stride(2) == 1
                if r is y:
                    assert y.stride(0) * y.element_size() % 16 == 0 and y.stride(1) * y.element_size() % 16 == 0


def test_refusals():
    codes, scales = kv8_empty(4, 2, 8, 16, "int8")
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q, k, sl = torch.zeros(3, 2, 8), torch.zeros(5, 2, 8), torch.zeros(5, dtype=torch.int64)
    free, cnt = torch.arange(4, dtype=torch.int32), torch.tensor([4], dtype=torch.int32)
    bad = [
        lambda: kv8_empty(4, 2, 8, 24, "int8"),
        lambda: kv8_empty(4, 2, 8, 16, "fp8"),
        lambda: ops.kv8_write(k, k.half(), sl, codes, scales),
        lambda: ops.kv8_write(k.double(), k.double(), sl, codes, scales),
        lambda: ops.kv8_write(k[:, :1], k[:, :1], sl, codes, scales),
        lambda: ops.kv8_write(k, k, sl.int(), codes, scales),
        lambda: ops.kv8_write(k, k, sl[:4], codes, scales),
        lambda: ops.kv8_write(k, k, sl, codes.transpose(2, 3), scales),
        lambda: ops.kv8_write(k, k, sl, codes, scales.double()),
        lambda: ops.kv8_write(k, k, sl, torch.zeros(codes.numel() + 1, dtype=torch.int8)[1:].view(codes.shape), scales),
        lambda: ops.attention_decode_kv8(q[:2], codes, scales, table, lens),
        lambda: ops.attention_decode_kv8(q[:, :1], codes, scales, table, lens),
        lambda: ops.attention_decode_kv8(q, codes, scales, table.long(), lens),
        lambda: ops.attention_decode_kv8(q, codes, scales, table, lens.long()),
        lambda: ops.attention_decode_kv8(q, codes, scales[:, :3], table, lens),
        lambda: ops.kv8_plan(table, lens, lens[:2], free, cnt, 16, 3),
        lambda: ops.kv8_plan(table, lens, lens, free, cnt, 8, 3),
        lambda: ops.kv8_plan(table, lens, lens, free, cnt, 16, -1),
        lambda: ops.kv8_plan(table, lens, lens, free.long(), cnt, 16, 3),
        lambda: ops.kv8_plan(table, lens, lens, free, cnt, 16, 3, release=lens),
        lambda: ops.kv8_plan(table[:1].expand(3, 2), lens, lens, free, cnt, 16, 3),
        lambda: ops.token_logprobs(torch.zeros(2, 3, dtype=torch.float64), torch.zeros(2, dtype=torch.int64)),
        lambda: ops.token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32)),
        lambda: ops.token_logprobs(torch.zeros(2, 3), torch.zeros(3, dtype=torch.int64)),
        lambda: ops.token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64), top_k=4),
        lambda: ops.token_logprobs(torch.zeros(2, 90), torch.zeros(2, dtype=torch.int64), top_k=33),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_a_kernel_that_reads_anothers_workspace_runs_only_behind_it():
    """Calls of two kernels, the second of which follows indexes that the first one leaves: not launched where the first was refused."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(ops.__file__))), "csrc")
    for name, first, second in (("kv8_attention.cu", "kv8_attention_kernel<D, E4M3, SETS><<<", "cudaLaunchKernelEx("),
                                ("kv8.cu", "kv8_plan_kernel<<<", "kv8_slots_kernel<<<")):
        text = open(os.path.join(csrc, name)).read()
        between = text[text.index(first):text.index(second, text.index(first))]
        assert re.search(r"cudaGetLastError\(\)[^;]*;(?s:.*)\breturn\b", between), name
