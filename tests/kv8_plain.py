"""Plain 64-bit statements of the 8-bit cache operators and of the per-token scores, written from their definitions (numpy / python loops,
nothing of the package), and the bounds that the tests hold the kernels to."""
import math

import numpy as np
import torch

LARGEST = {"int8": 127.0, "e4m3": 448.0}
DT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def value_of(codes: torch.Tensor) -> np.ndarray:
    return codes.cpu().float().numpy().astype(np.float64)


def round_code(x: np.ndarray, kind: str) -> np.ndarray:
    """Nearest code value, ties to even: int8 whole numbers, e4m3 three bits behind the leading one down to 2^-9."""
    if kind == "int8":
        return np.rint(x)
    mag = np.maximum(np.abs(x), 2.0 ** -6)
    step = 2.0 ** (np.floor(np.log2(mag)) - 3)
    return np.rint(x / step) * step


def scale_for(amax: float, kind: str) -> float:
    e = -100
    while amax > LARGEST[kind] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def write(k, v, slots, codes, scales, kind):
    """-> (code values [2, nb, H, bs, D], scales) after the write; runs of a block taken together."""
    cv, sc = value_of(codes), scales.cpu().numpy().astype(np.float64)
    _, nb, H, bs, D = cv.shape
    sl = slots.cpu().tolist()
    for i, x in enumerate((k, v)):
        x = x.detach().cpu().double().numpy()
        blocks = {}
        for t, s in enumerate(sl):
            if 0 <= s < nb * bs:
                blocks.setdefault(s // bs, []).append((s % bs, t))
        for b, toks in blocks.items():
            first = min(o for o, _ in toks)
            for h in range(H):
                rows = np.stack([x[t, h] for _, t in toks])
                old = sc[i, b, h]
                if not np.isfinite(rows).all() or (first > 0 and math.isnan(old)):
                    sc[i, b, h] = math.nan
                    for o, t in toks:
                        cv[i, b, h, o] = 0.0
                    continue
                s = scale_for(float(np.abs(rows).max()), kind)
                if first > 0 and old > s:
                    s = old
                if first > 0 and old < s:
                    cv[i, b, h, :first] = round_code(cv[i, b, h, :first] * (old / s), kind)
                for o, t in toks:
                    cv[i, b, h, o] = round_code(x[t, h] / s, kind)
                sc[i, b, h] = s
    return cv, sc


def attend(q, codes, scales, table, lens, scale):
    """-> (out [N, Hq, D] float64, bound [N, Hq, 1]: how far fp32 sums and 21-bit splits may move the value before the final rounding)."""
    cv, sc = value_of(codes), scales.cpu().double().numpy()
    q = q.detach().cpu().double().numpy()
    N, Hq, D = q.shape
    _, nb, H, bs, _ = cv.shape
    out, bound = np.zeros((N, Hq, D)), np.zeros((N, Hq, 1))
    for n in range(N):
        length = min(max(int(lens[n]), 0), table.shape[1] * bs)
        at = [(int(table[n, j // bs]), j % bs) for j in range(length)]
        at = [(b, o) for b, o in at if 0 <= b < nb]
        if not at:
            continue
        b, o = np.array([a[0] for a in at]), np.array([a[1] for a in at])
        for g in range(Hq):
            h = g // (Hq // H)
            k = cv[0, b, h, o] * sc[0, b, h][:, None]
            v = cv[1, b, h, o] * sc[1, b, h][:, None]
            s = (k @ q[n, g]) * scale
            p = np.exp(s - s.max())
            out[n, g] = (p / p.sum()) @ v
            # scores in log2 units: sum of |products| A; the query keeps 21 bits, 2D fp32 additions, three roundings of the scale
            A = float((np.abs(k) @ np.abs(q[n, g])).max()) * abs(scale) * math.log2(math.e)
            err = A * (2.0 ** -21 + (2 * D + 8) * 2.0 ** -24) + 2.0 ** -21
            # probabilities off by a factor 2^err either way, their 21-bit split, fp32 sums over the tokens, the join's rescaling
            bound[n, g] = (2 * math.log(2) * err + 2.0 ** -20 + (length / 8 + 64) * 2.0 ** -24) * np.abs(v).max()
    return out, bound


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def check_attend(got, q, codes, scales, table, lens, scale):
    ref, bound = attend(q, codes, scales, table.cpu(), lens.cpu(), scale)
    g = got.detach().cpu().double().numpy()
    assert np.isfinite(g).all() or np.isnan(ref).any()
    nan = np.isnan(ref)
    assert np.array_equal(np.isnan(g), nan)
    off = np.abs(g - ref)[~nan]
    tol = (half_step(got.dtype) * (np.abs(ref) + bound) + bound)[~nan]
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25                                  # half a step of fp16's subnormals
    assert (off <= tol).all(), f"off by {float((off - tol).max())} beyond the bound"


def plan(table, lens, new, free, count, bs, tokens, release=None):
    """The plan by lists: -> (slots, lens, count, served, table, free) as python lists."""
    table, free = [list(map(int, r)) for r in table.tolist()], list(map(int, free.tolist()))
    M = len(table[0])
    lens = [min(max(int(x), 0), M * bs) for x in lens.tolist()]
    new = [max(int(x), 0) for x in new.tolist()]
    stack = free[:max(0, min(int(count), len(free)))]
    rel = [bool(x) for x in release.tolist()] if release is not None else [False] * len(lens)
    for n, r in enumerate(rel):
        if r:
            stack += table[n][:-(-lens[n] // bs)]
            lens[n] = 0
    stack = stack[:len(free)]
    mem = stack + free[len(stack):]                             # the list as it stands in memory: pops leave their entries
    cu, slots, served, blocked, end = [0], [-1] * tokens, [], False, 0
    for n in range(len(lens)):
        end += new[n]
        cu.append(end)
        if new[n] == 0:
            served.append(True)
            continue
        have, want = -(-lens[n] // bs), -(-(lens[n] + new[n]) // bs)
        ok = not rel[n] and want <= M and lens[n] + new[n] <= M * bs and end <= tokens
        if ok and want > have:
            if blocked or want - have > len(stack):
                ok, blocked = False, True
        served.append(ok)
        if not ok:
            continue
        for j in range(have, want):
            table[n][j] = stack.pop()
        for i in range(new[n]):
            p = lens[n] + i
            b = table[n][p // bs]
            slots[end - new[n] + i] = b * bs + p % bs if b >= 0 else -1
        lens[n] += new[n]
    return slots, lens, [len(stack)], served, table, mem


def scores(logits, ids, top):
    """float64 (logprob, entropy, top values, top ids), rows one at a time."""
    z = logits.detach().cpu().double().numpy()
    lp, ent, tv, ti = [], [], [], []
    for t in range(z.shape[0]):
        row, y = z[t], int(ids[t])
        inside = 0 <= y < row.size
        order = sorted(range(row.size), key=lambda i: (not math.isnan(row[i]), -row[i] if not math.isnan(row[i]) else 0, i)) if top else []
        if np.isneginf(row).all():
            lp.append(-math.inf if inside else 0.0); ent.append(0.0)
            tv.append([-math.inf] * top); ti.append(order[:top])
            continue
        with np.errstate(all="ignore"):
            d = row - row.max()
            lse = math.log(np.exp(d).sum()) if np.isfinite(row.max()) else math.nan
            logp = d - lse if np.isfinite(row.max()) else np.full(row.size, np.nan)
            p = np.exp(logp)
            lp.append(logp[y] if inside else 0.0)
            ent.append(-(p[p > 0] * logp[p > 0]).sum() if np.isfinite(row.max()) else math.nan)
        tv.append([logp[i] for i in order[:top]]); ti.append(order[:top])
    return np.array(lp), np.array(ent), np.array(tv).reshape(len(lp), top), np.array(ti, dtype=np.int64).reshape(len(lp), top)
