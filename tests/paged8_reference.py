"""The 8-bit paged cache from its definitions: tables and appends step by step in Python, attention in 64 bits."""

import math

import numpy as np
import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def extend(table, lens, new, free, pool, bs, max_tokens):
    """numpy / lists in, new ones out: (table, slots, starts, lens, pool)."""
    table = table.copy()
    left, missed = min(max(int(pool[0]), 0), len(free)), max(int(pool[1]), 0)
    slots, starts, after = [], [0], []
    for i, (L, N) in enumerate(zip(lens, new)):
        L, asked = max(int(L), 0), max(int(N), 0)
        N = min(asked, max_tokens - len(slots))
        pages = min(-(-L // bs), table.shape[1])
        while pages < min(-(-(L + N) // bs), table.shape[1]) and left > 0:
            left -= 1
            table[i, pages] = free[left]
            pages += 1
        can = min(N, max(0, pages * bs - L))
        slots += [int(table[i, p // bs]) * bs + p % bs if table[i, p // bs] >= 0 else -1 for p in range(L, L + can)]
        slots += [-1] * (N - can)
        missed += asked - can
        starts.append(len(slots))
        after.append(L + can)
    return table, slots + [-1] * (max_tokens - len(slots)), starts, after, [left, min(missed, 2 ** 31 - 1)]      # a 32-bit count


def shrink(table, lens, keep, free, pool, bs):
    """(lens, free, pool) after the pages behind the kept tokens went back."""
    free, left = list(free), int(pool[0])
    back, after = [], []
    for i, (L, K) in enumerate(zip(lens, keep)):
        L = max(int(L), 0)
        K = min(max(int(K), 0), L)
        w = table.shape[1]
        back += [int(table[i, j]) for j in range(min(-(-K // bs), w), min(-(-L // bs), w))]
        after.append(K)
    for k, page in enumerate(back):
        at = left + len(back) - 1 - k
        if at < len(free):
            free[at] = page
    return after, free, [min(left + len(back), len(free)), int(pool[1])]


def rounded(y, dtype):
    """y (fp64 numpy) as the nearest code, ties to even."""
    if dtype == torch.int8:
        return np.clip(np.rint(y), -127, 127)
    _, e = np.frexp(y)
    unit = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.clip(np.rint(y / unit) * unit, -448, 448)


def append(x, codes, scales, slots, bs, dtype):
    """x (T, H, d), codes (blocks, H, bs, d) and scales (blocks, H), all fp64 numpy: runs one by one, in place."""
    runs = []
    for t, s in enumerate(slots):
        if s < 0 or s >= codes.shape[0] * bs:
            continue
        if runs and runs[-1][0] + runs[-1][1] == t and slots[t - 1] + 1 == s and s % bs:
            runs[-1][1] += 1
        else:
            runs.append([t, 1])
    for t, n in runs:
        page, at = divmod(int(slots[t]), bs)
        for h in range(codes.shape[1]):
            mine = x[t:t + n, h]
            top = np.abs(mine).max()
            new = math.nan if not np.isfinite(mine).all() else 0.0 if top == 0 else 2.0 ** max(-120, math.ceil(math.log2(top / TOP[dtype])))
            old = scales[page, h] if at else 0.0
            s = math.nan if math.isnan(new) or math.isnan(old) else max(new, old)
            if s > 0 and old != s and at:
                codes[page, h, :at] = rounded(codes[page, h, :at] * (old / s), dtype)
            codes[page, h, at:at + n] = rounded(mine / s, dtype) if s > 0 else 0
            scales[page, h] = s


def attention(q, pages, table, lens, scale, causal, starts=None):
    """(exact, bound) in 64 bits: `bound` is how far a result may be off, from the arithmetic:

    scores   fp32 sums of exact products of 16-bit queries (fp32 queries: 2^-22 of the products besides) over d / 16 steps, each truncating
             at 2^-23 of what has been summed, so |error| <= (2^-22 + (d / 16 + 2) 2^-23) scale sum |q k| in natural units, twice (numerator, denominator)
    weights  base-2 exponentials, 2^-20 with their arguments' rounding; with 16-bit queries rounded to fp16 once, 2^-11,
             besides 2^-25 (half of fp16's least step) where the largest weight times its page's scale is at least 1/2, so
             2^-24 max(p s) sum |code|; as hi + lo the largest is at least 2^9: 2^-34 max(p s) sum |code|
    sums     fp32, 2^-23 a step of 16 tokens and its two terms in each of the partial sums
    store    half a step of the type: eps / 2 (and of fp16's subnormal numbers, 2^-25)"""
    k_codes, v_codes, k_scales, v_scales = pages
    dtype, nb, bs, d, H = k_codes.dtype, k_codes.shape[0], k_codes.shape[2], k_codes.shape[3], k_codes.shape[1]
    flat = lambda c: c.contiguous().view(torch.uint8)      # noqa: E731
    kb, vb = flat(k_codes), flat(v_codes)
    exact, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    low = q.dtype != torch.float32
    half = torch.finfo(q.dtype).eps / 2
    for i in range(table.shape[0]):
        n = int(min(max(int(lens[i]), 0), table.shape[1] * bs))
        x = q[i].transpose(0, 1) if starts is None else q[starts[i]:starts[i + 1]]            # (Q, Hq, d)
        Q, G = x.shape[0], x.shape[1] // H
        if Q == 0:
            continue
        ids = table[i, :-(-n // bs)].long()
        good = (ids >= 0) & (ids < nb)
        at = torch.where(good, ids, torch.zeros_like(ids))
        known = good.repeat_interleave(bs)[:n]
        hide = torch.zeros(Q, n, dtype=torch.bool, device=q.device)
        if causal:
            hide = torch.ones(Q, n, dtype=torch.bool, device=q.device).triu(n - Q + 1)
        hide = hide | ~known[None]
        for h in range(H):
            K = (kb[at, h].view(dtype).double() * k_scales[at, h].double()[:, None, None]).reshape(-1, d)[:n]
            V = (vb[at, h].view(dtype).double() * v_scales[at, h].double()[:, None, None]).reshape(-1, d)[:n]
            y = x[:, h * G:(h + 1) * G].double().transpose(0, 1)                              # (G, Q, d)
            t = (y @ K.T * scale).masked_fill(hide[None], -math.inf)
            off = (y.abs() @ K.abs().T * abs(scale)).masked_fill(hide[None], 0).amax(-1, keepdim=True) if n else torch.zeros(G, Q, 1, device=q.device)
            # NaN of a token that a row does not see is not the row's
            w = torch.nan_to_num(torch.softmax(t, -1), nan=0.0) if not K.isnan().any() else torch.softmax(t, -1)
            w = torch.where(hide.all(-1)[None, :, None], torch.zeros_like(w), w)
            Vc = torch.nan_to_num(V, nan=0.0)
            bad = (~hide).double() @ V.isnan().double()                                       # (Q, d)
            o = torch.where(bad[None] > 0, math.nan, w @ Vc)
            a = torch.nan_to_num(w) @ Vc.abs()
            score = off * (2.0 ** -22 + (d / 16 + 2) * 2.0 ** -23)
            rel = 2 * score + 2.0 ** -19 + (n / 16 * 2 + 8) * 2.0 ** -23 + (2.0 ** -11 if low else 0.0)
            sv = torch.nan_to_num(v_scales[at, h].double()).repeat_interleave(bs)[:n]
            codes = vb[at, h].view(dtype).double().reshape(-1, d)[:n].nan_to_num().abs().sum(0)
            most = (torch.nan_to_num(w) * sv).amax(-1, keepdim=True) if n else torch.zeros(G, Q, 1, device=q.device)
            e = a * rel + half * o.abs() + (2.0 ** -24 if low else 2.0 ** -34) * most * codes + (2.0 ** -25 if low else 0)
            o, e = o.transpose(0, 1), e.transpose(0, 1)                                       # (Q, G, d)
            if starts is None:
                exact[i, h * G:(h + 1) * G], bound[i, h * G:(h + 1) * G] = o.transpose(0, 1), e.transpose(0, 1)
            else:
                exact[starts[i]:starts[i + 1], h * G:(h + 1) * G] = o
                bound[starts[i]:starts[i + 1], h * G:(h + 1) * G] = e
    return exact, bound


def random_pages(g, total, H, bs, d, dtype, layout="hnd", spread=0.5, pow2=True):
    """Codes and scales of `total` pages: normal vectors with a large channel, scales spread by 2^(spread * N(0, 1))."""
    out = []
    for _ in range(2):
        x = torch.randn(total, H, bs, d, generator=g, device=g.device)
        x[..., ::29] *= 6
        s = x.abs().amax((2, 3)) / TOP[dtype]
        y = (x / s[..., None, None]).clamp(-TOP[dtype], TOP[dtype])
        codes = y.round().to(torch.int8) if dtype == torch.int8 else y.to(dtype)
        s = s * torch.exp2(spread * torch.randn(total, H, generator=g, device=g.device))
        if pow2:
            s = torch.exp2(torch.ceil(torch.log2(s)))
        if layout == "nhd":
            codes = codes.view(torch.uint8).transpose(1, 2).contiguous().view(dtype).transpose(1, 2)
        out.append((codes, s))
    (k, ks), (v, vs) = out
    return k, v, ks, vs


def random_tables(lens, bs, total, seed):
    """A block table of distinct pages of `total` in random order."""
    need = [-(-n // bs) for n in lens]
    order = np.random.RandomState(seed).permutation(total)
    table = np.full((len(lens), max(1, max(need))), 0, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table)
