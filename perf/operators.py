"""Operators of the 8-bit paged cache: what is measured, and each operator in its plain form.

  extend     block tables and slot maps from request lengths: pages from a stack of free ones, a slot for each new token.
  append     keys and values quantised to 8 bits into their pages, a scale for each page and head.
  attention  queries over the pages: one token a sequence, whole prompts, or a ragged batch of both.
  step       the three of them in the order of a serving loop.

A case holds plain values only; `draw` gives more cases of the same ranges.  `prepare` makes the same tensors whoever uses
them; `run` is the plain form in elementary torch operations, or, where `own` is true, the framework's calls.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}
MOST_PAIRS = 2 * 32 * 4096 * 4096            # query rows x padded tokens of a prompt
MOST_TOKENS = 32 * 8 * 32768                 # tokens x KV heads of a cache


def listed():
    heads = {"kv_heads": 8, "q_heads": 32, "dim": 128}
    small = {"kv_heads": 4, "q_heads": 32, "dim": 64}
    return [
        # A serving step takes one token from each of 32 requests: their tables grow now and then by a page.
        {"name": "extend_32x1", "kind": "extend", "seqs": 32, "held": 16384, "new": 1, "ragged": True, "block": 16},
        # A server fills up: prompts of all lengths arrive for 512 requests at once.
        {"name": "extend_512_prompts", "kind": "extend", "seqs": 512, "held": 1000, "new": 1024, "ragged": True, "block": 16},
        # The new token of 32 requests goes to its page.
        {"name": "append_32x1", "kind": "append", "seqs": 32, "held": 1277, "new": 1, "ragged": False, "kv_heads": 8, "dim": 128,
         "block": 16, "codes": "e4m3", "dtype": "bf16", "layout": "hnd"},
        # Two long prompts go to their pages: bound by the bytes.
        {"name": "append_2x4096", "kind": "append", "seqs": 2, "held": 0, "new": 4096, "ragged": False, "kv_heads": 8, "dim": 128,
         "block": 16, "codes": "int8", "dtype": "bf16", "layout": "hnd"},
        # Interactive decode: one sequence with a short history; latency and launches count.
        {"name": "decode_1x1000", "kind": "attention", "seqs": 1, "tokens": 1000, "q_len": 1, "ragged": False, **heads,
         "block": 16, "codes": "e4m3", "dtype": "bf16", "layout": "hnd", "scales": "pow2"},
        # One layer of a decode step of a small model: head size 64, eight query heads a KV head, an odd length.
        {"name": "decode_8x1277_d64", "kind": "attention", "seqs": 8, "tokens": 1277, "q_len": 1, "ragged": False, **small,
         "block": 32, "codes": "int8", "dtype": "fp16", "layout": "nhd", "scales": "any"},
        # The benchmark's batch over a long cache: bound by the bytes of the pages.
        {"name": "decode_32x32768", "kind": "attention", "seqs": 32, "tokens": 32768, "q_len": 1, "ragged": False, **heads,
         "block": 16, "codes": "e4m3", "dtype": "bf16", "layout": "hnd", "scales": "pow2"},
        # A serving step of 32 requests of different lengths in fp32, four draft tokens each to be verified.
        {"name": "verify_32x4_16384_fp32", "kind": "attention", "seqs": 32, "tokens": 16384, "q_len": 4, "ragged": True, **heads,
         "block": 16, "codes": "int8", "dtype": "fp32", "layout": "hnd", "scales": "pow2"},
        # Two long prompts at the same layer shape: bound by the tensor cores.
        {"name": "prompt_2x4096", "kind": "attention", "seqs": 2, "tokens": 4096, "q_len": 4096, "ragged": False, **heads,
         "block": 16, "codes": "e4m3", "dtype": "bf16", "layout": "hnd", "scales": "pow2"},
        # A batch of prompts of the small model.
        {"name": "prompt_8x1024_d64", "kind": "attention", "seqs": 8, "tokens": 1024, "q_len": 1024, "ragged": False, **small,
         "block": 16, "codes": "int8", "dtype": "bf16", "layout": "nhd", "scales": "pow2"},
        # Steps of a loop that serves prompts and decodes together: 15 requests give a token, the last one a piece of its prompt.
        {"name": "step_16_chunk_512", "kind": "step", "seqs": 16, "held": 4096, "new": 512, **heads, "block": 16,
         "codes": "e4m3", "dtype": "bf16", "layout": "hnd"},
        # The same at a single token each.
        {"name": "step_32_decode", "kind": "step", "seqs": 32, "held": 1277, "new": 1, **heads, "block": 16, "codes": "e4m3",
         "dtype": "bf16", "layout": "nhd"},
    ]


# ---- more cases of the same ranges ----------------------------------------------------------------------------

def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["extend", "append", "attention", "attention", "attention", "step"])
    case = {"kind": kind, "seqs": _log_int(rng, 1, 512 if kind == "extend" else 64), "block": rng.choice([16, 16, 16, 32, 48, 64, 128])}
    if kind == "extend":
        case.update(held=_log_int(rng, 1, 16384), new=_log_int(rng, 1, 1024), ragged=rng.random() < 0.7)
        return case
    kv_heads, q_heads = rng.choice([(8, 32), (8, 8), (4, 32), (8, 64), (2, 8), (1, 16), (3, 12)])
    case.update(kv_heads=kv_heads, dim=rng.choice([128, 128, 64]), codes=rng.choice(["e4m3", "int8"]),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), layout=rng.choice(["hnd", "hnd", "nhd"]))
    if kind == "append":
        case.update(new=_log_int(rng, 1, 4096), held=_log_int(rng, 1, 4096), ragged=rng.random() < 0.5)
        case["seqs"] = max(1, min(case["seqs"], 2 * 4096 // case["new"]))
        return case
    case["q_heads"] = q_heads
    if kind == "step":
        case["held"] = _log_int(rng, 100, 4096)
        case["new"] = _log_int(rng, 1, 512)
        case["seqs"] = max(1, min(case["seqs"], 16 * 32 * 512 * 4608 // (q_heads * case["new"] * (case["held"] + case["new"]))))
        return case
    use = rng.choice(["decode", "decode", "verify", "prompt"])
    tokens = _log_int(rng, 16, 4096 if use == "prompt" else 32768)
    q_len = {"decode": 1, "verify": rng.randint(2, 8), "prompt": tokens if rng.random() < 0.7 else _log_int(rng, 9, max(9, tokens))}[use]
    limit = min(MOST_TOKENS // (kv_heads * tokens), MOST_PAIRS // (q_heads * q_len * tokens))
    if case["dtype"] == "fp32" and use == "prompt":
        limit //= 8
    case.update(tokens=tokens, q_len=q_len, ragged=rng.random() < 0.5, scales=rng.choice(["pow2", "pow2", "any"]))
    case["seqs"] = max(1, min(case["seqs"], limit))
    if case["seqs"] * q_heads * q_len * tokens > MOST_PAIRS // (8 if case["dtype"] == "fp32" and use == "prompt" else 1):
        case["q_len"] = 1
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(case, what, least, salt=0):
    """A length for each sequence: `what` itself, or spread between an eighth of it and it (the first one has it all)."""
    n, most = case["seqs"], case[what]
    if not case.get("ragged", True) or most <= least:
        return np.full(n, most, dtype=np.int64)
    lens = np.random.RandomState(salt + n + most).randint(max(least, most // 8), most + 1, n).astype(np.int64)
    lens[0] = most
    return lens


def _lens_of(case):
    """(tokens held, new tokens) of each sequence: the case's own, which a seed only brings into another order."""
    if case["kind"] == "attention":
        return _lengths(case, "tokens", 1), np.full(case["seqs"], case["q_len"], dtype=np.int64)
    if case["kind"] == "step":
        new = np.ones(case["seqs"], dtype=np.int64)
        new[-1] = case["new"]
        return _lengths(case, "held", 1), new
    return _lengths(case, "held", 0), _lengths(case, "new", 1, 7)


def _tables(lens, room, bs, seed):
    """Pages for `lens` tokens of each sequence in random order, and a stack of the others; tables have `room` pages a row."""
    have = -(-lens // bs)
    want = -(-room // bs)
    total = int(want.sum())
    order = np.random.RandomState((seed + 1) % (1 << 31)).permutation(total).astype(np.int32)
    table = np.zeros((len(lens), max(1, int(want.max()))), dtype=np.int32)
    ends = np.cumsum(have)
    row = np.repeat(np.arange(len(lens)), have)
    table[row, np.arange(int(have.sum())) - np.repeat(ends - have, have)] = order[:int(have.sum())]
    free = np.zeros(total, dtype=np.int32)
    rest = order[int(have.sum()):]
    free[:len(rest)] = rest
    to = lambda a: torch.from_numpy(a).to(DEV)      # noqa: E731
    return {"block_table": to(table), "seq_lens": to(lens.astype(np.int32)), "free_pages": to(free),
            "pool": torch.tensor([len(rest), 0], dtype=torch.int32, device=DEV)}, total


def _vectors(g, shape, dtype):
    """N(0, 1) with a few channels eight times as large, the same ones over the tokens (shape ends in heads, dim)."""
    heads, dim = shape[-2:]
    scale = torch.ones(heads, dim, device=DEV)
    scale.scatter_(1, torch.rand(heads, dim, generator=g, device=DEV).argsort(1)[:, :4], 8.0)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _pages(case, g, total, scales):
    """Filled pages: (blocks, heads, block, dim) codes (in memory heads before tokens, or tokens before heads) and scales."""
    H, bs, d, kind = case["kv_heads"], case["block"], case["dim"], case["codes"]
    out = {}
    for name in ("k", "v"):
        shape = (total, H, bs, d) if case["layout"] == "hnd" else (total, bs, H, d)
        codes = torch.empty(shape, dtype=CODES[kind], device=DEV)
        view = codes if case["layout"] == "hnd" else codes.transpose(1, 2)
        sc = torch.empty(total, H, device=DEV)
        step = max(1, (1 << 26) // (H * bs * d))
        for at in range(0, total, step):
            m = min(step, total - at)
            x = _vectors(g, (m, bs, H, d), torch.float32).transpose(1, 2)
            x = x * torch.exp(0.5 * torch.randn(m, H, 1, 1, generator=g, device=DEV))
            s = x.abs().amax((2, 3)) / TOP[kind]
            if scales == "pow2":
                s = torch.exp2(torch.ceil(torch.log2(s)))
            y = (x / s[..., None, None]).clamp(-TOP[kind], TOP[kind])
            view[at:at + m] = y.round().to(torch.int8) if kind == "int8" else y.to(CODES[kind])
            sc[at:at + m] = s
        out[name + "_codes"], out[name + "_scales"] = view, sc
    return out


def prepare(case, seed):
    g = _gen(seed)
    bs = case["block"]
    state = {"case": dict(case)}
    held, new = _lens_of(case)
    order = np.random.RandomState((seed + 2) % (1 << 31)).permutation(case["seqs"])
    held, new = held[order], new[order]
    if case["kind"] == "attention":
        tables, total = _tables(held, held, bs, seed)
        state.update(tables, **_pages(case, g, total, case["scales"]))
        q = torch.randn(case["seqs"], case["q_heads"], case["q_len"], case["dim"], generator=g, device=DEV)
        state.update(queries=q.to(DTYPES[case["dtype"]]), max_kv_len=int(held.max()))
        return state
    tables, total = _tables(held, held + new, bs, seed)
    state.update(tables, new_lens=torch.from_numpy(new.astype(np.int32)).to(DEV))
    T = int(new.sum())
    state["max_tokens"] = T if case["kind"] == "append" else T + 5         # a captured step has room for more
    if case["kind"] == "extend":
        return state
    state.update(_pages(case, g, total, "pow2"))
    # Projections of all heads lie side by side in the rows that a model computes.
    qh = case.get("q_heads", 0)
    rows = _vectors(g, (state["max_tokens"], 2 * case["kv_heads"] + qh, case["dim"]), torch.float32)
    rows = rows.to(DTYPES[case["dtype"]])
    h = case["kv_heads"]
    state.update(keys=rows[:, qh:qh + h], values=rows[:, qh + h:], queries=rows[:, :qh], max_q_len=int(new.max()),
                 max_kv_len=int((held + new).max()))
    if case["kind"] == "append":
        # Slots as the tables give them; the last token of the call is padding where there is more than one.
        slots = _plain_extend(state)["slots"]
        if T > 1:
            slots[-1] = -1
        state["slots"] = slots
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------

def _plain_extend(s):
    bs = s["case"]["block"]
    table, held, new, free, pool = s["block_table"], s["seq_lens"].long(), s["new_lens"].long(), s["free_pages"], s["pool"]
    n, width = table.shape
    have = (held + bs - 1) // bs
    need = (((held + new + bs - 1) // bs).clamp(max=width) - have).clamp(min=0)
    before = need.cumsum(0) - need
    left = pool[0].long()
    got = torch.minimum((left - before).clamp(min=0), need)
    granted = torch.minimum(new, ((have + got) * bs - held).clamp(min=0))
    column = torch.arange(width, device=DEV)[None]
    at = left - 1 - (before[:, None] + column - have[:, None])
    fresh = (column >= have[:, None]) & (column < (have + got)[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), new.cumsum(0)])
    token = torch.arange(s["max_tokens"], device=DEV)
    row = torch.searchsorted(starts[1:], token, right=True)
    real = row < n
    row = row.clamp(max=n - 1)
    inside = token - starts[row]
    pos = held[row] + inside
    page = table[row, (pos // bs).clamp(max=width - 1)].long()
    slots = torch.where(real & (inside < granted[row]), page * bs + pos % bs, torch.full_like(pos, -1))
    counts = torch.stack([left - got.sum(), pool[1].long() + (new - granted).sum()])
    return {"slots": slots, "query_starts": starts.int(), "seq_lens": (held + granted).int(), "pool": counts.int(),
            "block_table": table}


def _codes_of(x, kind):
    x = x.clamp(-TOP[kind], TOP[kind])
    return x.round().to(torch.int8) if kind == "int8" else x.to(CODES[kind])


def _plain_append_one(x, codes, scales, slots, kind, bs):
    """x (T, H, d) into codes (blocks, H, bs, d) and scales (blocks, H)."""
    nb, H, _, d = codes.shape
    x = x.float()
    real = slots >= 0
    page = torch.where(real, slots, torch.zeros_like(slots)) // bs
    off = torch.where(real, slots % bs, torch.full_like(slots, bs))
    top = torch.where(real[:, None], x.abs().amax(2), torch.zeros((), device=DEV))
    first = torch.full((nb,), bs, dtype=torch.int64, device=DEV).scatter_reduce(0, page, off, "amin")
    most = torch.zeros(nb, H, device=DEV).scatter_reduce(0, page[:, None].expand(-1, H), top, "amax")
    part, power = torch.frexp(most)
    power = power - (9 if kind == "e4m3" else 7) + (part > (0.875 if kind == "e4m3" else 0.9921875)).to(power.dtype)
    fresh = torch.where(most > 0, torch.ldexp(torch.ones_like(most), power.clamp(min=-120)), torch.zeros_like(most))
    new = torch.where((first < bs)[:, None], torch.maximum(fresh, torch.where((first > 0)[:, None], scales, torch.zeros_like(scales))), scales)
    held = torch.arange(bs, device=DEV)[None] < torch.where(first < bs, first, torch.zeros_like(first))[:, None]
    ratio = torch.where(new > 0, scales / new, torch.ones_like(new))
    moved = held[:, None, :] & (ratio != 1)[:, :, None]
    old = torch.where(moved[..., None], _codes_of(codes.float() * ratio[:, :, None, None], kind).view(torch.uint8), codes.view(torch.uint8))
    inverse = torch.where(new > 0, 1 / new, torch.zeros_like(new))
    mine = _codes_of(x * inverse[page][..., None], kind).view(torch.uint8)
    source = torch.full((nb * bs + 1,), -1, dtype=torch.int64, device=DEV)
    source.scatter_(0, torch.where(real, slots, torch.full_like(slots, nb * bs)), torch.arange(slots.numel(), device=DEV))
    source = source[:-1].view(nb, bs)
    put = mine[source.clamp(min=0)].transpose(1, 2)
    codes.view(torch.uint8).copy_(torch.where((source >= 0)[:, None, :, None], put, old))
    scales.copy_(new)


def _plain_append(s, slots):
    c = s["case"]
    _plain_append_one(s["keys"], s["k_codes"], s["k_scales"], slots, c["codes"], c["block"])
    _plain_append_one(s["values"], s["v_codes"], s["v_scales"], slots, c["codes"], c["block"])
    return {k: s[k] for k in ("k_codes", "v_codes", "k_scales", "v_scales")}


def _plain_attention(s, q, q_lens, kv_lens):
    """q (n, Hq, Q, d), the first q_lens rows of each sequence real; causal."""
    c = s["case"]
    n, Hq, Q, d = q.shape
    H, bs = c["kv_heads"], c["block"]
    width = -(-s["max_kv_len"] // bs)
    pages = s["block_table"][:, :width].long()

    def dense(name):
        x = s[name + "_codes"].view(torch.uint8)[pages].view(CODES[c["codes"]]).float() * s[name + "_scales"][pages][..., None, None]
        return x.transpose(1, 2).reshape(n, H, width * bs, d)

    pos = torch.arange(width * bs, device=DEV)
    row = torch.arange(Q, device=DEV)
    last = (kv_lens - q_lens)[:, None] + row[None]                                        # (n, Q)
    see = (pos[None, None] <= last[:, :, None]) & (pos[None, None] < kv_lens[:, None, None]) & (row[None] < q_lens[:, None])[:, :, None]
    see = see[:, None, None]
    k = dense("k")
    score = torch.matmul(q.float().reshape(n, H, Hq // H * Q, d) * (1.0 / math.sqrt(d)), k.transpose(2, 3))
    del k
    score = score.view(n, H, Hq // H, Q, width * bs).masked_fill(~see, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    del score
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(n, H, Hq // H * Q, width * bs), dense("v")).view(n, H, Hq // H, Q, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.reshape(n, Hq, Q, d)


def _plain_ragged(s, q, starts, kv_lens):
    """q (T, Hq, d), rows starts[i] .. starts[i + 1] of sequence i; rows behind the last sequence give zeros."""
    starts, kv_lens = starts.long(), kv_lens.long()
    q_lens = starts[1:] - starts[:-1]
    row = torch.arange(s["max_q_len"], device=DEV)
    at = (starts[:-1, None] + row[None]).clamp(max=q.shape[0] - 1)
    out = _plain_attention(s, q[at].transpose(1, 2), q_lens, kv_lens)                  # (n, Hq, Q, d)
    token = torch.arange(q.shape[0], device=DEV)
    seq = torch.searchsorted(starts[1:], token, right=True)
    real = seq < q_lens.numel()
    seq = seq.clamp(max=q_lens.numel() - 1)
    picked = out[seq, :, (token - starts[seq]).clamp(max=s["max_q_len"] - 1)]
    return torch.where(real[:, None, None], picked, torch.zeros_like(picked)).to(q.dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        from quashkv_b200.integrations import paged8
        pages = () if c["kind"] == "extend" else (s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
        if c["kind"] == "attention":
            return paged8.attention_paged8(s["queries"], *pages, s["block_table"], s["seq_lens"], s["max_kv_len"], causal=True)
        if c["kind"] == "append":
            paged8.append_paged8(s["keys"], s["values"], *pages, s["slots"])
            return {k: s[k] for k in ("k_codes", "v_codes", "k_scales", "v_scales")}
        plan = paged8.extend_pages(s["block_table"], s["seq_lens"], s["new_lens"], s["free_pages"], s["pool"], c["block"],
                                   s["max_tokens"])
        if c["kind"] == "extend":
            return {"slots": plan.slots, "query_starts": plan.query_starts, "seq_lens": plan.seq_lens, "pool": plan.pool,
                    "block_table": s["block_table"]}
        paged8.append_paged8(s["keys"], s["values"], *pages, plan.slots)
        out = paged8.attention_paged8(s["queries"], *pages, s["block_table"], plan.seq_lens, s["max_kv_len"], causal=True,
                                      query_starts=plan.query_starts, max_q_len=s["max_q_len"])
        return {"slots": plan.slots, "seq_lens": plan.seq_lens, "k_codes": s["k_codes"], "v_codes": s["v_codes"],
                "k_scales": s["k_scales"], "v_scales": s["v_scales"], "out": out}
    if c["kind"] == "attention":
        q = s["queries"]
        n = q.shape[0]
        return _plain_attention(s, q, torch.full((n,), q.shape[2], device=DEV), s["seq_lens"].long()).to(q.dtype)
    if c["kind"] == "append":
        return _plain_append(s, s["slots"])
    plan = _plain_extend(s)
    if c["kind"] == "extend":
        return plan
    cache = _plain_append(s, plan["slots"])
    out = _plain_ragged(s, s["queries"], plan["query_starts"], plan["seq_lens"])
    return {"slots": plan["slots"], "seq_lens": plan["seq_lens"], **cache, "out": out}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    c, bs = case, case["block"]
    held, new = _lens_of(c)
    if c["kind"] == "attention":
        return _attention_work(c, held, new)
    T = int(new.sum())
    pages = int((-(-(held + new) // bs) - -(-held // bs)).sum())
    tables = 12 * c["seqs"] + 8 * pages + 8 * T
    if c["kind"] == "extend":
        return {"bytes": tables, "flops": 0}
    item = 4 if c["dtype"] == "fp32" else 2
    store = 2 * T * c["kv_heads"] * c["dim"] * (item + 1) + 8 * T
    if c["kind"] == "append":
        return {"bytes": store, "flops": 2 * T * c["kv_heads"] * c["dim"]}
    w = _attention_work(c, held + new, new)
    return {"bytes": tables + store + w["bytes"], "flops": w["flops"]}


def _attention_work(c, lens, q):
    item = 4 if c["dtype"] == "fp32" else 2
    kv = float(lens.sum()) * c["kv_heads"] * 2 * c["dim"] + float((-(-lens // c["block"])).sum()) * (8 * c["kv_heads"] + 4)
    rows = float(q.sum()) * c["q_heads"] * c["dim"] * item * 2
    q = np.minimum(q, lens)
    pairs = float((q * lens - q * (q - 1) // 2).sum())
    return {"bytes": int(kv + rows), "flops": int(4 * c["dim"] * c["q_heads"] * pairs)}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c, bs = case, case["block"]
    if c["kind"] == "extend":
        return _exact_extend(s, bs)
    if c["kind"] == "attention":
        q = s["queries"].double()
        lens = s["seq_lens"].tolist()
        return torch.stack([_exact_rows(s, q[i].transpose(0, 1), i, lens[i]).transpose(0, 1) for i in range(len(lens))])
    if c["kind"] == "append":
        return _exact_append(s, s["slots"].tolist())
    plan = _exact_extend(s, bs)
    s["block_table"] = plan["block_table"].to(DEV)
    cache = _exact_append(s, plan["slots"].tolist())
    starts, lens = plan["query_starts"].tolist(), plan["seq_lens"].tolist()
    s = {**s, "k_values": cache["k_codes"], "v_values": cache["v_codes"], "k_scales": cache["k_scales"], "v_scales": cache["v_scales"]}
    out = torch.zeros(s["queries"].shape, dtype=torch.float64, device=DEV)
    for i, n in enumerate(lens):
        out[starts[i]:starts[i + 1]] = _exact_rows(s, s["queries"][starts[i]:starts[i + 1]].double(), i, n)
    return {"slots": plan["slots"], "seq_lens": plan["seq_lens"], **cache, "out": out}


def _exact_rows(s, q, i, n):
    """q (Q, Hq, d): the last Q positions of sequence i of n tokens."""
    c = s["case"]
    bs, H, d, Q = c["block"], c["kv_heads"], c["dim"], q.shape[0]
    pages = s["block_table"][i, :-(-n // bs)].long()
    heads = []
    for h in range(H):
        def flat(name):
            codes = s[name + "_values"][:, h] if name + "_values" in s else s[name + "_codes"][:, h].view(torch.uint8)
            x = codes[pages]
            x = x if x.dtype == torch.float64 else x.view(CODES[c["codes"]]).double()
            return (x * s[name + "_scales"][pages, h].double()[:, None, None]).reshape(-1, d)[:n]
        x = q[:, h * (c["q_heads"] // H):(h + 1) * (c["q_heads"] // H)].transpose(0, 1)        # (G, Q, d)
        t = x @ flat("k").T / math.sqrt(d)
        hide = torch.ones(Q, n, dtype=torch.bool, device=DEV).triu(n - Q + 1)
        w = torch.softmax(t.masked_fill(hide[None], -math.inf), -1)
        heads.append(torch.nan_to_num(w) @ flat("v"))
    return torch.cat(heads).transpose(0, 1)


def _exact_extend(s, bs):
    table, free = s["block_table"].cpu().numpy().copy(), s["free_pages"].tolist()
    held, new = s["seq_lens"].tolist(), s["new_lens"].tolist()
    left, missed = s["pool"].tolist()
    slots, starts, lens = [], [0], []
    for i, (L, N) in enumerate(zip(held, new)):
        pages = -(-L // bs)
        while pages < min(-(-(L + N) // bs), table.shape[1]) and left > 0:
            left -= 1
            table[i, pages] = free[left]
            pages += 1
        can = min(N, max(0, pages * bs - L))
        slots += [int(table[i, p // bs]) * bs + p % bs for p in range(L, L + can)] + [-1] * (N - can)
        missed += N - can
        starts.append(starts[-1] + N)
        lens.append(L + can)
    slots += [-1] * (s["max_tokens"] - len(slots))
    return {"slots": torch.tensor(slots), "query_starts": torch.tensor(starts, dtype=torch.int32),
            "seq_lens": torch.tensor(lens, dtype=torch.int32), "pool": torch.tensor([left, missed], dtype=torch.int32),
            "block_table": torch.from_numpy(table)}


def _exact_append(s, slots):
    """Runs of slots one by one on the host, in numpy."""
    c, bs = s["case"], s["case"]["block"]
    top = TOP[c["codes"]]
    out = {}

    def rounded(y):
        if c["codes"] == "int8":
            return np.rint(y)
        _, e = np.frexp(y)
        unit = np.ldexp(1.0, np.maximum(e - 4, -9))            # four bits of a normal number, 2^-9 below
        return np.rint(y / unit) * unit

    runs = []
    for t, slot in enumerate(slots):
        if slot < 0:
            continue
        if runs and runs[-1][0] + runs[-1][1] == t and slots[t - 1] + 1 == slot and slot % bs:
            runs[-1][1] += 1
        else:
            runs.append([t, 1])
    for name, key in (("k", "keys"), ("v", "values")):
        codes = s[name + "_codes"].float().cpu().numpy().astype(np.float64)
        scales = s[name + "_scales"].cpu().numpy().astype(np.float64)
        x = s[key].float().cpu().numpy().astype(np.float64)
        for t, n in runs:
            page, at = divmod(slots[t], bs)
            mine = x[t:t + n].transpose(1, 0, 2)                # (H, n, d)
            most = np.abs(mine).max((1, 2))
            fresh = np.where(most > 0, 2.0 ** np.maximum(np.ceil(np.log2(np.maximum(most, 1e-300) / top)), -120), 0)
            old = scales[page] if at else np.zeros_like(fresh)
            new = np.maximum(fresh, old)
            ratio = np.where(new > 0, old / np.where(new > 0, new, 1), 1)
            codes[page, :, :at] = np.where(ratio[:, None, None] != 1, rounded(codes[page, :, :at] * ratio[:, None, None]), codes[page, :, :at])
            codes[page, :, at:at + n] = rounded(mine / np.where(new > 0, new, np.inf)[:, None, None])
            scales[page] = new
        out[name + "_codes"] = torch.from_numpy(codes).to(DEV)
        out[name + "_scales"] = torch.from_numpy(scales).to(DEV)
    return out
