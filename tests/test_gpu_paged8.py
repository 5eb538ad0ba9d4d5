"""The 8-bit paged cache on the GPU: tables and slots and appends equal to the definitions, attention within the error that its
arithmetic allows, and the three together as a serving loop uses them."""

import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import paged8_reference as ref
from quashkv_b200.integrations import paged8
from quashkv_b200.integrations.vllm_backend import QuashKVPagedCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def _i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(DEV)


# ---- tables and slots -------------------------------------------------------------------------------------------------

def _random_state(rs, n, w, bs, spare):
    lens = rs.randint(0, w * bs + 1, n)
    have = -(-lens // bs)
    total = int(have.sum()) + spare
    order = rs.permutation(total).astype(np.int32)
    table = rs.randint(1000, 2000, (n, w)).astype(np.int32)
    at = 0
    for i, k in enumerate(have):
        table[i, :k] = order[at:at + k]
        at += k
    free = np.full(max(total, 1), -7, dtype=np.int32)
    free[:spare] = order[at:]
    return lens, table, free, [spare, 5]


def _check_extend(rs, n, w, bs, new, spare, max_tokens=None, lens=None):
    held, table, free, pool = _random_state(rs, n, w, bs, spare)
    held = held if lens is None else np.asarray(lens)
    T = int(np.maximum(new, 0).sum()) + 3 if max_tokens is None else max_tokens
    want = ref.extend(table, held, new, free, pool, bs, T)
    t, f, p, h = _i32(table), _i32(free), _i32(pool), _i32(held)
    plan = paged8.extend_pages(t, h, _i32(new), f, p, bs, T)
    assert t.cpu().numpy().tolist() == want[0].tolist()
    assert plan.slots.tolist() == want[1] and plan.query_starts.tolist() == want[2]
    assert plan.seq_lens.tolist() == want[3] and plan.pool.tolist() == want[4]
    assert h.tolist() == list(held) and p.tolist() == pool and f.tolist() == free.tolist()      # nothing else is written
    return t, plan, f, held, table


@pytest.mark.parametrize("n", [1, 2, 31, 33, 255, 1000, 4097])
@pytest.mark.parametrize("bs", [1, 16, 48])
def test_extend_equals_the_definition(n, bs):
    rs = np.random.RandomState(n + bs)
    w = 5
    for most, spare in ((1, n), (2 * bs + 1, 3 * n), (2 * bs + 1, n // 2)):
        _check_extend(rs, n, w, bs, rs.randint(0, most + 1, n), spare)


def test_extend_at_its_limits():
    rs = np.random.RandomState(1)
    _check_extend(rs, 3, 4, 16, np.array([0, 0, 0]), 2)                                   # nothing new
    _check_extend(rs, 3, 4, 16, np.array([64, 64, 64]), 0)                                # an empty stack
    _check_extend(rs, 3, 4, 16, np.array([500, 1, 700]), 12)                              # rows of the table full
    _check_extend(rs, 4, 6, 16, np.array([9, 9, 9, 9]), 12, max_tokens=20)                # less room than tokens
    _check_extend(rs, 4, 6, 16, np.array([9, 9, 9, 9]), 12, max_tokens=0)
    _check_extend(rs, 4, 6, 16, np.array([-3, 9, -1, 4]), 12)                             # negative counts are none
    _check_extend(rs, 3, 4, 16, np.array([2 ** 31 - 1, 2 ** 31 - 1, 2]), 9, max_tokens=100)      # sums beyond 32 bits
    _check_extend(rs, 2, 4, 16, np.array([3, 3]), 4, lens=[1000, 5])                      # more tokens than the row has pages
    _check_extend(rs, 16384, 2, 16, rs.randint(0, 20, 16384), 20000)                      # as many sequences as are taken
    _check_extend(rs, 7, 600, 16, rs.randint(0, 9000, 7), 4000)                           # long ones


@pytest.mark.parametrize("spare", [40, 900])
def test_a_large_step_updates_lengths_in_place(spare):
    """More tokens than one CTA takes: lengths and counts change behind all that read them, pages lasting and not."""
    n, w, bs, most = 50, 60, 16, 9000
    tables = paged8.PageTables(spare, n, w, block_size=bs)
    rs, free = np.random.RandomState(spare), tables.free_pages.cpu().numpy()
    held, pool, table = [0] * n, tables.pool.tolist(), tables.block_table.cpu().numpy()
    for _ in range(3):
        new = rs.randint(0, 200, n)
        plan = tables.extend(_i32(new), most)
        table, slots, starts, after, pool = ref.extend(table, held, new.tolist(), free, pool, bs, most)
        assert plan.slots.tolist() == slots and plan.query_starts.tolist() == starts and plan.start_lens.tolist() == held
        assert tables.seq_lens.tolist() == after and tables.pool.tolist() == pool
        have = [-(-x // bs) for x in after]
        assert all(np.array_equal(tables.block_table[i, :k].cpu().numpy(), table[i, :k]) for i, k in enumerate(have))
        held = after


@pytest.mark.parametrize("n,bs", [(1, 16), (33, 16), (700, 1), (16384, 48)])
def test_shrink_restores_what_extend_took(n, bs):
    rs = np.random.RandomState(n)
    new = rs.randint(0, 3 * bs + 1, n)
    held, table, free, pool = _random_state(rs, n, 6, bs, 2 * n)
    t, f, p, h = _i32(table), _i32(free), _i32(pool), _i32(held)
    T = int(new.sum())
    slots, starts, before = torch.ops.quashkv_b200.extend_pages_(t, h, _i32(new), f, p, bs, T)
    want = ref.extend(table, held, new, free, pool, bs, T)
    assert slots.tolist() == want[1] and h.tolist() == want[3] and p.tolist() == want[4] and before.tolist() == list(held)
    keep = np.minimum(rs.randint(0, 6 * bs, n), want[3])
    after, free2, count = ref.shrink(want[0], want[3], keep, free, want[4], bs)
    h2, f2, p2 = h.clone(), f.clone(), p.clone()
    torch.ops.quashkv_b200.shrink_pages_(t, h2, _i32(keep), f2, p2, bs)
    assert h2.tolist() == after and f2.tolist() == free2 and p2.tolist() == count
    torch.ops.quashkv_b200.shrink_pages_(t, h, _i32(held), f, p, bs)
    assert h.tolist() == list(held) and f.tolist() == list(free) and p.tolist() == [pool[0], want[4][1]]


def test_pages_returned_twice_stay_inside_the_stack():
    t, f, p, h = _i32([[0, 1, 2]]), _i32([3, 4]), _i32([2, 0]), _i32([40])
    torch.ops.quashkv_b200.shrink_pages_(t, h, _i32([0]), f, p, 16)
    assert h.tolist() == [0] and p.tolist() == [2, 0]


# ---- append -------------------------------------------------------------------------------------------------------------

def _pool(total, H, bs, d, dtype, layout, seed=0, fill=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    k, v, ks, vs = ref.random_pages(g, total, H, bs, d, dtype, layout)
    return k, v, ks, vs


def _host(pages):
    return [p.float().cpu().numpy().astype(np.float64) for p in pages]


def _check_append(keys, values, pages, slots, bs, dtype, call):
    want = _host(pages)
    for x, codes, scales in ((keys, want[0], want[2]), (values, want[1], want[3])):
        ref.append(x.float().cpu().numpy().astype(np.float64), codes, scales, slots, bs, dtype)
    call()
    for got, exact in zip(_host(pages), want):
        assert np.array_equal(got, exact, equal_nan=True)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,H,bs,layout", [(128, 2, 16, "hnd"), (64, 3, 48, "nhd"), (96, 1, 32, "hnd"), (32, 2, 16, "nhd")])
def test_append_equals_the_definition(d, H, bs, layout, x_dtype, dtype):
    g = torch.Generator(device=DEV).manual_seed(d + bs)
    rs = np.random.RandomState(d)
    for T, seqs in ((1, 1), (5, 3), (2 * bs + 3, 2), (700, 4)):
        pages = _pool(-(-T * seqs // bs) + 4 * seqs, H, bs, d, dtype, layout, seed=T)
        order, at, slots = rs.permutation(pages[0].shape[0]), 0, []
        for _ in range(seqs):                                      # each sequence from a position of its own
            first = int(rs.randint(0, 2 * bs))
            need = -(-(first + T) // bs)
            slots += [int(order[at + p // bs - first // bs]) * bs + p % bs for p in range(first, first + T)]
            at += need - first // bs
        slots = np.array(slots)
        page = slots // bs                                         # pages are left out as a whole: what is stored of one is one run
        for p in rs.choice(page, 1 + len(slots) // 100):
            slots[page == p] = -1 if rs.rand() < 0.5 else pages[0].shape[0] * bs + 3
        n = len(slots)
        x = torch.randn(n, 2 * H + 1, d, generator=g, device=DEV) * torch.exp2(6 * torch.rand(n, 2 * H + 1, 1, generator=g, device=DEV) - 3)
        x = x.to(x_dtype)
        keys, values = x[:, :H], x[:, H:2 * H]                     # strided, as a projection gives them
        _check_append(keys, values, pages, slots, bs, dtype, lambda: paged8.append_paged8(keys, values, *pages, torch.from_numpy(slots).to(DEV)))


@pytest.mark.parametrize("total", [300, 900, 1500, 2600, 5000])
def test_append_of_runs_of_any_length(total):
    """Runs of 1 to 20 tokens on pages of their own, in calls whose warps look for the runs of few or many tokens."""
    rs, g = np.random.RandomState(total), torch.Generator(device=DEV).manual_seed(total)
    H, d, bs = 4, 32, 32
    slots, page = [], 0
    while len(slots) < total:
        n, at = rs.randint(1, 21), rs.randint(0, 12)
        slots += list(range(page * bs + at, page * bs + at + n))
        page += 1
    slots = np.array(slots[:total])
    order = rs.permutation(page)                             # pages in any order
    slots = order[slots // bs] * bs + slots % bs
    slots[slots // bs == slots[total // 2] // bs] = -1       # a page that is left out
    k, v = (torch.randn(total, H, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    pages = _pool(page, H, bs, d, E4M3, "hnd")
    _check_append(k, v, pages, slots.tolist(), bs, E4M3, lambda: paged8.append_paged8(k, v, *pages, torch.from_numpy(slots).to(DEV)))


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_token_by_token_the_scale_rises_and_old_codes_follow(dtype):
    """Tokens that grow and shrink by large factors, one a call: every rise rounds what the page holds again."""
    H, bs, d = 2, 16, 64
    pages = _pool(3, H, bs, d, dtype, "hnd")
    g = torch.Generator(device=DEV).manual_seed(3)
    size = [1, 0.01, 3, 100, 0, 1e-30, 1e4, 1e4, 2e4, 1e-3, 1, 1, 7e4, 1, 1e30, 0, 1, 2]
    for i, s in enumerate(size):
        x = torch.randn(1, H, d, generator=g, device=DEV) * s
        slot = (1 if i < bs else 2) * bs + i % bs
        _check_append(x, -x, pages, [slot], bs, dtype, lambda: paged8.append_paged8(x, -x, *pages, torch.tensor([slot], device=DEV)))


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_infinities_and_nan_mark_their_page_and_head(dtype):
    H, bs, d = 3, 16, 128
    pages = _pool(4, H, bs, d, dtype, "hnd")
    x = torch.randn(32, H, d, device=DEV)
    x[3, 1, 5], x[20, 2, 127], x[21, 0, 0] = float("nan"), float("inf"), float("-inf")
    slots = np.r_[np.arange(16, 32), np.arange(48, 64)]
    y = torch.randn(32, H, d, device=DEV)
    call = lambda: paged8.append_paged8(x, y, *pages, torch.from_numpy(slots).to(DEV))      # noqa: E731
    _check_append(x, y, pages, slots, bs, dtype, call)
    assert pages[2].isnan().sum() == 3 and not pages[3].isnan().any()
    z = torch.randn(1, H, d, device=DEV)
    for slot in (16, 17):            # a page begun anew forgets it, one that goes on keeps it
        _check_append(z, z, pages, [slot], bs, dtype, lambda: paged8.append_paged8(z, z, *pages, torch.tensor([slot], device=DEV)))
    assert pages[2].isnan().sum() == 2


def test_append_through_tables_drops_and_counts_what_has_no_place():
    H, bs, d = 2, 16, 64
    pages = _pool(6, H, bs, d, E4M3, "hnd")
    table, starts = _i32([[3, 1], [5, -1], [2, 99]]), _i32([30, 12, 16])
    x, y = torch.randn(3, H, 9, d, device=DEV), torch.randn(3, H, 9, d, device=DEV)
    place = lambda i, p: int(table[i, p // bs]) * bs + p % bs if p < 2 * bs and 0 <= int(table[i, p // bs]) < 6 else -1      # noqa: E731
    slots = [place(i, int(starts[i]) + t) for i in range(3) for t in range(9)]
    before = paged8.dropped_tokens()
    flat = lambda a: a.transpose(1, 2).reshape(27, H, d)      # noqa: E731
    _check_append(flat(x), flat(y), pages, slots, bs, E4M3, lambda: paged8.append_paged8(x, y, *pages, block_table=table, start_lens=starts))
    assert paged8.dropped_tokens() - before == H * slots.count(-1) == H * (7 + 5 + 9)
    wide = _i32(np.zeros((3, 7)))                                  # the same table as part of a wider one
    wide[:, 2:4] = table
    again = _pool(6, H, bs, d, E4M3, "hnd")
    paged8.append_paged8(x, y, *again, block_table=wide[:, 2:4], start_lens=starts)
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(_host(again), _host(pages)))
    paged8.append_paged8(x[:, :, :0], y[:, :, :0], *again, block_table=table, start_lens=starts)      # no tokens
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(_host(again), _host(pages)))


def test_misaligned_and_other_inputs_are_taken():
    """Rows that do not start on 16 bytes, a transposed last dimension, fp64: copied, with the same result."""
    H, bs, d = 2, 16, 64
    x = torch.randn(20, H, d, device=DEV, dtype=torch.bfloat16)
    slots = torch.arange(20, device=DEV)
    want = _pool(2, H, bs, d, INT8, "hnd")
    paged8.append_paged8(x, x, *want, slots)
    odd = torch.empty(20, H, d + 1, device=DEV, dtype=torch.bfloat16)[:, :, 1:]
    flat = torch.empty(20 * H * d + 3, device=DEV, dtype=torch.bfloat16)[3:].view(20, H, d)
    turned = torch.empty(20, d, H, device=DEV, dtype=torch.bfloat16).transpose(1, 2)
    for t in (odd, flat, turned):
        t.copy_(x)
    for t in (odd, flat, turned, x.double()):
        got = _pool(2, H, bs, d, INT8, "hnd")
        paged8.append_paged8(t, t, *got, slots)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        table, lens = _i32([[0, 1]]), _i32([20])
        q = t[:1].unsqueeze(2)
        out = paged8.attention_paged8(q, *got, table, lens, 20)
        ref_out = paged8.attention_paged8(x[:1].unsqueeze(2), *want, table, lens, 20)
        assert torch.allclose(out.float(), ref_out.float(), atol=1e-2)


# ---- attention ------------------------------------------------------------------------------------------------------------

def _check_attention(q, pages, table, lens, causal=True, starts=None, scale=None, max_kv_len=None, max_q_len=None):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    exact, bound = ref.attention(q, pages, table, lens, scale, causal, starts)
    got = paged8.attention_paged8(q, *pages, table, lens, int(max(int(lens.max()), 1)) if max_kv_len is None else max_kv_len, scale=scale, causal=causal,
                                  query_starts=None if starts is None else _i32(starts), max_q_len=max_q_len)
    assert got.shape == q.shape and got.dtype == q.dtype
    most = torch.finfo(q.dtype).max                          # fp16: what lies beyond its range is an infinity
    got = got.double()
    assert torch.equal(got.isnan(), exact.isnan())
    beyond = exact.abs() - bound > most * (1 + torch.finfo(q.dtype).eps)
    assert torch.equal(got[beyond], torch.full_like(got[beyond], math.inf).copysign(exact[beyond]))
    beyond |= exact.abs() + bound > most
    got, exact = got.masked_fill(beyond, 0), exact.masked_fill(beyond, 0)
    worst = ((got - exact).abs() - bound).nan_to_num(nan=0.0)
    assert worst.max() <= 0, (float(worst.max()), float(((got - exact).abs() / bound.clamp(min=1e-300)).nan_to_num().max()))


LENS = [[1], [0, 1, 15, 16, 17], [63, 64, 65, 130], [1000, 3], [257] * 9]


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,H,G,bs,layout", [(128, 2, 4, 16, "hnd"), (64, 2, 8, 48, "nhd"), (96, 3, 1, 32, "hnd"), (32, 1, 16, 16, "nhd"), (128, 1, 12, 64, "nhd")])
def test_attention_of_single_tokens(d, H, G, bs, layout, x_dtype, dtype):
    g = torch.Generator(device=DEV).manual_seed(d + G)
    for lens in LENS:
        total = sum(-(-n // bs) for n in lens) + 2
        pages = ref.random_pages(g, total, H, bs, d, dtype, layout, pow2=G > 2)
        table = ref.random_tables(lens, bs, total, len(lens)).to(DEV)
        q = torch.randn(len(lens), H * G, 1, d, generator=g, device=DEV).to(x_dtype)
        _check_attention(q, pages, table, _i32(lens), causal=len(lens) % 2 == 0)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,H,G,bs,layout", [(128, 2, 4, 16, "hnd"), (64, 1, 8, 32, "nhd"), (96, 2, 2, 16, "hnd"), (32, 1, 3, 48, "hnd")])
@pytest.mark.parametrize("q_len", [2, 7, 33, 64, 130, 300])
def test_attention_of_many_rows(q_len, d, H, G, bs, layout, x_dtype, dtype):
    """Blocks of queries shorter and longer than the sequences: rows in front of the first position see nothing."""
    g = torch.Generator(device=DEV).manual_seed(q_len)
    lens = [q_len, 0, 1, q_len + 17, 3 * q_len + 5, max(1, q_len // 2)]
    total = sum(-(-n // bs) for n in lens) + 2
    pages = ref.random_pages(g, total, H, bs, d, dtype, layout)
    table = ref.random_tables(lens, bs, total, q_len).to(DEV)
    q = torch.randn(len(lens), q_len, H * G, d, generator=g, device=DEV).to(x_dtype).transpose(1, 2)      # strided
    for causal in (True, False):
        _check_attention(q, pages, table, _i32(lens), causal=causal)


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,H,G", [(128, 2, 4), (64, 2, 8)])
def test_attention_of_a_ragged_batch(d, H, G, x_dtype):
    """Decodes, short blocks and a piece of a prompt in one call, sequences without queries, rows of no sequence, and more
    sequences in the tables than tokens."""
    g = torch.Generator(device=DEV).manual_seed(d)
    bs = 16
    for new, lens in (([1, 1, 0, 200, 3, 1], [70, 1, 50, 333, 3, 900]), ([0, 0, 1], [5, 0, 18]), ([129, 128, 1, 1, 127], [129, 500, 0, 1, 100])):
        total = sum(-(-n // bs) for n in lens) + 1
        pages = ref.random_pages(g, total, H, bs, d, E4M3)
        table = ref.random_tables(lens, bs, total, 5).to(DEV)
        starts = np.r_[0, np.cumsum(new)].tolist()
        q = torch.randn(starts[-1] + 6, H * G + 2, d, generator=g, device=DEV).to(x_dtype)[:, :H * G]
        _check_attention(q, pages, table, _i32(lens), starts=starts, max_q_len=max(new))
        _check_attention(q, pages, table, _i32(lens), starts=starts, max_kv_len=5000)      # bounds that are far too large


def test_attention_over_a_long_cache():
    """Splits of many granules a warp, and lengths of which most splits are empty."""
    g = torch.Generator(device=DEV).manual_seed(0)
    H, G, bs, d = 8, 4, 16, 64
    lens = [16000, 1] + [100] * 62
    total = sum(-(-n // bs) for n in lens)
    pages = ref.random_pages(g, total, H, bs, d, INT8)
    table = ref.random_tables(lens, bs, total, 1).to(DEV)
    for x_dtype in (torch.float32, torch.bfloat16):
        _check_attention(torch.randn(64, H * G, 1, d, generator=g, device=DEV).to(x_dtype), pages, table, _i32(lens))


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,H,G,q_len", [(128, 2, 4, 70), (64, 1, 8, 33), (128, 1, 1, 257), (64, 2, 40, 1), (128, 1, 40, 3)])
def test_pieces_of_prompts_over_a_long_cache(d, H, G, q_len, x_dtype):
    """Few query rows over many tokens, so that the tokens are split; many token tiles in a row; more heads than a tile of
    rows; a scale below zero."""
    g = torch.Generator(device=DEV).manual_seed(q_len)
    bs, lens = 48, [5000, 130, 2100]
    total = sum(-(-n // bs) for n in lens) + 2
    pages = ref.random_pages(g, total, H, bs, d, E4M3, "nhd")
    table = ref.random_tables(lens, bs, total, q_len).to(DEV)
    q = torch.randn(3, H * G, q_len, d, generator=g, device=DEV).to(x_dtype)
    _check_attention(q, pages, table, _i32(lens), scale=-0.1)
    starts = [0, q_len, q_len + 1, 2 * q_len + 1]
    flat = q.transpose(1, 2).reshape(-1, H * G, d)[:starts[-1] + 2].contiguous()
    _check_attention(flat, pages, table, _i32(lens), starts=starts, max_q_len=q_len)


def _a_wait_runs_out(d):
    from quashkv_b200 import _lib
    g = torch.Generator(device=DEV).manual_seed(1)
    pages = ref.random_pages(g, 80, 2, 16, d, E4M3)
    table = ref.random_tables([600, 500], 16, 80, 1).to(DEV)
    q = torch.randn(2, 4, 300, d, generator=g, device=DEV).bfloat16()
    want = paged8.attention_paged8(q, *pages, table, _i32([600, 500]), 600, causal=True)
    before = _lib.lib().qkv_tensor_core_timeouts()
    os.environ["QUASHKV_B200_TEST_DROP_MMA"] = "1"
    got = paged8.attention_paged8(q, *pages, table, _i32([600, 500]), 600, causal=True)
    torch.cuda.synchronize()
    del os.environ["QUASHKV_B200_TEST_DROP_MMA"]
    assert _lib.lib().qkv_tensor_core_timeouts() > before
    bad = got.isnan().all(-1)
    assert bad.any() and not bad[1].any() and not bad[0, 2:].any() and torch.equal(got[~bad], want[~bad])
    assert torch.equal(paged8.attention_paged8(q, *pages, table, _i32([600, 500]), 600, causal=True), want)


@pytest.mark.parametrize("d,H,G", [(128, 2, 4), (64, 3, 5), (128, 1, 32)])
def test_a_padded_ragged_batch(d, H, G):
    """Many sequences, most of one token, some of pieces that end anywhere in a tile of rows; rows in front of the first
    sequence and far behind the last; more rows allowed for a sequence than any has, and fewer."""
    g = torch.Generator(device=DEV).manual_seed(G)
    for new, front, behind in (([1] * 30 + [9, 500, 1, 0, 65, 64, 63, 0, 1], 0, 700), ([300] + [1] * 70, 3, 1), ([1] * 40 + [128] * 3, 5, 0), ([40] * 33, 0, 2000)):
        lens = [n + (37 * i) % 900 for i, n in enumerate(new)]
        total = sum(-(-n // 16) for n in lens) + 1
        pages = ref.random_pages(g, total, H, 16, d, INT8, "nhd")
        table = ref.random_tables(lens, 16, total, 5).to(DEV)
        starts = (front + np.r_[0, np.cumsum(new)]).tolist()
        q = torch.randn(starts[-1] + behind, H * G, d, generator=g, device=DEV).bfloat16()
        torch.full_like(q, math.nan)                         # (what the result's memory may hold)
        _check_attention(q, pages, table, _i32(lens), starts=starts)
        torch.full_like(q, math.nan)
        got = paged8.attention_paged8(q, *pages, table, _i32(lens), max(lens), query_starts=_i32(starts), max_q_len=60, causal=True)
        exact, bound = ref.attention(q, pages, table, _i32(lens), 1 / math.sqrt(d), True, starts)
        for i, n in enumerate(new):                          # the rows that are allowed for see what they saw
            kept = slice(starts[i], starts[i] + min(n, 60))
            assert ((got[kept].double() - exact[kept]).abs() <= bound[kept]).all()
            assert not got[starts[i] + min(n, 60):starts[i + 1]].any()
        assert not got[:front].any() and not got[starts[-1]:].any()


def test_graphs_of_a_mixed_batch_on_two_streams():
    """Prompt pieces and single tokens over caches long enough that both are split, captured twice and replayed side by
    side with lengths that change between replays."""
    g = torch.Generator(device=DEV).manual_seed(3)
    H, G, d, bs, n, T = 2, 4, 128, 16, 12, 160
    pages = ref.random_pages(g, n * 400, H, bs, d, E4M3)
    table = ref.random_tables([6400] * n, bs, n * 400, 1).to(DEV)
    sides = []
    for _ in range(2):
        q, lens, starts = torch.randn(T, H * G, d, generator=g, device=DEV).bfloat16(), _i32([1] * n), _i32([0] * (n + 1))
        call = lambda q=q, lens=lens, starts=starts: paged8.attention_paged8(q, *pages, table, lens, 6400, causal=True, query_starts=starts)      # noqa: E731
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            call()
        stream.synchronize()
        with torch.cuda.graph(graph):
            out = call()
        sides.append((q, lens, starts, call, stream, graph, out))
    rs = np.random.RandomState(0)
    for step in range(6):
        for q, lens, starts, call, stream, graph, out in sides:
            new = np.ones(n, dtype=np.int64)
            new[rs.randint(n)] = [1, 40, 149, 9, 100, 0][step]
            lens.copy_(_i32(rs.randint(149, 6400, n)))
            starts.copy_(_i32(np.r_[0, np.cumsum(new)]))
        want = [side[3]() for side in sides]
        torch.cuda.synchronize()
        for _ in range(3):
            for side in sides:
                with torch.cuda.stream(side[4]):
                    side[5].replay()
        torch.cuda.synchronize()
        for side, exact in zip(sides, want):
            assert torch.equal(side[6], exact)
            _check_attention(side[0], pages, table, side[1], starts=side[2].tolist(), max_kv_len=6400)


@pytest.mark.parametrize("d", [64, 128])
def test_a_wait_that_runs_out_gives_nan_and_is_counted(d):
    """The first CTA leaves out the products of one tile (nothing is left in flight): its waits give up, its rows are NaN
    and no others, and the context stays usable.  In a process of its own: others count the waits of this one."""
    here = os.path.dirname(os.path.abspath(__file__))
    path = os.pathsep.join([here, os.path.dirname(here), os.environ.get("PYTHONPATH", "")])
    child = subprocess.run([sys.executable, "-c", f"import test_gpu_paged8 as t; t._a_wait_runs_out({d})"], timeout=300, capture_output=True,
                           text=True, env={**os.environ, "PYTHONPATH": path})
    assert child.returncode == 0, child.stderr


@pytest.mark.parametrize("q_len", [1, 90])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float32])
def test_what_is_hidden_may_be_anything(q_len, x_dtype):
    """NaN codes and scales behind the last token, pages that do not exist, NaN scales of pages that only later rows see."""
    g = torch.Generator(device=DEV).manual_seed(4)
    H, G, bs, d = 2, 4, 16, 128
    lens = [37, 100, 5, 0, 120]
    total = 30
    pages = ref.random_pages(g, total, H, bs, d, E4M3)
    table = ref.random_tables(lens, bs, total, 2).to(DEV)
    used = {int(p) for i, n in enumerate(lens) for p in table[i, :-(-n // bs)]}
    codes = [pages[0].view(torch.uint8), pages[1].view(torch.uint8)]
    for p in range(total):
        if p not in used:
            for c in codes:
                c[p] = 0x7f
            pages[2][p] = pages[3][p] = float("nan")
    for i, n in enumerate(lens):
        if n % bs:
            for c in codes:
                c[int(table[i, n // bs]), :, n % bs:] = 0xff
    q = torch.randn(5, H * G, q_len, d, generator=g, device=DEV).to(x_dtype)
    _check_attention(q, pages, table, _i32(lens))
    table[1, 2], table[1, 4], table[4, 0], table[0, 2] = -1, total, 2 ** 31 - 1, -2 ** 31
    _check_attention(q, pages, table, _i32(lens))
    pages[3][int(table[1, 6]), 0] = float("nan")            # seen by the last rows of one head only
    pages[2][int(table[4, 6]), 1] = float("nan")
    _check_attention(q, pages, table, _i32(lens))


@pytest.mark.parametrize("q_len", [1, 70])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_scales_of_any_size(q_len, x_dtype):
    """Pages whose value scales lie 2^40 apart, zeros among them, with rows that weigh mostly the small ones; queries far from 1."""
    g = torch.Generator(device=DEV).manual_seed(6)
    H, G, bs, d = 2, 2, 16, 64
    lens = [200, 90]
    pages = ref.random_pages(g, 19, H, bs, d, INT8)
    table = ref.random_tables(lens, bs, 19, 3).to(DEV)
    q = torch.randn(2, H * G, q_len, d, generator=g, device=DEV)
    pages[3].mul_(torch.exp2(torch.randint(-20, 21, pages[3].shape, generator=g, device=DEV).float()))
    pages[3][int(table[0, 1])] = 0
    pages[3][int(table[1, 0])] = 0
    pages[2][int(table[0, 3])] = 0
    big = 2.0 ** 10 if x_dtype == torch.float16 else 2.0 ** 60
    for up in (1.0, big, 1 / big):
        _check_attention((q * up).to(x_dtype), pages, table, _i32(lens), scale=3 / up / math.sqrt(d))
    pages[3].fill_(0)                                        # nothing to sum
    _check_attention(q.to(x_dtype), pages, table, _i32(lens))
    # the page that nearly all weight falls on holds small values, another one large ones
    pages = ref.random_pages(g, 19, H, bs, d, INT8)
    pages[3].copy_(torch.where(torch.arange(19, device=DEV)[:, None] == int(table[0, 2]), 2.0 ** -12, 2.0 ** 12))
    pages[2][int(table[0, 2])] *= 60
    _check_attention(q.to(x_dtype), pages, table, _i32(lens))


def test_rows_with_infinities_and_nan_keep_to_themselves():
    g = torch.Generator(device=DEV).manual_seed(7)
    pages = ref.random_pages(g, 8, 1, 16, 128, E4M3)
    table, lens = ref.random_tables([100], 16, 8, 3).to(DEV), _i32([100])
    q = torch.randn(1, 8, 40, 128, generator=g, device=DEV).bfloat16()
    clean = paged8.attention_paged8(q, *pages, table, lens, 100, causal=True)
    q[0, 3, 5, 7], q[0, 6, 20, 0] = float("nan"), float("inf")
    got = paged8.attention_paged8(q, *pages, table, lens, 100, causal=True)
    touched = torch.zeros(1, 8, 40, dtype=torch.bool, device=DEV)
    touched[0, 3, 5] = touched[0, 6, 20] = True
    assert got[touched].isnan().all() and torch.equal(got[~touched], clean[~touched])


def test_attention_reads_no_more_than_it_is_told():
    """Lengths beyond the bound given, beyond the table, and negative ones are clamped; a batch of none and queries of none give nothing."""
    g = torch.Generator(device=DEV).manual_seed(8)
    pages = ref.random_pages(g, 8, 2, 16, 64, E4M3)
    table = ref.random_tables([64, 64], 16, 8, 1).to(DEV)
    q = torch.randn(2, 4, 1, 64, generator=g, device=DEV)
    full = paged8.attention_paged8(q, *pages, table, _i32([64, 64]), 64)
    assert torch.equal(paged8.attention_paged8(q, *pages, table, _i32([900, 64]), 900), full)
    some = paged8.attention_paged8(q, *pages, table, _i32([40, 40]), 64)
    assert torch.allclose(paged8.attention_paged8(q, *pages, table, _i32([64, 64]), 40), some, rtol=1e-5, atol=1e-5)
    assert not paged8.attention_paged8(q, *pages, table, _i32([-5, 0]), 64).any()
    assert not paged8.attention_paged8(q, *pages, table, _i32([64, 64]), 0).any()
    assert paged8.attention_paged8(q[:, :, :0], *pages, table, _i32([64, 64]), 64).shape == (2, 4, 0, 64)
    assert paged8.attention_paged8(q[:0], *pages, table[:0], _i32([64, 64])[:0], 64).shape == (0, 4, 1, 64)
    rows = paged8.attention_paged8(q[:, :, 0], *pages, table, _i32([64, 64]), 64, query_starts=_i32([0, 1, 9]))
    assert torch.equal(rows, full[:, :, 0])                  # a start beyond the tokens
    assert not paged8.attention_paged8(q[:, :, 0], *pages, table, _i32([64, 64]), 64, query_starts=_i32([0, 0, 0])).any()


def test_wrong_arguments_are_refused():
    g = torch.Generator(device=DEV).manual_seed(9)
    pages = ref.random_pages(g, 8, 2, 16, 64, E4M3)
    table, lens, q = _i32([[0, 1]]), _i32([20]), torch.randn(1, 4, 1, 64, device=DEV)
    attend = lambda q=q, pages=pages, table=table, lens=lens, **kw: paged8.attention_paged8(q, *pages, table, lens, 20, **kw)      # noqa: E731
    k, v, ks, vs = pages
    for bad in (dict(q=q[0]), dict(q=q[..., :32]), dict(q=torch.randn(1, 3, 1, 64, device=DEV)), dict(q=q.expand(2, 4, 1, 64)), dict(lens=lens.long()),
                dict(table=table.long()), dict(table=table[0]), dict(lens=_i32([1, 2])), dict(pages=(k, v.view(INT8), ks, vs)),
                dict(pages=(k.view(torch.uint8), v.view(torch.uint8), ks, vs)), dict(pages=(k, v, ks.double(), vs)), dict(pages=(k, v, ks[:7], vs)),
                dict(pages=(k[:7], v, ks, vs)), dict(pages=(k.transpose(2, 3), v.transpose(2, 3), ks, vs)), dict(query_starts=_i32([0, 1])),
                dict(lens=lens.cpu()), dict(table=table.cpu()), dict(pages=(k.cpu(), v, ks, vs)), dict(q=q[:, :, 0], query_starts=_i32([0, 1, 2]))):
        with pytest.raises(ValueError):
            attend(**bad)
    for bad in (dict(pages=tuple(ref.random_pages(g, 4, 2, 8, 64, E4M3))), dict(q=q[..., :48], pages=tuple(p[..., :48] if p.dim() == 4 else p for p in pages))):
        with pytest.raises(RuntimeError, match="failed"):
            attend(**bad)
    x, slots = torch.randn(3, 2, 64, device=DEV), torch.arange(3, device=DEV)
    for bad in ((x, x[:2], slots), (x, x.half(), slots), (x[:, :1], x[:, :1], slots), (x, x, slots.int()), (x, x, slots[:2]), (x, x, slots.cpu()), (x, x, None)):
        with pytest.raises(ValueError):
            paged8.append_paged8(bad[0], bad[1], *pages, bad[2])
    i = _i32([0])
    for bad in ((table.long(), i, i, i, _i32([1, 0])), (table, i, i, i, i), (table, _i32([0, 0]), i, i, _i32([1, 0])), (table, i, i.long(), i, _i32([1, 0])),
                (table, i, i, i.cpu(), _i32([1, 0]))):
        with pytest.raises(ValueError):
            paged8.extend_pages(*bad, 16, 4)
    with pytest.raises(ValueError):
        paged8.extend_pages(table, i, i, i, _i32([1, 0]), 0, 4)


def test_a_call_on_another_stream_and_two_at_once():
    g = torch.Generator(device=DEV).manual_seed(10)
    lens = [3000, 700]
    pages = ref.random_pages(g, 240, 2, 16, 128, E4M3)
    table = ref.random_tables(lens, 16, 240, 1).to(DEV)
    q = torch.randn(2, 8, 1, 128, generator=g, device=DEV).bfloat16()
    want = paged8.attention_paged8(q, *pages, table, _i32(lens), 3000)
    torch.cuda.synchronize()
    n, streams, outs = _i32(lens), [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(paged8.attention_paged8(q, *pages, table, n, 3000))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---- together ---------------------------------------------------------------------------------------------------------------

def _serve(codes, layout, graph):
    """A loop over six rows: prompts arrive, every request decodes, drafts are taken back, requests end and others take
    their pages.  Each step's codes equal those of appends by the definition, and its attention is that over them."""
    H, G, d, bs, rows, T = 2, 4, 64, 16, 6, 80
    g = torch.Generator(device=DEV).manual_seed(11)
    dtype = paged8.CODES[codes]
    cache = paged8.QuashKVPaged8Cache(40, H, d, block_size=bs, codes=codes, layout=layout)
    tables = paged8.PageTables(40, rows, 12, block_size=bs)
    new, x = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros(T, 2 * H + H * G, d, device=DEV, dtype=torch.bfloat16)

    def step():
        plan = tables.extend(new, T)
        cache.append_slots(x[:, :H], x[:, H:2 * H], plan.slots)
        out = cache.attention_with_tables(x[:, 2 * H:], tables.block_table, tables.seq_lens, 12 * bs, causal=True,
                                          query_starts=plan.query_starts, max_q_len=T)
        return plan, out
    run = step
    if graph:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()                                           # (no new tokens: changes nothing)
        side.synchronize()
        record = torch.cuda.CUDAGraph()
        with torch.cuda.graph(record):
            kept = step()

        def run():
            record.replay()
            return kept
    held, free, pool = [0] * rows, tables.free_pages.tolist(), tables.pool.tolist()
    table = tables.block_table.cpu().numpy()
    want = _host(cache.planes)
    for asked, keep in (([30, 0, 17, 0, 0, 1], None), ([1, 25, 1, 0, 0, 1], None), ([4, 4, 4, 0, 0, 4], [31, 28, 19, 0, 0, 3]),
                        ([1, 1, 1, 60, 1, 1], [0, 29, 20, 60, 1, 0]), ([50, 1, 1, 1, 1, 5], None), ([1, 1, 70, 1, 1, 1], [51, 0, 90, 0, 3, 0]),
                        ([1, 64, 1, 0, 0, 0], None)):
        new.copy_(_i32(asked))
        x.copy_(torch.randn(x.shape, generator=g, device=DEV) * 2)
        plan, out = run()
        table, slots, starts, after, pool = ref.extend(table, held, asked, free, pool, bs, T)
        assert plan.slots.tolist() == slots and plan.query_starts.tolist() == starts and tables.seq_lens.tolist() == after
        assert plan.start_lens.tolist() == held and tables.pool.tolist() == pool and -1 not in slots[:starts[-1]]
        xs = x.float().cpu().numpy().astype(np.float64)
        ref.append(xs[:, :H], want[0], want[2], slots, bs, dtype)
        ref.append(xs[:, H:2 * H], want[1], want[3], slots, bs, dtype)
        for got, exact in zip(_host(cache.planes), want):
            assert np.array_equal(got, exact)
        exact, bound = ref.attention(x[:, 2 * H:], cache.planes, tables.block_table, tables.seq_lens, 1 / math.sqrt(d), True, starts)
        assert ((out.double() - exact).abs() <= bound).all()
        held = after
        if keep is not None:
            tables.shrink(_i32(keep))
            held, free, pool = ref.shrink(table, held, keep, free, pool, bs)
            assert tables.seq_lens.tolist() == held and tables.free_pages.tolist() == free and tables.pool.tolist() == pool
    tables.release(torch.ones(rows, dtype=torch.bool, device=DEV))
    assert tables.free_blocks() == 40 and sorted(tables.free_pages.tolist()) == list(range(40)) and not tables.seq_lens.any()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("codes,layout", [("e4m3", "hnd"), ("int8", "nhd")])
def test_a_serving_loop(codes, layout, graph):
    _serve(codes, layout, graph)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_cache_by_sequence_ids(codes):
    """The pool's own bookkeeping: appends of any size (an id listed more than once among them) give what one append gives but for
    the rounding of codes that moved to a larger scale; attention is that over the decompressed cache."""
    g = torch.Generator(device=DEV).manual_seed(12)
    H, G, d = 2, 2, 64
    cache = paged8.QuashKVPaged8Cache(32, H, d, codes=codes)
    K, V = torch.randn(2, H, 60, d, generator=g, device=DEV), torch.randn(2, H, 60, d, generator=g, device=DEV)
    cache.append(["a", "b"], K[:, :, :20], V[:, :, :20])
    both = lambda X, i, lo, hi: X[i, :, lo:hi]      # noqa: E731
    cut = lambda X: torch.stack([both(X, 0, 20, 25), both(X, 1, 20, 25), both(X, 0, 25, 30), both(X, 0, 30, 35)])      # noqa: E731
    cache.append(["a", "b", "a", "a"], cut(K), cut(V))
    for t in range(35, 60):
        cache.append(["a"], K[:1, :, t:t + 1], V[:1, :, t:t + 1])
    assert cache.seq_len("a") == 60 and cache.seq_len("b") == 25
    step = 2.0 ** -4 if codes == "e4m3" else 1 / 127
    for i, s in enumerate("ab"):
        n = cache.seq_len(s)
        for got, X in zip(cache.decompress(s), (K, V)):
            x = X[i, :, :n]
            top = torch.nn.functional.pad(x, (0, 0, 0, -n % 16)).reshape(H, -1, 16, d).abs().amax((2, 3)).repeat_interleave(16, 1)[:, :n, None]
            # a code is off by half a step, of its own size (e4m3; of the subnormal ones 2^-10 of a scale that is at most top / 224) or of the
            # scale (int8, at most top / 63.5); at a raised scale the old code is rounded again, each time to a step at least twice the last
            if codes == "e4m3":
                assert ((got - x).abs() <= x.abs() * step * (1 + step) + 2 * top / 224 * 2.0 ** -10).all()
            else:
                assert ((got - x).abs() <= top / 63.5).all()
    q = torch.randn(2, H * G, 1, d, generator=g, device=DEV)
    out = cache.attention(["a", "b"], q)
    for i, s in enumerate("ab"):
        k, v = (t.double().repeat_interleave(G, 0) for t in cache.decompress(s))
        w = torch.softmax((q[i].double() @ k.transpose(1, 2)) / math.sqrt(d), -1)
        assert torch.allclose(out[i].double(), w @ v, rtol=1e-5, atol=1e-5)
    cache.free("a")
    assert cache.free_blocks == 30
    with pytest.raises(ValueError):
        cache.append(["a"], K, V)
    with pytest.raises(ValueError):
        cache.attention(["nobody"], q[:1])


def test_device_tables_serve_the_3_bit_cache_too():
    """The tables and start lengths of a step feed QuashKVPagedCache, with the result of its own bookkeeping."""
    g = torch.Generator(device=DEV).manual_seed(13)
    H, d = 2, 128
    own, pool = QuashKVPagedCache(32, H, d), QuashKVPagedCache(32, H, d)
    tables = paged8.PageTables(32, 3, 8)
    q = torch.randn(3, 2 * H, 1, d, generator=g, device=DEV)
    for T in (20, 1, 1, 13):
        K, V = torch.randn(3, H, T, d, generator=g, device=DEV), torch.randn(3, H, T, d, generator=g, device=DEV)
        own.append(["a", "b", "c"], K, V)
        plan = tables.extend(torch.full((3,), T, dtype=torch.int32, device=DEV), 3 * T)
        pool.append_with_tables(K, V, tables.block_table, plan.start_lens)
        a, b = own.attention(["a", "b", "c"], q), pool.attention_with_tables(q, tables.block_table, tables.seq_lens, 40)
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
