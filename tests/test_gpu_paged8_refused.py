"""A step in which the pool runs out: the tokens that were stored see what they would have seen otherwise."""

import math

import numpy as np
import pytest
import torch

import paged8_reference as ref
from quashkv_b200.integrations import paged8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(DEV)


def _check(out, q, pages, table, before, after, starts, scale):
    """Row t of sequence i at position before[i] + t, seeing the positions up to it of the after[i] that are held."""
    want, bound = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for i in range(len(before)):
        kept = after[i] - before[i]
        for lo, hi, causal in ((starts[i], starts[i] + kept, True), (starts[i] + kept, starts[i + 1], False)):      # stored, refused
            want[lo:hi], bound[lo:hi] = ref.attention(q[lo:hi], pages, table[i:i + 1], _i32(after[i:i + 1]), scale, causal, [0, hi - lo])
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,H,G", [(64, 2, 4), (128, 1, 8)])
def test_a_step_that_exhausts_the_pool(d, H, G, x_dtype, graph):
    """Single tokens, short blocks and pieces of prompts, of which the last find no page or a full row; then a step in which no token does."""
    g = torch.Generator(device=DEV).manual_seed(d)
    n, bs, width, T = 5, 16, 20, 320
    cache = paged8.QuashKVPaged8Cache(42, H, d, block_size=bs)
    tables = paged8.PageTables(42, n, width, block_size=bs)
    x = torch.zeros(T, (2 + G) * H, d, device=DEV, dtype=x_dtype)
    new = torch.zeros(n, dtype=torch.int32, device=DEV)

    def step():
        plan = tables.extend(new, T)
        cache.append_slots(x[:, :H], x[:, H:2 * H], plan.slots)
        return plan, cache.attention_with_tables(x[:, 2 * H:], tables.block_table, tables.seq_lens, width * bs, causal=True,
                                                 query_starts=plan.query_starts, start_lens=plan.start_lens)
    run = step
    if graph:
        with torch.cuda.stream(torch.cuda.Stream()):
            step()
        torch.cuda.synchronize()
        record = torch.cuda.CUDAGraph()
        with torch.cuda.graph(record):
            kept = step()

        def run():
            record.replay()
            return kept
    held, refused = [0] * n, 0
    for asked in ([100, 10, 1, 0, 200], [30, 1, 100, 3, 150], [1, 40, 90, 70, 1], [9, 9, 9, 9, 60]):
        new.copy_(_i32(asked))
        x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        plan, out = run()
        starts, after = plan.query_starts.tolist(), tables.seq_lens.tolist()
        assert plan.start_lens.tolist() == held and starts == np.r_[0, np.cumsum(asked)].tolist()
        refused += sum(asked) - (sum(after) - sum(held))
        _check(out, x[:, 2 * H:], cache.planes, tables.block_table, held, after, starts, 1 / math.sqrt(d))
        assert not out[starts[-1]:].any()
        held = after
    assert tables.refused_tokens() == refused > 100 and tables.free_blocks() == 0


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_len", [1, 5, 90])
def test_positions_of_a_dense_batch(q_len, x_dtype):
    """Blocks of queries at any position of what is held, beyond it, and in front of all of it; splits that are joined among them."""
    g = torch.Generator(device=DEV).manual_seed(q_len)
    H, G, bs, d, lens = 2, 4, 16, 128, [4000, 300, 1, 0, 128]
    total = sum(-(-m // bs) for m in lens)
    pages = ref.random_pages(g, total, H, bs, d, torch.int8)
    table = ref.random_tables(lens, bs, total, 1).to(DEV)
    q = torch.randn(len(lens), H * G, q_len, d, generator=g, device=DEV).to(x_dtype)
    call = lambda first: paged8.attention_paged8(q, *pages, table, _i32(lens), 4000, causal=True, start_lens=_i32(first))      # noqa: E731
    plain = paged8.attention_paged8(q, *pages, table, _i32(lens), 4000, causal=True)
    assert torch.equal(call([max(m - q_len, 0) for m in lens])[:2], plain[:2])      # its last positions: the same rows
    for first in ([0, 0, 0, 0, 0], [3999, 299, 0, 0, 127], [2000, 150, 5, 7, 100], [-3, -1, -1, -1, -1]):
        got = call(first)
        for i, (m, at) in enumerate(zip(lens, first)):
            for t in range(0, q_len, max(1, q_len // 7)):
                see = min(max(at, 0) + t + 1, m)
                want, bound = ref.attention(q[i:i + 1, :, t:t + 1], pages, table[i:i + 1], _i32([see]), 1 / math.sqrt(d), False)
                # (the bound's splits and truncations are those of `see` tokens; the masked ones add none)
                assert ((got[i:i + 1, :, t:t + 1].double() - want).abs() <= bound).all(), (i, t)
    loose = paged8.attention_paged8(q, *pages, table, _i32(lens), 4000, causal=False, start_lens=_i32([0] * 5))      # nothing to do with it
    assert torch.equal(loose, paged8.attention_paged8(q, *pages, table, _i32(lens), 4000))
    for bad in (_i32([0, 0]), _i32([0] * 5).long(), _i32([[0] * 5]), _i32([0] * 5).cpu()):
        with pytest.raises(ValueError):
            paged8.attention_paged8(q, *pages, table, _i32(lens), 4000, causal=True, start_lens=bad)
