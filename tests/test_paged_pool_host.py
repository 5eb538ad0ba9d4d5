"""Bookkeeping of the page pools without a GPU: an append that cannot be carried out changes nothing."""

import pytest
import torch

from quashkv_b200 import ops
from quashkv_b200.integrations import paged8
from quashkv_b200.integrations.vllm_backend import QuashKVPagedCache

T = 20                                                       # two pages of 16 for a new sequence


def _pools():
    return [paged8.QuashKVPaged8Cache(6, 1, 32, device="cpu"), QuashKVPagedCache(6, 1, 32, device="cpu")]


@pytest.fixture
def stores(monkeypatch):
    """The appends of both pools as records of their starts and tables; raises where `fail` counts down to 0."""
    calls, fail = [], [-1]

    def store(table, starts):
        fail[0] -= 1
        if fail[0] == 0:
            raise ValueError("refused")
        calls.append((starts.tolist(), table.tolist()))
    monkeypatch.setattr(ops, "_need_cuda", lambda t, what: None)
    monkeypatch.setattr(ops, "append_paged8", lambda k, v, kc, vc, ks, vs, slots, table, starts: store(table, starts))
    monkeypatch.setattr(QuashKVPagedCache, "_store", lambda self, k, v, table, starts: store(table, starts))
    return calls, fail


def _state(pool, ids="abcd"):
    return ([pool.seq_len(s) for s in ids], [pool.blocks_of(s) for s in ids], list(pool._free), sorted(pool._blocks), sorted(pool._lens))


def _x(n):
    return torch.zeros(n, 1, T, 32)


@pytest.mark.parametrize("which", [0, 1])
def test_an_append_that_exhausts_the_pool_changes_nothing(which, stores):
    pool = _pools()[which]
    pool.append(["a"], _x(1), _x(1))
    before = _state(pool)
    for ids in (["b", "c", "d"], ["a", "a", "a", "a", "a"], ["b", "a", "b", "b"]):      # the last entries find no page
        with pytest.raises(RuntimeError, match="pool exhausted"):
            pool.append(ids, _x(len(ids)), _x(len(ids)))
        assert _state(pool) == before
    assert len(stores[0]) == 1
    pool.free("a")                                           # what was refused fits then, at its own positions
    pool.append(["b", "c", "d"], _x(3), _x(3))
    assert stores[0][-1][0] == [0, 0, 0] and pool.free_blocks == 0 and [pool.seq_len(s) for s in "bcd"] == [T] * 3


@pytest.mark.parametrize("which", [0, 1])
def test_an_append_whose_store_is_refused_changes_nothing(which, stores):
    pool = _pools()[which]
    pool.append(["a"], _x(1), _x(1))
    before = _state(pool)
    for nth in ([1, 2] if which == 0 else [1]):              # (an id listed twice takes two stores in the 8-bit pool)
        stores[1][0] = nth
        with pytest.raises(ValueError, match="refused"):
            pool.append(["b", "a", "a"], _x(3), _x(3))
        assert _state(pool) == before
    pool.append(["b", "a", "a"], _x(3), _x(3))
    assert pool.seq_len("a") == 3 * T and pool.seq_len("b") == T and pool.free_blocks == 0
    pool.clear()
    assert pool.free_blocks == 6 and pool.seq_len("a") == 0


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_decompress_of_a_sequence_without_tokens(codes, layout):
    pool = paged8.QuashKVPaged8Cache(6, 2, 32, codes=codes, layout=layout, device="cpu")
    for x in pool.decompress("nobody"):
        assert x.shape == (2, 0, 32) and x.dtype == torch.float32
    pool._grow("a", T)
    pool._lens["a"] = T
    pool.k_scales.fill_(2.0)
    pool.k_codes.view(torch.uint8).fill_(0x38 if codes == "e4m3" else 1)      # 1
    k, v = pool.decompress("a")
    assert k.shape == v.shape == (2, T, 32) and (k == 2).all() and not v.any()
