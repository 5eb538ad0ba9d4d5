"""Rows of attention over 8-bit pages that belong to no sequence or see no token: zeros, in an output whose memory held NaN
(the C entry writes to the caller's tensor; what an allocator hands out may be zeros already)."""

import ctypes
import math

import numpy as np
import pytest
import torch

import paged8_reference as ref
from quashkv_b200 import _lib
from quashkv_b200.integrations import paged8

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
I64 = ctypes.c_int64


def _i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(DEV)


def attend_into(out, q, pages, table, lens, max_kv_len, starts=None, max_q_len=None, causal=True, entry="qkv_attention_paged8", extra=()):
    """qkv_attention_paged8 on the current stream, into `out` (like q: (n, Hq, q_len, d), or ragged (T, Hq, d))."""
    L, (k, v, ks, vs) = _lib.lib(), pages
    p = _lib.Pages8()
    p.k_codes, p.v_codes, p.k_scales, p.v_scales = (t.data_ptr() for t in pages)
    for i in range(3):
        p.k_stride[i], p.v_stride[i] = k.stride(i), v.stride(i)
    for i in range(2):
        p.ks_stride[i], p.vs_stride[i] = ks.stride(i), vs.stride(i)
    p.num_blocks, p.Hkv, p.block_size, p.d = k.shape
    p.code = int(k.dtype == INT8)
    n, d, dtype = table.shape[0], q.shape[-1], {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[q.dtype]
    ragged = starts is not None
    total, q_len = (q.shape[0], q.shape[0] if max_q_len is None else min(max_q_len, q.shape[0])) if ragged else (0, q.shape[2])      # as the op does
    strides = lambda t: (I64 * 3)(0, t.stride(0), t.stride(1)) if ragged else (I64 * 3)(t.stride(0), t.stride(2), t.stride(1))      # noqa: E731
    need = L.qkv_attention_paged8_workspace_bytes(n, q.shape[1], p.Hkv, q_len, int(ragged), total, max_kv_len, d, dtype)
    ws = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device=DEV)
    rc = getattr(L, entry)(q.data_ptr(), dtype, strides(q), p, table.data_ptr(), table.stride(0), table.shape[1], lens.data_ptr(),
                           starts.data_ptr() if ragged else None, total, *extra, n, q.shape[1], q_len, max_kv_len, 1 / math.sqrt(d), int(causal),
                           out.data_ptr(), strides(out), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, rc
    return out


def test_dtype_numbers_of_the_c_interface():
    from quashkv_b200 import ops
    assert {t: ops._DT[t] for t in (torch.float32, torch.bfloat16, torch.float16)} == {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,H,G", [(128, 2, 4), (64, 2, 8), (128, 1, 1)])
def test_prompts_that_see_nothing_are_zeros(d, H, G, x_dtype):
    """Many sequences without a token, and row tiles in front of a short sequence's first position: nothing orders the warps of
    such a CTA but what the kernel does for it.  Queries are not zero, caches are cold or warm."""
    g = torch.Generator(device=DEV).manual_seed(d + G)
    q_len, n = -(-600 // G) + 7, 200
    lens = [0, 1, 0, 0, 40, 0] * (n // 6) + [0] * (n % 6)
    pages = ref.random_pages(g, 3 * n, H, 16, d, E4M3)
    table = ref.random_tables([48] * n, 16, 3 * n, 1).to(DEV)
    q = torch.randn(n, q_len, H * G, d, generator=g, device=DEV).to(x_dtype).transpose(1, 2)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    seen = torch.tensor([[max(0, min(m, m - q_len + t + 1)) for t in range(q_len)] for m in lens], device=DEV) > 0
    starts = _i32(np.arange(n + 1) * q_len)
    flat = q.transpose(1, 2).reshape(n * q_len, H * G, d)
    for turn in range(6):
        out = torch.full((n, q_len, H * G, d), math.nan, dtype=x_dtype, device=DEV)
        flush.fill_(turn)
        attend_into(out.transpose(1, 2), q, pages, table, _i32(lens), 48)
        assert not out[~seen].view(torch.int16).any() and out[seen].isfinite().all() and out[seen].any(-1).all()
        rows = torch.full_like(flat, math.nan)               # the same sequences as a ragged batch
        flush.fill_(turn)
        attend_into(rows, flat, pages, table, _i32(lens), 48, starts=starts, max_q_len=q_len)
        rows = rows.view(n, q_len, H * G, d)
        assert not rows[~seen].view(torch.int16).any() and rows[seen].isfinite().all()
    every = torch.full((n, q_len, H * G, d), math.nan, dtype=x_dtype, device=DEV)      # a bound of no tokens at all
    attend_into(every.transpose(1, 2), q, pages, table, _i32(lens), 0, causal=False)
    assert not every.view(torch.int16).any()


RAGGED = [([1] * 30 + [9, 500, 1, 0, 65, 64, 63, 0, 1], 0, 700), ([300] + [1] * 70, 3, 1), ([1] * 40 + [128] * 3, 5, 0), ([40] * 33, 0, 2000),
          ([1] * 9, 2, 40), ([0, 0, 3, 0], 7, 9), ([0, 0], 0, 33), ([200], 1, 1)]


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,H,G", [(128, 2, 4), (64, 3, 5), (128, 1, 40), (96, 2, 2), (32, 1, 1)])
def test_rows_of_no_sequence_are_cleared(d, H, G, x_dtype):
    """Rows in front of the first sequence, behind the last one, and beyond the most that a sequence is allowed; sequences
    without a token; partial sums in a workspace that held NaN.  Everything else is what the public call gives."""
    g = torch.Generator(device=DEV).manual_seed(G)
    for new, front, behind in RAGGED:
        for long in (0, 5000):                               # short caches, and one that is split
            lens = [0 if i % 11 == 7 else n + (37 * i) % 900 + (long if i == 0 else 0) for i, n in enumerate(new)]
            total = sum(-(-m // 16) for m in lens) + 1
            pages = ref.random_pages(g, total, H, 16, d, INT8, "nhd")
            table = ref.random_tables(lens, 16, total, 5).to(DEV)
            starts = front + np.r_[0, np.cumsum(new)]
            q = torch.randn(starts[-1] + behind, H * G, d, generator=g, device=DEV).to(x_dtype)
            for most in (q.shape[0], 60):
                out = torch.full_like(q, math.nan)
                attend_into(out, q, pages, table, _i32(lens), max(max(lens), 1), starts=_i32(starts), max_q_len=most)
                none = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
                for i, n in enumerate(new):
                    see = torch.arange(min(n, most), device=DEV) + lens[i] - n + 1 > 0
                    none[starts[i]:starts[i] + min(n, most)] = ~see
                bits = out.view(torch.int16 if x_dtype == torch.bfloat16 else torch.int32)
                assert not bits[none].any() and out.isfinite().all() and out[~none].any(-1).all()
                assert torch.equal(out, paged8.attention_paged8(q, *pages, table, _i32(lens), max(max(lens), 1), causal=True,
                                                                query_starts=_i32(starts), max_q_len=most))


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,H,G,q_len", [(128, 2, 4, 1), (64, 2, 8, 1), (96, 1, 3, 5), (32, 4, 1, 2), (128, 1, 4, 90)])
def test_every_row_of_a_dense_batch_is_written(d, H, G, q_len, x_dtype):
    g = torch.Generator(device=DEV).manual_seed(q_len)
    for lens in ([0], [0, 0, 1], [1000, 0, 17, 3], [0] * 40 + [6000]):
        total = sum(-(-m // 16) for m in lens) + 1
        pages = ref.random_pages(g, total, H, 16, d, E4M3)
        table = ref.random_tables(lens, 16, total, 2).to(DEV)
        q = torch.randn(len(lens), H * G, q_len, d, generator=g, device=DEV).to(x_dtype)
        out = attend_into(torch.full_like(q, math.nan), q, pages, table, _i32(lens), max(max(lens), 1))
        see = torch.tensor([[m - q_len + t + 1 > 0 for t in range(q_len)] for m in lens], device=DEV)[:, None].expand(-1, H * G, -1)
        assert out.isfinite().all() and not out[~see].view(torch.int16).any() and out[see].any(-1).all()
        assert torch.equal(out, paged8.attention_paged8(q, *pages, table, _i32(lens), max(max(lens), 1), causal=True))


def test_queries_of_other_types_are_taken_as_fp32():
    g = torch.Generator(device=DEV).manual_seed(0)
    pages = ref.random_pages(g, 8, 2, 16, 64, INT8)
    table, lens = ref.random_tables([64, 50], 16, 8, 1).to(DEV), _i32([64, 50])
    q = torch.randint(-3, 4, (2, 4, 3, 64), generator=g, device=DEV)
    want = paged8.attention_paged8(q.float(), *pages, table, lens, 64, causal=True)
    for x in (q, q.double()):
        got = paged8.attention_paged8(x, *pages, table, lens, 64, causal=True)
        assert got.dtype == torch.float32 and torch.equal(got, want)


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_len", [1, 90])
def test_the_least_value_scales(q_len, x_dtype):
    """2^-126 is a scale like any other; subnormal ones count as 0."""
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v, ks, vs = ref.random_pages(g, 8, 2, 16, 128, INT8)
    table, lens = ref.random_tables([100], 16, 8, 1).to(DEV), _i32([100])
    q = torch.randn(1, 8, q_len, 128, generator=g, device=DEV).to(x_dtype)
    call = lambda s: paged8.attention_paged8(q, k, v, ks, torch.full_like(vs, s), table, lens, 100, causal=True)      # noqa: E731
    assert torch.allclose(call(2.0 ** -126).double() * 2.0 ** 126, call(1.0).double(), rtol=0.02, atol=2.0 ** -7)
    assert not call(2.0 ** -127).any() and not call(2.0 ** -149).any()
