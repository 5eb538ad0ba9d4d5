"""The 8-bit paged cache without a GPU: refusals on the host, tracing, bookkeeping, and the index and scale arithmetic that
the kernels share with the host."""

import ctypes
import math
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import paged8_reference as ref
from quashkv_b200 import _lib
from quashkv_b200.integrations import paged8
from quashkv_b200.integrations.vllm_backend import QuashKVPagedCache

HERE = os.path.dirname(os.path.abspath(__file__))
I64 = ctypes.c_int64


def _pages(**kw):
    p = _lib.Pages8()
    p.k_codes = p.v_codes = 256
    p.k_scales = p.v_scales = 64
    for i, s in enumerate((4096, 2048, 128)):
        p.k_stride[i] = p.v_stride[i] = s
    for i, s in enumerate((2, 1)):
        p.ks_stride[i] = p.vs_stride[i] = s
    p.num_blocks, p.Hkv, p.block_size, p.d, p.code = 4, 2, 16, 128, 0
    for name, v in kw.items():
        if isinstance(v, tuple):
            for i, s in enumerate(v):
                getattr(p, name)[i] = s
        else:
            setattr(p, name, v)
    return p


BAD_PAGES = [(dict(k_codes=None), -1), (dict(v_scales=None), -1), (dict(code=2), -4), (dict(d=80), -2), (dict(d=256), -2),
             (dict(block_size=8), -2), (dict(block_size=24), -2), (dict(block_size=0), -2), (dict(Hkv=0), -2), (dict(num_blocks=0), -2),
             (dict(k_codes=264), -5), (dict(v_stride=(4096, 2048, 72)), -5), (dict(k_stride=(4096, -2048, 128)), -5),
             (dict(k_scales=66), -5), (dict(ks_stride=(-2, 1)), -8)]


@pytest.mark.parametrize("bad,code", BAD_PAGES)
def test_bad_pools_are_refused_without_launching(bad, code):
    L, one, s3 = _lib.lib(), ctypes.c_void_p(256), (I64 * 3)(0, 256, 128)
    assert L.qkv_append_paged8(one, one, 1, s3, s3, 1, 4, _pages(**bad), one, None, 0, 0, None, None) == code
    assert L.qkv_attention_paged8(one, 1, s3, _pages(**bad), one, 4, 4, one, None, 0, 1, 8, 1, 64, 1.0, 0, one, s3, one, 1 << 30, None) == code


def test_bad_arguments_are_refused_without_launching():
    L, one, s3, odd3 = _lib.lib(), ctypes.c_void_p(256), (I64 * 3)(0, 256, 128), (I64 * 3)(0, 256, 129)
    at8 = ctypes.c_void_p(264)

    def append(keys=one, values=one, dtype=1, ks=s3, vs=s3, n=1, tokens=4, slots=one, table=None, blocks=0, starts=None):
        return L.qkv_append_paged8(keys, values, dtype, ks, vs, n, tokens, _pages(), slots, table, blocks, blocks, starts, None)
    assert append(keys=None) == -1 and append(slots=None) == -1 and append(slots=None, table=one, blocks=4) == -1
    assert append(dtype=3) == -4 and append(tokens=-1) == -2 and append(slots=None, table=one, starts=one) == -2
    assert append(n=2) == -8 and append(keys=at8) == -5 and append(vs=odd3) == -5
    assert append(tokens=0) == 0                                            # nothing to do

    def attend(q=one, dtype=1, qs=s3, table=one, stride=4, blocks=4, lens=one, starts=None, total=0, n=1, hq=8, q_len=1, kv=64, out=one,
               os_=s3, ws=one, size=1 << 30):
        return L.qkv_attention_paged8(q, dtype, qs, _pages(), table, stride, blocks, lens, starts, total, n, hq, q_len, kv, 1.0, 0, out, os_, ws, size, None)
    assert attend(q=None) == -1 and attend(lens=None) == -1 and attend(table=None) == -1 and attend(out=None) == -1
    assert attend(dtype=7) == -4 and attend(hq=7) == -2 and attend(hq=0) == -2 and attend(blocks=0) == -2 and attend(stride=3) == -2
    assert attend(kv=-1) == -2 and attend(kv=1 << 31) == -2 and attend(total=-1) == -2 and attend(q_len=-1) == -2
    assert attend(q=at8) == -5 and attend(os_=odd3) == -5 and attend(ws=at8, kv=9000) == -5
    assert attend(kv=9000, size=16) == -6 and attend(kv=9000, ws=None) == -6
    assert attend(n=0) == 0 and attend(q_len=0) == 0                        # nothing to do
    assert L.qkv_attention_paged8_workspace_bytes(1, 32, 8, 1, 0, 0, 9000, 128, 1) > 0
    assert L.qkv_attention_paged8_workspace_bytes(1, 7, 2, 1, 0, 0, 4096, 128, 1) == 0

    def extend(table=one, stride=8, blocks=8, n=4, bs=16, tokens=10, slots=one, pool=one, free=4):
        return L.qkv_extend_pages(table, stride, blocks, one, one, one, free, pool, n, bs, tokens, slots, one, one, None, one, None)
    assert extend(table=None) == -1 and extend(pool=None) == -1 and extend(slots=None) == -1
    assert extend(stride=7) == -2 and extend(blocks=0) == -2 and extend(n=0) == -2 and extend(n=16385) == -2 and extend(bs=0) == -2
    assert extend(tokens=-1) == -2 and extend(tokens=1 << 31) == -2 and extend(free=-1) == -2
    assert extend(blocks=1 << 28, stride=1 << 28) == -2                     # positions beyond 32 bits
    assert L.qkv_shrink_pages(None, 8, 8, one, one, one, 4, one, 4, 16, None) == -1
    assert L.qkv_shrink_pages(one, 8, 8, one, one, one, -4, one, 4, 16, None) == -2


def test_calls_refuse_cpu_tensors():
    cache = paged8.QuashKVPaged8Cache(4, 2, 64, device="cpu")
    x, i32 = torch.zeros(1, 2, 3, 64), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    tables = paged8.PageTables(4, 2, 4, device="cpu")
    for call in (lambda: cache.append(["a"], x, x), lambda: cache.append_slots(x[0], x[0], i32.long()),
                 lambda: cache.attention_with_tables(x, table, i32, 3), lambda: tables.extend(i32, 3), lambda: tables.shrink(i32),
                 lambda: paged8.extend_pages(table, i32, i32, i32, torch.zeros(2, dtype=torch.int32), 16, 3)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()


def test_constructors_and_bookkeeping_without_gpu():
    for bad in (dict(num_blocks=0), dict(block_size=8), dict(block_size=0), dict(head_size=80), dict(codes="e5m2"), dict(layout="dhn")):
        with pytest.raises(ValueError):
            paged8.QuashKVPaged8Cache(**{**dict(num_blocks=4, num_kv_heads=2, head_size=64, device="cpu"), **bad})
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 16385, 1)):
        with pytest.raises(ValueError):
            paged8.PageTables(*bad, device="cpu")
    for layout in ("hnd", "nhd"):
        c = paged8.QuashKVPaged8Cache(4, 2, 64, block_size=32, codes="int8", layout=layout, device="cpu")
        assert c.k_codes.shape == (4, 2, 32, 64) and c.k_codes.dtype == torch.int8 and c.v_scales.shape == (4, 2)
        assert c.k_codes.is_contiguous() == (layout == "hnd")
    c._grow("a", 40)
    c._lens["a"] = 40
    assert c.free_blocks == 2 and c.blocks_of("a") == [0, 1] and c.block_table(["a"])[2] == 40
    c.free("a")
    assert c.free_blocks == 4 and isinstance(c, paged8.PagePool) and issubclass(QuashKVPagedCache, paged8.PagePool)
    t = paged8.PageTables(3, 2, 4, device="cpu")
    assert t.free_pages.tolist() == [2, 1, 0] and t.free_blocks() == 3 and t.refused_tokens() == 0


def test_append_of_a_repeated_sequence_id_takes_turns(monkeypatch):
    """Entries of one id can share a page: each goes in a call of its own, behind the one before it."""
    c = paged8.QuashKVPaged8Cache(8, 1, 32, device="cpu")
    calls = []
    monkeypatch.setattr(paged8.ops, "_need_cuda", lambda t, what: None)
    monkeypatch.setattr(paged8.ops, "append_paged8", lambda k, v, kc, vc, ks, vs, slots, table, starts: calls.append((k[:, 0, 0, 0].tolist(), starts.tolist())))
    k = torch.arange(4.0)[:, None, None, None].expand(4, 1, 3, 32)
    c.append(["a", "b", "a", "a"], k, k)
    assert calls == [([0.0, 1.0], [0, 0]), ([2.0], [3]), ([3.0], [6])]
    assert c.seq_len("a") == 9 and c.seq_len("b") == 3
    c.append(["b", "a"], k[:2], k[:2])
    assert calls[-1] == ([0.0, 1.0], [3, 9])


def test_ops_trace_and_carry_no_derivative():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import ShapeEnv
    _lib.load_host()
    O, env = torch.ops.quashkv_b200, ShapeEnv()
    with FakeTensorMode(allow_non_fake_inputs=True, shape_env=env):
        make = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device="cuda")      # noqa: E731
        i32 = lambda *s: make(*s, dt=torch.int32)      # noqa: E731
        pages = (make(4, 2, 16, 64, dt=torch.int8), make(4, 2, 16, 64, dt=torch.int8), make(4, 2), make(4, 2))
        n = env.create_unbacked_symint()
        q = make(2, 4, 1, 64, dt=torch.bfloat16).requires_grad_()
        out = O.attention_paged8(q, *pages, i32(2, 4), i32(2), n, None, 0, 1.0, True)
        assert out.shape == q.shape and out.dtype == q.dtype and out.requires_grad
        table, lens, pool, free = i32(2, 4), i32(2), i32(2), i32(4)
        slots, starts, after, count = O.extend_pages(table, lens, i32(2), free, pool, 16, 8)
        assert slots.shape == (8,) and slots.dtype == torch.int64 and starts.shape == (3,) and after.shape == (2,) and count.shape == (2,)
        assert len(O.extend_pages_(table, lens, i32(2), free, pool, 16, 8)) == 3
        O.shrink_pages_(table, lens, i32(2), free, pool, 16)
        assert [t._version for t in (table, lens, pool, free)] == [2, 2, 2, 1]
        x = make(8, 2, 64)
        O.append_paged8(x, x, *pages, slots, None, None)
        O.append_paged8(x.view(4, 2, 2, 64), x.view(4, 2, 2, 64), *pages, None, i32(4, 4), i32(4))
        assert [p._version for p in pages] == [2, 2, 2, 2] and x._version == 0
    for name in ("append_paged8", "attention_paged8", "extend_pages", "extend_pages_", "shrink_pages_"):
        assert torch.Tag.pt2_compliant_tag in getattr(O, name).default.tags


def test_slots_and_scales_on_the_host(tmp_path):
    """The functions that decide slots and scales in the kernels, compiled for the host: every length around a page's end,
    tables with bad entries, magnitudes around every power of two."""
    nvcc = shutil.which("nvcc")
    if nvcc is None:
        pytest.skip("no nvcc")
    exe = tmp_path / "paged8_check"
    subprocess.run([nvcc, "-std=c++17", "-arch=sm_100a", "-o", str(exe), os.path.join(HERE, "paged8_check.cu")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and "paged8 host checks OK" in out.stdout, out.stdout + out.stderr


def test_reference_rounding_is_that_of_the_type():
    """The oracle's e4m3 rounding against torch's conversion, at every code, every midpoint and both sides of it."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[codes.isfinite()].unique().numpy()
    mids = (codes[1:] + codes[:-1]) / 2
    y = np.concatenate([codes, mids, np.nextafter(mids, 500, dtype=np.float32), np.nextafter(mids, -500, dtype=np.float32)])
    want = torch.from_numpy(y).float().to(torch.float8_e4m3fn).double().numpy()
    assert (ref.rounded(y.astype(np.float32).astype(np.float64), torch.float8_e4m3fn) == want).all()
    assert ref.rounded(np.array([0.5, 1.5, -2.5, 126.5, 300.0]), torch.int8).tolist() == [0, 2, -2, 126, 127]


def test_reference_shrink_undoes_extend():
    rs = np.random.RandomState(0)
    for _ in range(50):
        n, bs, w = rs.randint(1, 9), int(rs.choice([1, 5, 16])), rs.randint(1, 6)
        lens = rs.randint(0, w * bs + 1, n)
        free = list(range(rs.randint(1, 30)))
        table = rs.randint(100, 200, (n, w)).astype(np.int32)
        pool = [len(free) - rs.randint(0, len(free)), 0]
        new = rs.randint(0, 2 * bs + 2, n)
        t2, slots, starts, after, count = ref.extend(table, lens, new, free, pool, bs, int(new.sum()) + 3)
        assert starts[-1] == new.sum() and all(a <= w * bs for a in after)
        back, free2, count2 = ref.shrink(t2, after, lens, free, count, bs)
        assert back == list(lens) and free2 == free and count2[0] == pool[0]
        assert math.isclose(count[1], int(new.sum()) - (sum(after) - int(lens.sum())))


def test_types_of_the_result():
    """fp32, bf16 and fp16 queries give their type, all others fp32, and tracing says the same."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    _lib.load_host()
    with FakeTensorMode(allow_non_fake_inputs=True):
        make = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device="cuda")      # noqa: E731
        pages = (make(4, 2, 16, 64, dt=torch.int8), make(4, 2, 16, 64, dt=torch.int8), make(4, 2), make(4, 2))
        table, lens = make(2, 4, dt=torch.int32), make(2, dt=torch.int32)
        for dt in (torch.float32, torch.bfloat16, torch.float16, torch.float64, torch.int32):
            out = paged8.attention_paged8(make(2, 4, 1, 64, dt=dt), *pages, table, lens, 64)
            assert out.shape == (2, 4, 1, 64) and out.dtype == (dt if dt in (torch.bfloat16, torch.float16) else torch.float32)
