"""Appends to pages whose scales are a caller's own."""

import numpy as np
import pytest
import torch

import paged8_reference as ref
from quashkv_b200.integrations import paged8

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("scale", [2.0 ** -149, 2.0 ** -130, 2.0 ** -126, 2.0 ** -120, 3.0, 2.0 ** 100])
def test_zeros_and_numbers_behind_any_scale(scale, dtype):
    """A run of zeros keeps the page's scale, however small, and its codes are zeros; a run of numbers raises it or not."""
    H, bs, d = 2, 16, 64
    g = torch.Generator(device=DEV).manual_seed(0)
    for size in (0.0, 1.0, 1e30):
        pages = list(ref.random_pages(g, 2, H, bs, d, dtype))
        pages[2].fill_(scale)
        pages[3].fill_(scale)
        x = torch.randn(5, H, d, generator=g, device=DEV) * size
        slots = np.arange(16 + 4, 16 + 9)
        want = [p.float().cpu().numpy().astype(np.float64) for p in pages]
        for codes, scales in ((want[0], want[2]), (want[1], want[3])):
            # a scale that is no power of two: the kernel multiplies by its rounded inverse
            y = x.float().cpu().numpy().astype(np.float64)
            ref.append(y, codes, scales, slots, bs, dtype)
        paged8.append_paged8(x, x, *pages, torch.from_numpy(slots).to(DEV))
        got = [p.float().cpu().numpy().astype(np.float64) for p in pages]
        assert np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3])
        for a, b in zip(got[:2], want[:2]):
            assert np.isfinite(a).all()
            if scale != 3.0 or size != 1.0:
                assert np.array_equal(a, b)
            else:                                            # a tie that the inverse's rounding tips: at most one code apart
                step = np.abs(b) * 2.0 ** -3 + (1.0 if dtype == torch.int8 else 2.0 ** -9)
                assert (np.abs(a - b) <= step).all()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_a_pool_beyond_32_bits_of_bytes(layout, dtype):
    """The last pages of a pool of 5.4 GB of keys and as many of values hold what the same tokens in a small pool hold, and are read alike."""
    H, bs, d, blocks, lens = 8, 16, 128, 330_000, [300, 1, 90]
    g = torch.Generator(device=DEV).manual_seed(0)
    n = [-(-m // bs) for m in lens]
    codes = "int8" if dtype == torch.int8 else "e4m3"
    big = paged8.QuashKVPaged8Cache(blocks, H, d, codes=codes, layout=layout)
    small = paged8.QuashKVPaged8Cache(sum(n), H, d, codes=codes, layout=layout)
    assert big.k_codes.numel() > 2 ** 32
    table = torch.zeros(3, max(n), dtype=torch.int32, device=DEV)
    for i in range(3):
        table[i, :n[i]] = torch.arange(sum(n[:i]), sum(n[:i + 1]), device=DEV)
    far = blocks - 1 - table                                 # from the end
    x = torch.randn(2, sum(lens), H, d, generator=g, device=DEV).bfloat16()
    slots = torch.cat([t[torch.arange(m, device=DEV) // bs].long() * bs + torch.arange(m, device=DEV) % bs for t, m in zip(table, lens)])
    small.append_slots(x[0], x[1], slots)
    big.append_slots(x[0], x[1], (blocks - 1 - slots // bs) * bs + slots % bs)
    for a, b in zip(big.planes, small.planes):
        assert torch.equal(a[-sum(n):].flip(0).float(), b.float()) and not a[:1000].float().any()
    held = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for q_len in (1, 3, 80):
        for x_dtype in (torch.bfloat16, torch.float32):
            q = torch.randn(3, 4 * H, q_len, d, generator=g, device=DEV).to(x_dtype)
            want = small.attention_with_tables(q, table, held, 300, causal=True)
            assert want.any() and torch.equal(big.attention_with_tables(q, far, held, 300, causal=True), want)
    small.append_with_tables(x[0, :6].view(3, 2, H, d).transpose(1, 2), x[1, :6].view(3, 2, H, d).transpose(1, 2), table, held - 1)
    big.append_with_tables(x[0, :6].view(3, 2, H, d).transpose(1, 2), x[1, :6].view(3, 2, H, d).transpose(1, 2), far, held - 1)
    for a, b in zip(big.planes, small.planes):
        assert torch.equal(a[-sum(n):].flip(0).float(), b.float())
