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
