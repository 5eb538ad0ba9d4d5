"""Many tokens of little weight beside one of much: what fp16 holds of weights must not lose their sum."""

import math

import numpy as np
import pytest
import torch

from quashkv_b200.integrations import paged8

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("n", [4096, 131072])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,G,q_len", [(128, 4, 40), (64, 8, 40), (128, 1, 300), (64, 1, 600), (128, 4, 1)])
def test_many_small_weights_are_summed(d, G, q_len, x_dtype, n):
    """Token 0 has nearly all the weight and values of zero, the n - 1 others 2^-S of it each, S from 16 to 34 by the row, and values of
    1: the output is their share alone.

    A weight is held as fp16 beside the largest one, which is at least 2^9: half of fp16's least step, 2^-25, is 2^-34 of the largest,
    so n of them are off by n 2^-34 of it at most, besides 2^-11 of each (fp16's half step), the arithmetic of scores and exponentials
    (an argument of up to 34, off by a few times 2^-24 of it, and the exponential's own 2^-22: below 2^-12), fp32 sums of n / 16
    steps, which truncate (2^-23 each), and the output's half step."""
    rows = q_len * G
    S = torch.linspace(16, 34, rows, device=DEV, dtype=torch.float64)
    q = torch.zeros(1, G, q_len, d, device=DEV, dtype=x_dtype)
    q[0, :, :, 0] = (S / 16).to(x_dtype).view(q_len, G).T
    k = torch.zeros(n // 16, 1, 16, d, device=DEV, dtype=torch.int8)
    v = torch.full_like(k, 64)
    k[0, 0, 0, 0], v[0, 0, 0] = 64, 0
    ks = torch.full((n // 16, 1), 2.0 ** -6, device=DEV)
    table = torch.arange(n // 16, dtype=torch.int32, device=DEV)[None]
    lens = torch.full((1,), n, dtype=torch.int32, device=DEV)
    scale = float(np.float32(16 * math.log(2)))              # a unit of the first coordinate is 2^16
    got = paged8.attention_paged8(q, k, v, ks, ks, table, lens, n, scale=scale).double()
    small = torch.exp(-scale * q[..., 0].double())           # each small weight, the large one being 1
    want = ((n - 1) * small / (1 + (n - 1) * small))[..., None].expand_as(got)
    off = want * (2.0 ** -11 + 2.0 ** -12 + n / 16 * 2.0 ** -23 + torch.finfo(x_dtype).eps / 2) + n * 2.0 ** -34
    if x_dtype == torch.float16:
        off = off + 2.0 ** -25                               # half of the least step of the output
    worst = ((got - want).abs() / off).amax(-1)
    assert worst.max() <= 1, (float(worst.max()), (got - want)[0, 0, :, 0].tolist()[:40])
