"""Scores far beyond what fp32 resolves to a unit: the largest has all the weight, finite inputs give finite results."""

import numpy as np
import pytest
import torch

import paged8_reference as ref
from quashkv_b200.integrations import paged8

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("s", [12, 23, 27, 40, 100])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,G,q_len", [(128, 4, 1), (64, 8, 1), (96, 2, 5), (128, 4, 90), (64, 8, 70), (128, 1, 300)])
def test_large_scores_leave_the_largest(d, G, q_len, x_dtype, s):
    """Scores of whole numbers times 2^s, so that different ones are at least 2^s apart, which fp32 tells apart (each is rounded once,
    in order), and equal ones are equal: a row's output is the mean of the values of the visible tokens with its largest score.
    Value scales differ by page.  Off by at most, of the mean magnitude: 2^-11 for weights in fp16, 2^-19 for the exponentials and sums; and
    half a step of the output's type."""
    g = torch.Generator(device=DEV).manual_seed(s + d)
    bs, lens = 16, [9000, 300, 40, 3]
    total = sum(-(-m // bs) for m in lens)
    k = torch.zeros(total, 1, bs, d, dtype=torch.int8, device=DEV)
    k[..., 0] = torch.randint(-50, 51, (total, 1, bs), generator=g, device=DEV)
    v = torch.randint(-127, 128, (total, 1, bs, d), generator=g, device=DEV).to(torch.int8)
    ks = torch.full((total, 1), 2.0 ** s, device=DEV)
    vs = torch.exp2(torch.randint(-8, 9, (total, 1), generator=g, device=DEV).float())
    table = ref.random_tables(lens, bs, total, s).to(DEV)
    q = torch.zeros(len(lens), G, q_len, d, device=DEV)
    q[..., 0] = torch.randint(1, 4, q.shape[:3], generator=g, device=DEV) * torch.sign(torch.rand(q.shape[:3], generator=g, device=DEV) - 0.5)
    q = q.to(x_dtype)
    n = torch.as_tensor(np.asarray(lens), dtype=torch.int32).to(DEV)
    got = paged8.attention_paged8(q, k, v, ks, vs, table, n, max(lens), scale=1.0, causal=True).double()
    assert got.isfinite().all()
    low, half = x_dtype != torch.float32, torch.finfo(x_dtype).eps / 2
    for i, m in enumerate(lens):
        ids = table[i, :-(-m // bs)].long()
        a = k[ids, 0, :, 0].reshape(-1)[:m].double()
        V = (v[ids, 0].double() * vs[ids, 0].double()[:, None, None]).reshape(-1, d)[:m]
        t = q[i, :, :, 0].double()[..., None] * a                             # (G, q_len, m)
        t = t.masked_fill(torch.ones(q_len, m, dtype=torch.bool, device=DEV).triu(m - q_len + 1), -torch.inf)
        best = ((t == t.amax(-1, keepdim=True)) & (t > -torch.inf)).double()
        w = best / best.sum(-1, keepdim=True).clamp(min=1)
        want, mean = w @ V, w @ V.abs()
        off = mean * ((2.0 ** -11 if low else 0) + 2.0 ** -19) + half * want.abs() + (2.0 ** -25 if x_dtype == torch.float16 else 0)
        assert ((got[i] - want).abs() <= off).all(), (i, float(((got[i] - want).abs() / off.clamp(min=1e-300)).max()))
