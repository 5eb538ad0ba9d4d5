"""The tensors of a plan: as many storages, as the ops' schemas say (no result aliases another or an argument)."""

import os

import pytest
import torch

from quashkv_b200.integrations import paged8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _state(n=5, T=300):
    i32 = dict(dtype=torch.int32, device=DEV)
    return (torch.zeros(n, 20, **i32), torch.full((n,), 7, **i32), torch.arange(n, **i32) * 9, torch.arange(100, **i32), torch.tensor([100, 0], **i32), 16, T)


@pytest.mark.parametrize("op", ["extend_pages", "extend_pages_"])
def test_results_have_storages_of_their_own(op, tmp_path):
    args = _state()
    out = getattr(torch.ops.quashkv_b200, op)(*args)
    every = [t.untyped_storage() for t in (*out, *args[:5])]
    assert len({s.data_ptr() for s in every}) == len(every)
    assert all(s.nbytes() == t.numel() * t.element_size() for s, t in zip(every, out)) and all(t.is_contiguous() for t in out)
    lens = out[2]                                            # keeping or saving the small ones keeps nothing else
    torch.save(lens, tmp_path / "lens.pt")
    assert os.path.getsize(tmp_path / "lens.pt") < 8 * args[6]
    none = getattr(torch.ops.quashkv_b200, op)(*_state()[:6], 0)      # no room for tokens
    assert none[0].shape == (0,) and none[1].tolist() == [0] * 6


@pytest.mark.parametrize("op", ["extend_pages", "extend_pages_"])
def test_schemas_hold(op):
    torch.library.opcheck(getattr(torch.ops.quashkv_b200, op).default, _state(), test_utils=("test_schema", "test_faketensor"))


def test_plans_of_a_step_do_not_hold_one_another():
    tables = paged8.PageTables(64, 3, 8)
    plan = tables.extend(torch.tensor([5, 1, 20], dtype=torch.int32, device=DEV), 40)
    kept = plan.start_lens.untyped_storage().nbytes()
    assert kept == 3 * 4 and plan.query_starts.tolist() == [0, 5, 6, 26]
