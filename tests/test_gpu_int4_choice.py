"""The choice of pages where scores leave the range of 32 bits, where the query holds no numbers, and what it promises."""

import math

import pytest
import torch

import int4_cases as cases
import int4_reference as ref
from mla_kv_quant_b200 import int4

pytestmark = pytest.mark.gpu


def _view(cache, boxes=None):
    d, dr, pages = cache[0].shape[1] * 2, cache[2].shape[1], cache[0].shape[0] // 64
    empty = (torch.zeros(pages, d + dr, dtype=torch.int8, device="cuda"), torch.zeros(pages, d + dr, dtype=torch.uint8, device="cuda"),
             torch.zeros(pages, 2, dtype=torch.int32, device="cuda"))
    view = int4.Int4View(*cache, boxes=boxes or empty)
    if boxes is None:
        int4.update_boxes(view, torch.arange(pages, dtype=torch.int32, device="cuda"), torch.full((pages,), 64, dtype=torch.int32, device="cuda"))
    return view


def _select(view, q, table, lens, budget, **keep):
    ws = int4.Workspace(view, len(lens), 1, q.shape[1], table.shape[1], budget)
    int4.select_pages(q.cuda(), view, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), budget, ws.sel_table, ws.sel_lens, ws, **keep)
    return ws.sel_table.cpu()


@pytest.mark.parametrize("d,dr,heads", [(512, 64, 16), (256, 32, 40)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_elements_of_the_query_that_are_no_numbers_count_as_zero(d, dr, heads, value):
    lens, budget = [3000, 1500], 7
    table, pages = cases.pool_for(lens, 81)
    view = _view(ref.random_cache(pages * 64, d, dr, seed=82))
    q = torch.randn(2, heads, d + dr, generator=torch.Generator().manual_seed(83)).bfloat16()
    q[0, 2, 100], q[0, 2, 3], q[1, 1, d + 5] = value, value, value
    clean = torch.where(torch.isfinite(q), q, torch.zeros_like(q))
    got = _select(view, q, table, lens, budget)
    for i, n in enumerate(lens):
        kept = ref.choose(clean[i], view.boxes, table[i], n, budget, 1, 2)
        assert got[i].tolist() == [int(table[i, j]) for j in kept]
