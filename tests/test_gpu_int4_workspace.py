"""One workspace, made for the largest call, serves smaller ones; calls allocate nothing; tables of one row."""

import pytest
import torch

import int4_cases as cases
import int4_reference as ref
from mla_kv_quant_b200 import int4

pytestmark = pytest.mark.gpu


def _case(lens, d, dr, heads, q_len=1, seed=95):
    table, pages = cases.pool_for(lens, seed)
    cache = ref.random_cache(pages * 64, d, dr, seed=seed)
    boxes = (torch.zeros(pages, d + dr, dtype=torch.int8, device="cuda"), torch.zeros(pages, d + dr, dtype=torch.uint8, device="cuda"),
             torch.zeros(pages, 2, dtype=torch.int32, device="cuda"))
    view = int4.Int4View(*cache, boxes=boxes)
    int4.update_boxes(view, torch.arange(pages, dtype=torch.int32, device="cuda"), torch.full((pages,), 64, dtype=torch.int32, device="cuda"))
    q = torch.randn(len(lens), q_len, heads, d + dr, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
    out, lse = torch.empty(len(lens), q_len, heads, d, dtype=torch.bfloat16, device="cuda"), torch.empty(len(lens), q_len, heads, device="cuda")
    return view, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), q, out, lse


@pytest.mark.parametrize("d,dr,made,used", [(256, 32, (3, 16), (2, 16)), (256, 32, (8, 16), (7, 16)), (256, 64, (6, 8), (4, 8)), (256, 32, (1, 48), (1, 40)),
                                            (512, 64, (3, 16), (1, 16))])
def test_attention_in_a_larger_calls_workspace(d, dr, made, used):
    lens = [700, 3, 129]
    view, table, sl, q, out, lse = _case(lens, d, dr, used[1], used[0])
    ws = int4.Workspace(view, len(lens), *made, table.shape[1])
    fit = int4.Workspace(view, len(lens), *used, table.shape[1])
    int4.decode(q, view, table, sl, cases.SM, out, lse, ws)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    int4.decode(q, view, table, sl, cases.SM, again, lse2, fit)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
