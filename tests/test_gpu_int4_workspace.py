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


@pytest.mark.parametrize("batch,budget", [(4, 5), (2, 9), (1, 9), (3, 4), (4, 9)])
def test_chosen_pages_in_a_larger_calls_workspace(batch, budget):
    lens = [4000, 130, 0, 2777]
    view, table, sl, q, out, lse = _case(lens, 512, 64, 16)
    table, sl, q, out, lse = (x[:batch] for x in (table, sl, q, out, lse))
    ws = int4.Workspace(view, 4, 1, 16, table.shape[1], budget=9)
    fit = int4.Workspace(view, batch, 1, 16, table.shape[1], budget=budget)
    int4.sparse_decode(q, view, table, sl, cases.SM, budget, out, lse, ws)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    int4.sparse_decode(q, view, table, sl, cases.SM, budget, again, lse2, fit)
    assert torch.equal(ws.sel_table[:batch, :budget], fit.sel_table) and torch.equal(ws.sel_lens[:batch], fit.sel_lens)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_larger_selections_than_the_workspaces_are_refused():
    view, table, sl, q, out, lse = _case([300, 300], 512, 64, 16)
    ws = int4.Workspace(view, 1, 1, 16, table.shape[1], budget=4)
    for n, budget in ((2, 4), (1, 5)):
        with pytest.raises(ValueError, match="batch and budget"):
            int4.sparse_decode(q[:n], view, table[:n], sl[:n], cases.SM, budget, out[:n], lse[:n], ws)
    with pytest.raises(ValueError, match="sel_table"):
        int4.select_pages(q[:1], view, table[:1], sl[:1], 4, torch.zeros(4, 2, dtype=torch.int32, device="cuda").t()[:1], ws.sel_lens, ws)


def test_a_table_of_one_row_with_any_row_stride():
    view, table, sl, q, out, lse = _case([700], 512, 64, 16)
    ws = int4.Workspace(view, 1, 1, 16, table.shape[1], budget=4)
    int4.decode(q, view, table, sl, cases.SM, out, lse, ws)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    column = table[0].clone()[:, None].t()  # [1, pages], a row stride of 1
    int4.decode(q, view, column, sl, cases.SM, again, lse2, ws)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    int4.sparse_decode(q, view, column, sl, cases.SM, 4, again, lse2, ws)


def test_the_calls_allocate_nothing():
    lens = [900, 77]
    view, table, sl, q, out, lse = _case(lens, 512, 64, 16)
    ws = int4.Workspace(view, 4, 1, 16, table.shape[1], budget=8)
    rows, pe = torch.randn(5, 512, device="cuda"), torch.randn(5, 64, device="cuda").bfloat16()
    slots, pages = torch.arange(5, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    counts, lo, hi = torch.full((1,), 5, dtype=torch.int32, device="cuda"), torch.empty(1, 576, device="cuda"), torch.empty(1, 576, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def calls():
        int4.write(view, rows, pe, slots, err)
        int4.read(view, slots, rows, pe, err)
        int4.update_boxes(view, pages, counts, err)
        int4.read_boxes(view, pages, lo, hi, err)
        int4.decode(q, view, table, sl, cases.SM, out, lse, ws, err)
        int4.sparse_decode(q, view, table, sl, cases.SM, 5, out, lse, ws, err=err)

    calls()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    calls()
    torch.cuda.synchronize()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    assert err.item() == 0
