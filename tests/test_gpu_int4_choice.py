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


def _boxes(pages, w, dr, seed):
    g = torch.Generator().manual_seed(seed)
    center = torch.randint(-127, 128, (pages, w), generator=g).to(torch.int8)
    radius = torch.randint(0, 128, (pages, w), generator=g).to(torch.uint8)
    return center, radius


@pytest.mark.parametrize("d,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("e_page,e_q", [(120, 115), (115, 0), (-100, -95), (-100, -30), (0, 0)])
def test_scores_of_any_size_keep_their_order(d, dr, e_page, e_q):
    """Boxes and a query at the ends of FP32's range choose what the same ones in its middle do, the request's last
    pages always among them."""
    pages, heads, budget = 150, 5, 9
    center, radius = _boxes(pages, d + dr, dr, 84)
    spread = torch.randint(0, 3, (pages, 2), generator=torch.Generator().manual_seed(85)).int()
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(86)).int()[None]
    q = torch.randn(1, heads, d + dr, generator=torch.Generator().manual_seed(87)).bfloat16()
    middle = [center.cuda(), radius.cuda(), spread.cuda()]
    kept = ref.choose(q[0], middle, table[0], pages * 64, budget, 1, 2)
    cache = ref.random_cache(pages * 64, d, dr, seed=88)
    far = (center.cuda(), radius.cuda(), (spread + e_page).cuda())
    got = _select(_view(cache, far), (q.float() * 2.0**e_q).bfloat16(), table, [pages * 64], budget)
    assert got[0].tolist() == [int(table[0, j]) for j in kept]


@pytest.mark.parametrize("part", ["latent", "rotary"])
def test_a_part_of_the_query_that_is_zero(part):
    """The other part alone decides, however small it is."""
    d, dr, pages, budget = 512, 64, 90, 6
    center, radius = _boxes(pages, d + dr, dr, 89)
    q = torch.randn(1, 4, d + dr, generator=torch.Generator().manual_seed(90))
    q[..., slice(0, d) if part == "latent" else slice(d, d + dr)] = 0
    table = torch.arange(pages).int()[None]
    zero = torch.zeros(pages, 2, dtype=torch.int32)
    kept = ref.choose(q[0].bfloat16(), [center, radius, zero], table[0], pages * 64, budget, 1, 2)
    view = _view(ref.random_cache(pages * 64, d, dr, seed=91), (center.cuda(), radius.cuda(), (zero - 90).cuda()))
    got = _select(view, (q * 2.0**-95).bfloat16(), table, [pages * 64], budget)
    assert got[0].tolist() == kept


def test_equal_scores_of_any_size_leave_the_last_pages_their_place():
    d, dr, pages, budget = 256, 32, 100, 8
    boxes = (torch.full((pages, d + dr), 127, dtype=torch.int8, device="cuda"), torch.full((pages, d + dr), 127, dtype=torch.uint8, device="cuda"),
             torch.full((pages, 2), 121, dtype=torch.int32, device="cuda"))
    view = _view(ref.random_cache(pages * 64, d, dr, seed=92), boxes)
    q = torch.full((1, 3, d + dr), 3e38).bfloat16()
    got = _select(view, q, torch.arange(pages).int()[None], [pages * 64], budget)
    assert got[0].tolist() == [0, 1, 2, 3, 4, 5, 98, 99]


@pytest.mark.parametrize("d,dr,heads", [(512, 64, 16), (256, 32, 40)])
def test_scores_from_the_boxes_bound_the_logits_and_the_best_token_is_found(d, dr, heads):
    """The score that the rule forms of a box and the 8-bit query is no less than any token's logit but for that rounding;
    a page whose token outweighs all others' scores by itself is chosen."""
    lens, budget = [4000], 6
    table, pages = cases.pool_for(lens, 93)
    g = torch.Generator().manual_seed(94)
    q = torch.randn(1, heads, d + dr, generator=g).bfloat16()
    rows, pe = torch.randn(4000, d, generator=g), torch.randn(4000, dr, generator=g)
    best = 64 * 23 + 17
    rows[best], pe[best] = 40 * q[0, 1, :d].float(), 40 * q[0, 1, d:].float()
    cache = cases.stored([rows], [pe], table, lens, pages)
    view = _view(cache)
    center, radius, exps = (x.cpu().double() for x in view.boxes)
    qd = q[0].double()
    v = torch.cat([ref.values32(ref.unpack(cache[0].cpu()), cache[1].cpu()), cache[2].cpu().float()], 1).double()
    scores = []
    for j in range(-(-4000 // 64)):
        page = int(table[0, j])
        score = slack = 0
        for k, part in enumerate((slice(0, d), slice(d, d + dr))):
            unit = 2.0 ** ref.exponent(float(qd[:, part].abs().max()))
            q8 = torch.round(qd[:, part] / unit)
            size = 2.0 ** exps[page, k]
            score = score + unit * size * (q8 @ center[page, part] + q8.abs() @ radius[page, part])
            slack = slack + 0.5 * unit * size * (center[page, part].abs() + radius[page, part]).sum() + 2.0**-18 * size * qd[:, part].abs().sum(1)
        logit = (qd @ v[page * 64 : page * 64 + 64].T).amax(1)
        assert (logit <= score + slack).all()
        scores.append(float(score.max()))
    others = [s for j, s in enumerate(scores) if j != best // 64]
    assert scores[best // 64] > max(others)
    got = _select(view, q, table, lens, budget)
    assert int(table[0, best // 64]) in got[0].tolist()
