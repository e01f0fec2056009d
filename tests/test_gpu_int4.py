"""The 4-bit latent cache on the GPU: storing, attention, page boxes, page selection."""

import math

import pytest
import torch

import int4_reference as ref
from mla_kv_quant_b200 import _lib, int4

pytestmark = pytest.mark.gpu

SM = 1.0 / math.sqrt(192.0)


def _err():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _empty_view(slots, d, dr, boxes=False):
    box = None
    if boxes:
        box = (torch.zeros(slots // 64, d + dr, dtype=torch.int8, device="cuda"),
               torch.zeros(slots // 64, d + dr, dtype=torch.uint8, device="cuda"),
               torch.zeros(slots // 64, 2, dtype=torch.int32, device="cuda"))
    return int4.Int4View(torch.zeros(slots, d // 2, dtype=torch.uint8, device="cuda"),
                         torch.zeros(slots, d // 128, 2, device="cuda"),
                         torch.zeros(slots, dr, dtype=torch.bfloat16, device="cuda"), box)


# ---- store ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("d,dr", [(512, 64), (256, 32), (512, 32), (256, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [0, 1, 63, 1001])
def test_write_and_read_back_are_the_codec_bit_for_bit(d, dr, dtype, n):
    g = torch.Generator().manual_seed(n + d)
    slots_total = 1088
    view = _empty_view(slots_total, d, dr)
    wide = torch.randn(n, d + dr + 16, generator=g) * torch.exp(2 * torch.randn(n, 1, generator=g))
    wide[: n // 8, :128] = 0.75  # constant groups
    wide[n // 8 : n // 4, 128:256] = torch.round(wide[n // 8 : n // 4, 128:256] * 2) * 0.5  # many ties
    x = wide.to(dtype).cuda()
    pe = wide.to(torch.bfloat16).cuda()[:, d : d + dr]  # a strided view
    slots = torch.randperm(slots_total, generator=g)[:n].cuda()
    int4.write(view, x[:, :d], pe, slots if n != 63 else slots.int())
    code, params = ref.quantise(x[:, :d].cpu())
    assert torch.equal(view.codes[slots].cpu(), ref.pack(code))
    assert torch.equal(view.params[slots].cpu(), params)
    assert torch.equal(view.rope[slots], pe)
    untouched = torch.ones(slots_total, dtype=torch.bool)
    untouched[slots.cpu()] = False
    assert not view.codes.cpu()[untouched].any() and not view.params.cpu()[untouched].any()
    for out_dtype in (torch.bfloat16, torch.float32):
        out = torch.full((n, d + dr + 8), 7.0, dtype=out_dtype, device="cuda")
        out_pe = torch.empty(n, dr, dtype=torch.bfloat16, device="cuda")
        int4.read(view, slots, out[:, :d], out_pe)
        assert torch.equal(out[:, :d].cpu(), ref.values32(code, params).to(out_dtype))
        assert (out[:, d:] == 7.0).all() and torch.equal(out_pe, pe)


def test_bad_slots_are_skipped_and_reported_and_non_finite_groups_read_as_nan():
    view = _empty_view(128, 512, 64)
    x = torch.randn(5, 512, device="cuda")
    x[1, 3], x[2, 130], x[3, 400] = math.nan, math.inf, -math.inf
    pe = torch.randn(5, 64, device="cuda").bfloat16()
    err = _err()
    int4.write(view, x, pe, torch.tensor([3, 4, 5, 6, 127], device="cuda"), err)
    assert err.item() == 0
    out = torch.empty(5, 512, device="cuda")
    int4.read(view, torch.tensor([3, 4, 5, 6, 127], device="cuda"), out)
    bad = torch.isnan(out).reshape(5, 4, 128)
    want = torch.zeros(5, 4, dtype=torch.bool)
    want[1, 0] = want[2, 1] = want[3, 3] = True
    assert torch.equal(bad.all(-1).cpu(), want) and torch.equal(bad.any(-1).cpu(), want)
    before = [t.clone() for t in (view.codes, view.params, view.rope)]
    int4.write(view, x[:3], pe[:3], torch.tensor([-1, 128, 1 << 40], device="cuda"), err)
    assert err.item() == _lib.DEV_BAD_SLOT
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, (view.codes, view.params, view.rope)))
    err.zero_()
    out_pe = torch.empty(2, 64, dtype=torch.bfloat16, device="cuda")
    int4.read(view, torch.tensor([-5, 127], dtype=torch.int32, device="cuda"), out[:2], out_pe, err)
    assert err.item() == _lib.DEV_BAD_SLOT
    assert not out[0].any() and not out_pe[0].any() and torch.equal(out_pe[1], pe[4])


# ---- attention -----------------------------------------------------------------------------------------------------


def _requests(lens, seed, extra_pages=3):
    """A shuffled page table for the lengths; -> table [B, max_pages], pages of the pool."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // 64) for n in lens]
    total = sum(counts) + extra_pages
    order = torch.randperm(total, generator=g).int()
    table = torch.full((len(lens), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at : at + c]
        at += c
    return table.cuda(), total


def _poison_tail(cache, table, lens):
    """NaN and infinities in every slot that no request's length covers."""
    codes, params, rope = cache
    used = torch.zeros(codes.shape[0], dtype=torch.bool)
    for i, n in enumerate(lens):
        pos = torch.arange(n)
        used[table[i].cpu().long()[pos // 64] * 64 + pos % 64] = True
    free = (~used).cuda()
    params[free, :, 0] = math.nan
    params[free, :, 1] = math.inf
    rope[free] = -math.inf
    codes[free] = 0xFF


def _check(q, cache, table, lens, out, lse, sm_scale=SM):
    o, l, tol_o, tol_l = ref.attend(q, cache, table, lens, sm_scale)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.equal(torch.isinf(l), torch.isinf(lse))
    fine = torch.isfinite(l)
    assert not out[~fine].any()
    assert ((lse - l).abs() <= tol_l)[fine].all(), float(((lse - l).abs() - tol_l)[fine].max())
    assert ((out - o).abs() <= tol_o).all(), float(((out - o).abs() / tol_o).max())


@pytest.mark.parametrize("d,dr,heads", [(512, 64, 16), (512, 64, 8), (256, 32, 40), (256, 32, 16), (512, 32, 1), (256, 64, 17), (512, 64, 128)])
@pytest.mark.parametrize("q_len", [1, 3])
def test_attention_matches_64_bits(d, dr, heads, q_len):
    lens = [0, 1, 2, 63, 64, 65, 700, 1301, 128]
    table, pages = _requests(lens, seed=heads)
    cache = ref.random_cache(pages * 64, d, dr, seed=d + heads)
    _poison_tail(cache, table, lens)
    g = torch.Generator().manual_seed(heads)
    q = (2 * torch.randn(len(lens), q_len, heads, d + dr, generator=g)).bfloat16().cuda()
    view = int4.Int4View(*cache)
    ws = int4.Workspace(view, len(lens), q_len, heads, table.shape[1])
    out = torch.full((len(lens), q_len, heads, d), math.nan, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((len(lens), q_len, heads), math.nan, device="cuda")
    err = _err()
    int4.decode(q, view, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), SM, out, lse, ws, err)
    assert err.item() == 0
    _check(q, cache, table, lens, out, lse)


@pytest.mark.parametrize("batch,ctx,q_len", [(1, 20000, 1), (2, 9001, 4), (150, 130, 1), (3, 64, 64), (300, 65, 2)])
def test_attention_over_one_long_request_and_over_many_short_ones(batch, ctx, q_len):
    lens = [max(1, ctx - 7 * i) for i in range(batch)]
    table, pages = _requests(lens, seed=ctx)
    cache = ref.random_cache(pages * 64, 512, 64, seed=ctx)
    q = torch.randn(batch, q_len, 16, 576, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    view = int4.Int4View(*cache)
    ws = int4.Workspace(view, batch, q_len, 16, table.shape[1])
    out = torch.empty(batch, q_len, 16, 512, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(batch, q_len, 16, device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    int4.decode(q, view, table, sl, SM, out, lse, ws)
    _check(q, cache, table, lens, out, lse)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    int4.decode(q, view, table, sl, SM, again, lse2, ws)  # the scratch as the last call left it
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("lens", [[64 * 13 * 2, 64 * 300], [64 * 161, 64 * 160, 1, 0, 64 * 163 + 5], [64 * 97, 64 * 400, 64 * 30, 64 * 222], [30000] + [70] * 40])
@pytest.mark.parametrize("heads", [16, 40])
def test_requests_cut_into_few_and_many_partials(lens, heads):
    """Long requests next to one another and to short ones: partials joined in one and in two steps."""
    table, pages = _requests(lens, seed=sum(lens))
    cache = ref.random_cache(pages * 64, 256, 32, seed=len(lens))
    q = torch.randn(len(lens), 1, heads, 288, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    view = int4.Int4View(*cache)
    ws = int4.Workspace(view, len(lens), 1, heads, table.shape[1])
    out = torch.empty(len(lens), 1, heads, 256, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(len(lens), 1, heads, device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for _ in range(2):
        out.fill_(math.nan)
        int4.decode(q, view, table, sl, SM, out, lse, ws)
        _check(q, cache, table, lens, out, lse)


def test_attention_where_the_maximum_keeps_rising_and_where_it_falls():
    """Logits that grow by hundreds along the request (every reference maximum is left behind), and the reverse."""
    n = 1500
    table, pages = _requests([n, n], seed=2)
    cache = ref.random_cache(pages * 64, 512, 64, seed=3, spread=0.2)
    view = int4.Int4View(*cache)
    pos = torch.arange(n)
    for i, slope in enumerate((0.5, -0.5)):
        at = table[i].cpu().long()[pos // 64] * 64 + pos % 64
        cache[2][at.cuda(), 0] = (slope * pos.float()).bfloat16().cuda()
    q = torch.randn(2, 16, 576, generator=torch.Generator().manual_seed(4)).bfloat16()
    q[..., 512] = 8.0
    q = q.cuda()
    ws = int4.Workspace(view, 2, 1, 16, table.shape[1])
    out = torch.empty(2, 16, 512, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(2, 16, device="cuda")
    int4.decode(q, view, table, torch.tensor([n, n], dtype=torch.int32, device="cuda"), SM, out, lse, ws)
    _check(q[:, None], cache, table, [n, n], out[:, None], lse[:, None])


@pytest.mark.parametrize("factor", [1e-4, 1.0, 1e4])
def test_attention_with_small_and_large_scales(factor):
    """Groups whose scales drift by powers of ten along the request."""
    n = 900
    table, pages = _requests([n], seed=5)
    cache = ref.random_cache(pages * 64, 512, 64, seed=6, spread=0.5)
    pos = torch.arange(n)
    at = (table[0].cpu().long()[pos // 64] * 64 + pos % 64).cuda()
    cache[1][at, 1, 0] *= torch.logspace(0, 3, n, device="cuda")
    cache[1][..., 0] *= factor
    q = (torch.randn(1, 16, 576, generator=torch.Generator().manual_seed(7)) / max(factor, 1.0)).bfloat16().cuda()
    q[..., 128:256] *= 1e-3
    view = int4.Int4View(*cache)
    ws = int4.Workspace(view, 1, 1, 16, table.shape[1])
    out, lse = torch.empty(1, 16, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 16, device="cuda")
    int4.decode(q, view, table, torch.tensor([n], dtype=torch.int32, device="cuda"), SM, out, lse, ws)
    _check(q[:, None], cache, table, [n], out[:, None], lse[:, None])


def test_bad_pages_take_no_weight_and_lengths_are_cut_to_the_table():
    lens = [300, 400]
    table, pages = _requests(lens, seed=8)
    cache = ref.random_cache(pages * 64, 256, 32, seed=9)
    table[0, 1], table[0, 4], table[1, 0] = -1, pages, 1 << 30
    q = torch.randn(2, 16, 288, generator=torch.Generator().manual_seed(10)).bfloat16().cuda()
    view = int4.Int4View(*cache)
    ws = int4.Workspace(view, 2, 1, 16, table.shape[1])
    out, lse, err = torch.empty(2, 16, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(2, 16, device="cuda"), _err()
    int4.decode(q, view, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), SM, out, lse, ws, err)
    assert err.item() == _lib.DEV_BAD_PAGE
    _check(q[:, None], cache, table, lens, out[:, None], lse[:, None])
    err.zero_()
    long = torch.tensor([300, 5000], dtype=torch.int32, device="cuda")
    int4.decode(q[1:], view, table[1:], long[1:], SM, out[1:], lse[1:], ws, err)
    assert err.item() == _lib.DEV_BAD_PAGE | _lib.DEV_BAD_REQ
    _check(q[1:, None], cache, table[1:], [table.shape[1] * 64], out[1:, None], lse[1:, None])
    err.zero_()  # every page bad, and a negative length
    int4.decode(q, view, torch.full_like(table, -1), torch.tensor([300, -4], dtype=torch.int32, device="cuda"), SM, out, lse, ws, err)
    assert not out.any() and torch.isinf(lse).all()


def test_attention_with_strided_query_and_output_on_another_stream():
    lens = [500, 77]
    table, pages = _requests(lens, seed=11)
    cache = ref.random_cache(pages * 64, 512, 64, seed=12)
    view = int4.Int4View(*cache)
    ws = int4.Workspace(view, 2, 2, 16, table.shape[1])
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(2, 16, 3, 640, device="cuda").bfloat16()
        q = big.transpose(1, 2)[:, 1:, :, 32:608]  # [2, 2, 16, 576], heads outermost
        room = torch.full((16, 2, 2, 528), 3.0, dtype=torch.bfloat16, device="cuda")
        out = room.permute(1, 2, 0, 3)[..., 8:520]
        lse = torch.empty(2, 2, 16, device="cuda")
        int4.decode(q, view, table, sl, SM, out, lse, ws)
    side.synchronize()
    _check(q, cache, table, lens, out, lse)
    assert (room[..., :8] == 3.0).all() and (room[..., 520:] == 3.0).all()


def test_nan_in_one_query_row_stays_in_that_row():
    table, pages = _requests([200], seed=13)
    cache = ref.random_cache(pages * 64, 512, 64, seed=14)
    view = int4.Int4View(*cache)
    ws = int4.Workspace(view, 1, 1, 16, table.shape[1])
    q = torch.randn(1, 16, 576, generator=torch.Generator().manual_seed(15)).bfloat16().cuda()
    out, lse = torch.empty(1, 16, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 16, device="cuda")
    sl = torch.tensor([200], dtype=torch.int32, device="cuda")
    q[0, 5, 100] = math.nan
    q[0, 9, 560] = math.nan
    int4.decode(q, view, table, sl, SM, out, lse, ws)
    rows = [i for i in range(16) if i not in (5, 9)]
    assert torch.isnan(out[0, [5, 9]]).all() and torch.isnan(lse[0, [5, 9]]).all()
    _check(q[:, None, rows], cache, table, [200], out[:, None, rows], lse[:, None, rows])


def test_offsets_beyond_32_bits():
    """A pool of 8.5 million slots: its last pages start past 2^31 bytes of codes and rope elements past 2^29."""
    slots = 8_500_032
    view = _empty_view(slots, 512, 64, boxes=True)
    n = 150
    small = ref.random_cache(192, 512, 64, seed=16)
    last = slots // 64 - 1
    table = torch.tensor([[last, 0, last - 2]], dtype=torch.int32, device="cuda")
    where = (table[0].long()[:, None] * 64 + torch.arange(64, device="cuda")[None, :]).reshape(-1)
    x = torch.empty(192, 512, device="cuda")
    int4.read(int4.Int4View(*small), torch.arange(192, device="cuda"), x)
    int4.write(view, x, small[2], where)
    back, back_pe = torch.empty(192, 512, device="cuda"), torch.empty(192, 64, dtype=torch.bfloat16, device="cuda")
    int4.read(view, where, back, back_pe)
    code, params = ref.quantise(x.cpu())
    assert torch.equal(back.cpu(), ref.values32(code, params)) and torch.equal(back_pe, small[2])
    q = torch.randn(1, 16, 576, generator=torch.Generator().manual_seed(17)).bfloat16().cuda()
    ws = int4.Workspace(view, 1, 1, 16, 3, budget=2)
    out, lse, err = torch.empty(1, 16, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 16, device="cuda"), _err()
    int4.decode(q, view, table, torch.tensor([n], dtype=torch.int32, device="cuda"), SM, out, lse, ws, err)
    assert err.item() == 0
    near = [ref.pack(code).cuda(), params.cuda(), small[2]]
    local = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    _check(q[:, None], near, local, [n], out[:, None], lse[:, None])
    int4.update_boxes(view, table[0], torch.tensor([64, 64, 22], dtype=torch.int32, device="cuda"), err)
    for i, count in enumerate((64, 64, 22)):
        center, radius, exps = ref.boxes(near, i, count)
        page = int(table[0, i])
        assert torch.equal(view.boxes[0][page].cpu(), center) and torch.equal(view.boxes[1][page].cpu(), radius)
        assert view.boxes[2][page].tolist() == exps
    assert err.item() == 0


# ---- boxes and selection -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("d,dr", [(512, 64), (256, 32), (512, 32), (256, 64)])
def test_boxes_are_the_rule_and_hold_every_token(d, dr):
    cache = ref.random_cache(64 * 9, d, dr, seed=d + dr)
    cache[1][64 * 8 :, :, 0] = 0.0  # a page of zeros
    cache[2][64 * 8 :] = 0.0
    cache[1][64 * 7 + 10 : 64 * 8] = math.nan  # beyond the tokens counted
    cache[2][64 * 7 + 10 : 64 * 8] = math.inf
    view = int4.Int4View(*cache, boxes=_empty_view(64 * 9, d, dr, True).boxes)
    pages = torch.tensor([5, 0, 8, 7, 2], dtype=torch.int32, device="cuda")
    counts = torch.tensor([64, 1, 64, 10, 33], dtype=torch.int32, device="cuda")
    err = _err()
    int4.update_boxes(view, pages, counts, err)
    lo, hi = torch.empty(5, d + dr, device="cuda"), torch.empty(5, d + dr, device="cuda")
    int4.read_boxes(view, pages, lo, hi, err)
    assert err.item() == 0
    for i, (page, n) in enumerate(zip(pages.tolist(), counts.tolist())):
        center, radius, exps = ref.boxes(cache, page, n)
        assert torch.equal(view.boxes[0][page].cpu(), center) and torch.equal(view.boxes[1][page].cpu(), radius)
        assert view.boxes[2][page].tolist() == exps
        unit = torch.tensor([2.0 ** exps[0]] * d + [2.0 ** exps[1]] * dr)
        assert torch.equal(lo[i].cpu(), (center.float() - radius.float()) * unit)
        assert torch.equal(hi[i].cpu(), (center.float() + radius.float()) * unit)
        rows = slice(page * 64, page * 64 + n)
        v = torch.cat([ref.values32(ref.unpack(cache[0][rows].cpu()), cache[1][rows].cpu()), cache[2][rows].cpu().float()], 1)
        slack = 2.0**-22 * 127 * unit  # the bounds' own rounding
        assert (v >= lo[i].cpu() - slack).all() and (v <= hi[i].cpu() + slack).all()
    assert not view.boxes[1][3].any()  # a page not asked for
    before = [t.clone() for t in view.boxes]
    int4.update_boxes(view, torch.tensor([-1, 9, 3, 3], dtype=torch.int32, device="cuda"),
                      torch.tensor([64, 64, 0, 65], dtype=torch.int32, device="cuda"), err)
    assert err.item() == _lib.DEV_BAD_PAGE and all(torch.equal(a, b) for a, b in zip(before, view.boxes))
    err.zero_()
    int4.read_boxes(view, torch.tensor([9], dtype=torch.int32, device="cuda"), lo[:1], hi[:1], err)
    assert err.item() == _lib.DEV_BAD_PAGE and not lo[0].any() and not hi[0].any()


def _with_boxes(cache, pages):
    d, dr = cache[0].shape[1] * 2, cache[2].shape[1]
    view = int4.Int4View(*cache, boxes=_empty_view(pages * 64, d, dr, True).boxes)
    int4.update_boxes(view, torch.arange(pages, dtype=torch.int32, device="cuda"), torch.full((pages,), 64, dtype=torch.int32, device="cuda"))
    return view


@pytest.mark.parametrize("d,dr,heads,budget,keep", [(512, 64, 16, 8, (1, 2)), (256, 32, 40, 5, (0, 1)), (512, 32, 1, 4, (2, 2)), (256, 64, 128, 33, (1, 2)), (512, 64, 8, 1, (0, 1))])
def test_the_chosen_pages_are_the_rule(d, dr, heads, budget, keep):
    lens = [0, 1, 64 * budget, 64 * budget + 1, 3000, 5555, 64 * 37]
    table, pages = _requests(lens, seed=budget)
    cache = ref.random_cache(pages * 64, d, dr, seed=budget + d)
    view = _with_boxes(cache, pages)
    table[4, 3] = -1  # a bad page scores lowest
    table[5, 9] = table[5, 7]  # equal scores: the lower index first
    table[5, 11] = table[5, 7]
    q = torch.randn(len(lens), heads, d + dr, generator=torch.Generator().manual_seed(heads)).bfloat16().cuda()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = int4.Workspace(view, len(lens), 1, heads, table.shape[1], budget)
    err = _err()
    for _ in range(2):
        int4.select_pages(q, view, table, sl, budget, ws.sel_table, ws.sel_lens, ws, *keep, err=err)
    assert err.item() == _lib.DEV_BAD_PAGE
    for i, n in enumerate(lens):
        kept = ref.choose(q[i], view.boxes, table[i].cpu(), n, budget, *keep)
        want = [int(table[i, j]) for j in kept] + [-1] * (budget - len(kept))
        assert ws.sel_table[i].tolist() == want, i
        held = -(-n // 64)
        assert int(ws.sel_lens[i]) == (0 if n == 0 else (len(kept) - 1) * 64 + n - (held - 1) * 64)


@pytest.mark.parametrize("held", [70, 300, 2100, 5000])
def test_the_choice_among_many_pages_and_equal_scores(held):
    """Boxes with few different values, so that many pages score alike."""
    d, dr, heads, budget = 256, 32, 4, 64
    view = _empty_view(held * 64, d, dr, True)
    g = torch.Generator().manual_seed(held)
    view.boxes[0].copy_(torch.randint(-1, 2, (held, 1), generator=g).expand(held, d + dr).to(torch.int8))
    view.boxes[1].copy_(torch.randint(0, 2, (held, 1), generator=g).expand(held, d + dr).to(torch.uint8))
    table = torch.randperm(held, generator=g).int().cuda()[None]
    q = torch.randn(1, heads, d + dr, generator=g).bfloat16().cuda()
    ws = int4.Workspace(view, 1, 1, heads, held, budget)
    int4.select_pages(q, view, table, torch.tensor([held * 64 - 3], dtype=torch.int32, device="cuda"), budget, ws.sel_table, ws.sel_lens, ws)
    kept = ref.choose(q[0], view.boxes, table[0].cpu(), held * 64 - 3, budget, 1, 2)
    assert ws.sel_table[0].tolist() == [int(table[0, j]) for j in kept]
    assert int(ws.sel_lens[0]) == budget * 64 - 3


def test_scores_bound_every_token_of_the_page():
    """The selection's score is no less than any token's logit, but for q's rounding to 8 bits."""
    cache = ref.random_cache(64 * 6, 512, 64, seed=20)
    view = _with_boxes(cache, 6)
    q = torch.randn(16, 576, generator=torch.Generator().manual_seed(21)).bfloat16()
    lo, hi = torch.empty(6, 576, device="cuda"), torch.empty(6, 576, device="cuda")
    int4.read_boxes(view, torch.arange(6, dtype=torch.int32, device="cuda"), lo, hi)
    lo, hi = lo.cpu().double(), hi.cpu().double()
    v = torch.cat([ref.values32(ref.unpack(cache[0].cpu()), cache[1].cpu()), cache[2].cpu().float()], 1).double()
    for page in range(6):
        bound = torch.maximum(q.double() * lo[page], q.double() * hi[page]).sum(1)
        logit = (q.double() @ v[page * 64 : page * 64 + 64].T).max(1).values
        assert (logit <= bound * (1 + 1e-6) + 1e-6).all()


def test_sparse_decode_attends_to_the_chosen_pages():
    lens = [4000, 130, 0, 2777]
    table, pages = _requests(lens, seed=22)
    cache = ref.random_cache(pages * 64, 512, 64, seed=23)
    view = _with_boxes(cache, pages)
    q = torch.randn(4, 1, 16, 576, generator=torch.Generator().manual_seed(24)).bfloat16().cuda()
    ws = int4.Workspace(view, 4, 1, 16, table.shape[1], budget=7)
    out, lse = torch.empty(4, 1, 16, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(4, 1, 16, device="cuda")
    int4.sparse_decode(q, view, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), SM, 7, out, lse, ws)
    sel_lens = ws.sel_lens.tolist()
    assert sel_lens == [6 * 64 + 4000 - 62 * 64, 130, 0, 6 * 64 + 2777 - 43 * 64]
    _check(q, cache, ws.sel_table, sel_lens, out, lse)
    full, lse_full = torch.empty_like(out), torch.empty_like(lse)
    wide = int4.Workspace(view, 4, 1, 16, table.shape[1], budget=80)  # a budget that holds every page: plain attention
    int4.sparse_decode(q, view, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), SM, 80, full, lse_full, wide)
    _check(q, cache, table, lens, full, lse_full)


def test_the_calls_replay_from_a_graph():
    lens = [900, 2000]
    table, pages = _requests(lens, seed=25)
    cache = ref.random_cache(pages * 64, 512, 64, seed=26)
    view = _with_boxes(cache, pages)
    q = torch.randn(2, 1, 16, 576, generator=torch.Generator().manual_seed(27)).bfloat16().cuda()
    ws = int4.Workspace(view, 2, 1, 16, table.shape[1], budget=9)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = torch.empty(2, 1, 16, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(2, 1, 16, device="cuda")
    int4.sparse_decode(q, view, table, sl, SM, 9, out, lse, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        int4.sparse_decode(q, view, table, sl, SM, 9, out, lse, ws)
    q.copy_(torch.randn(2, 1, 16, 576, generator=torch.Generator().manual_seed(28)).bfloat16())
    for _ in range(3):
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        _check(q, cache, ws.sel_table, ws.sel_lens.tolist(), out, lse)


def test_the_wrappers_refuse_what_the_kernels_do_not_take():
    view = _empty_view(128, 512, 64)
    ws = int4.Workspace(view, 2, 1, 16, 4)
    table, sl = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    q, out = torch.zeros(2, 16, 576, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 16, 512, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="q must be"):
        int4.decode(q.float(), view, table, sl, SM, out, None, ws)
    with pytest.raises(ValueError, match="out must be"):
        int4.decode(q, view, table, sl, SM, out[:1], None, ws)
    with pytest.raises(TypeError, match="int32"):
        int4.decode(q, view, table.long(), sl, SM, out, None, ws)
    with pytest.raises(_lib.RolaqError, match="sm_scale"):
        int4.decode(q, view, table, sl, 0.0, out, None, ws)
    with pytest.raises(_lib.RolaqError, match="16-byte aligned"):
        int4.decode(torch.zeros(2 * 16 * 576 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 16, 576), view, table, sl, SM, out, None, ws)
    with pytest.raises(ValueError, match="one device"):
        int4.decode(q, view, table, sl.cpu(), SM, out, None, ws)
    with pytest.raises(ValueError, match="no page boxes"):
        int4.select_pages(q, view, table, sl, 4, ws.sel_table, ws.sel_lens, ws)
    with pytest.raises(ValueError, match="batch and budget"):
        int4.sparse_decode(q, view, table, sl, SM, 4, out, None, ws)
    with pytest.raises(TypeError, match="slots"):
        int4.write(view, out[:, 0], q[:, 0, 512:], sl.float())
    with pytest.raises(ValueError, match="k_pe must be"):
        int4.write(view, out[:, 0], q[:, 0, :64].repeat(1, 2), sl)
    tiny = int4.Workspace(view, 1, 1, 1, 1)
    tiny.nbytes = 1024
    with pytest.raises(_lib.RolaqError, match="workspace"):
        int4.decode(q, view, table, sl, SM, out, None, tiny)
    boxed = _empty_view(128, 512, 64, True)
    with pytest.raises(_lib.RolaqError, match="keep_first"):
        int4.select_pages(q, boxed, table, sl, 2, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), ws.sel_lens, ws)
    with pytest.raises(ValueError, match="one query token"):
        int4.select_pages(q.view(1, 2, 16, 576), boxed, table[:1], sl[:1], 4, ws.sel_table, ws.sel_lens, ws)
