"""Page boxes of values at the ends of the range, and of columns that hold no number or an infinity."""

import math

import pytest
import torch

import int4_reference as ref
from mla_kv_quant_b200 import int4

pytestmark = pytest.mark.gpu


def _boxes(cache, pages, counts):
    d, dr, n = cache[0].shape[1] * 2, cache[2].shape[1], cache[0].shape[0] // 64
    view = int4.Int4View(*cache, boxes=(torch.full((n, d + dr), 77, dtype=torch.int8, device="cuda"),
                                        torch.full((n, d + dr), 77, dtype=torch.uint8, device="cuda"),
                                        torch.full((n, 2), 77, dtype=torch.int32, device="cuda")))
    at = torch.tensor(pages, dtype=torch.int32, device="cuda")
    int4.update_boxes(view, at, torch.tensor(counts, dtype=torch.int32, device="cuda"))
    lo, hi = torch.empty(len(pages), d + dr, device="cuda"), torch.empty(len(pages), d + dr, device="cuda")
    int4.read_boxes(view, at, lo, hi)
    return view, lo.cpu().double(), hi.cpu().double()


@pytest.mark.parametrize("d,dr", [(512, 64), (256, 32), (512, 32), (256, 64)])
@pytest.mark.parametrize("count", [1, 10, 64])
def test_columns_without_a_box_leave_the_others_theirs(d, dr, count):
    """A group that is NaN in every token counted, and rotary columns that hold an infinity: their boxes are 0 -+ 0,
    the others as if those columns were 0."""
    cache = ref.random_cache(64 * 2, d, dr, seed=d + count)
    cache[1][64:, 1] = math.nan
    cache[2][64, 3], cache[2][64 + count - 1, 5] = math.inf, -math.inf
    cache[2][64:, 7] = math.nan
    view, lo, hi = _boxes(cache, [1], [count])
    clean = [x.clone() for x in cache]
    clean[1][64:, 1] = 0.0
    clean[2][64:, [3, 5, 7]] = 0.0
    center, radius, exps = ref.boxes(clean, 1, count)
    assert view.boxes[2][1].tolist() == exps
    assert torch.equal(view.boxes[0][1].cpu(), center) and torch.equal(view.boxes[1][1].cpu(), radius)
    gone = list(range(128, 256)) + [d + 3, d + 5, d + 7]
    assert not lo[0, gone].any() and not hi[0, gone].any()


def test_a_nan_among_numbers_is_passed_over():
    cache = ref.random_cache(64, 256, 32, seed=9)
    cache[1][5, 0] = math.nan
    cache[2][6, 2] = math.nan
    view, _, _ = _boxes(cache, [0], [64])
    v = torch.cat([ref.values32(ref.unpack(cache[0].cpu()), cache[1].cpu()), cache[2].cpu().float()], 1)
    lo, hi = torch.nan_to_num(v, nan=math.inf).amin(0), torch.nan_to_num(v, nan=-math.inf).amax(0)
    exps = view.boxes[2][0].tolist()
    top = torch.maximum(lo.abs(), hi.abs())
    assert exps == [ref.exponent(float(top[:256].max())), ref.exponent(float(top[256:].max()))]
    unit = torch.tensor([2.0 ** -exps[0]] * 256 + [2.0 ** -exps[1]] * 32)
    center = torch.round((lo + hi) * 0.5 * unit)
    assert torch.equal(view.boxes[0][0].cpu(), center.to(torch.int8))
    assert torch.equal(view.boxes[1][0].cpu(), torch.ceil(torch.maximum(hi * unit - center, center - lo * unit)).to(torch.uint8))


@pytest.mark.parametrize("d,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("sign", [1, -1])
def test_values_whose_sum_leaves_the_range(d, dr, sign):
    """Values of about 3e38, all of one sign: the box holds them."""
    g = torch.Generator().manual_seed(10)
    codes = torch.randint(0, 256, (64, d // 2), generator=g).to(torch.uint8) | 0x88
    params = torch.zeros(64, d // 128, 2)
    params[..., 0] = sign * 2e37
    rope = (sign * (2.5e38 + 0.5e38 * torch.rand(64, dr, generator=g))).bfloat16()
    cache = [codes.cuda(), params.cuda(), rope.cuda()]
    _, lo, hi = _boxes(cache, [0], [64])
    v = torch.cat([ref.values32(ref.unpack(codes), params), rope.float()], 1).double()
    assert torch.isfinite(v).all()
    slack = 2.0**-18 * 2.0**122  # the bounds' own rounding
    assert (v >= lo - slack).all() and (v <= hi + slack).all()
    assert ((hi - lo) <= v.amax(0) - v.amin(0) + 2 * 2.0**122).all()
