"""Attention at the ends of its inputs' range: an infinity in the query's rotary part, logits far below zero."""

import math

import pytest
import torch

import int4_cases as cases

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dr,heads", [(512, 64, 16), (256, 32, 40)])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinity_in_a_rows_rotary_part(d, dr, heads, value, sign):
    """The row gets NaN, whether the products are infinite upwards or downwards; the other rows do not notice."""
    lens = [200, 1]
    table, pages = cases.pool_for(lens, 71)
    g = torch.Generator().manual_seed(72)
    pe = [torch.randn(n, dr, generator=g) for n in lens]
    for x in pe:
        x[:, 5] = sign * (1 + x[:, 5].abs())
    cache = cases.stored([torch.randn(n, d, generator=g) for n in lens], pe, table, lens, pages)
    q = torch.randn(2, 1, heads, d + dr, generator=g).bfloat16()
    o, l, tol_o, tol_l = cases.attend(q, cache, table, lens)
    q[:, :, 5, d + 5] = value
    out, lse = cases.decode(q, cache, table, lens)
    assert torch.isnan(out[:, :, 5]).all() and torch.isnan(lse[:, :, 5]).all()
    others = [h for h in range(heads) if h != 5]
    assert cases.rounds(out, o, tol_o)[:, :, others].all() and ((lse - l).abs() <= tol_l)[:, :, others].all()
