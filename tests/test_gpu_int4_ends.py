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


@pytest.mark.parametrize("d,dr,heads", [(512, 64, 16), (256, 32, 40)])
@pytest.mark.parametrize("n", [1, 100, 3000])
def test_logits_far_below_zero(d, dr, heads, n):
    """One token's logit is -2e31, the others' -3e31: its row is the result."""
    table, pages = cases.pool_for([n], 73)
    g = torch.Generator().manual_seed(74)
    pe = torch.zeros(n, dr)
    pe[:, 0] = -1.5 * 2.0**42
    pe[n // 2, 0] = -(2.0**42)
    rows = torch.randn(n, d, generator=g)
    cache = cases.stored([rows], [pe], table, [n], pages)
    q = torch.zeros(1, 1, heads, d + dr)
    q[..., d] = 2.0**62
    out, lse = cases.decode(q.bfloat16(), cache, table, [n], 1.0)
    code, params = cases.ref.quantise(rows)
    want = cases.ref.values32(code, params)[n // 2].double()
    # weight times scale in 11 bits, as everywhere
    size = (code.float() + params[..., 1].repeat_interleave(128, 1).abs()) * params[..., 0].repeat_interleave(128, 1)
    assert cases.rounds(out, want, (2.0**-11 + 2.0**-13) * size[n // 2].double()).all()
    assert ((lse + 2.0**104).abs() <= 2.0**-20 * 2.0**104).all()
