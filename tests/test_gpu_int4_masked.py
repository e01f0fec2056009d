"""A token that is no number reaches the query tokens that see it, and no others."""

import math

import pytest
import torch

import int4_cases as cases

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dr,heads", [(512, 64, 16), (256, 32, 40), (512, 32, 3)])
@pytest.mark.parametrize("bad", ["scale", "zero", "group", "all groups", "rope nan", "rope inf"])
def test_a_bad_drafted_token_stays_hidden(d, dr, heads, bad):
    """Four query tokens a request; the last but one of the request's tokens is bad: rows 0 and 1 do not see it."""
    lens, q_len = [300, 64, 65, 130, 4], 4
    table, pages = cases.pool_for(lens, 61)
    g = torch.Generator().manual_seed(62)
    cache = cases.stored([torch.randn(n, d, generator=g) for n in lens], [torch.randn(n, dr, generator=g) for n in lens], table, lens, pages)
    for i, n in enumerate(lens):
        at = int(cases.slots_of(table, i, n)[n - 2])
        if bad == "scale":
            cache[1][at, 0, 0] = math.inf
        elif bad == "zero":
            cache[1][at, 1, 1] = math.nan
        elif bad == "group":  # as the store leaves a group that holds a NaN
            cache[1][at, 1] = math.nan
        elif bad == "all groups":
            cache[1][at] = math.nan
        else:
            cache[2][at, 3] = math.nan if bad == "rope nan" else math.inf
    q = torch.randn(len(lens), q_len, heads, d + dr, generator=g).bfloat16()
    q[..., d + 3] = 1.0
    out, lse = cases.check(q, cache, table, lens, rows=slice(0, 2))
    assert torch.isfinite(out[:, :2]).all()
    if bad not in ("scale",):  # an infinite scale's token may have a logit of minus infinity
        assert torch.isnan(out[:, 2:]).all()
