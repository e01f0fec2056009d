"""Attention over tokens whose groups' scales differ by orders of magnitude: what a token adds to a row is held to the
row's own largest, whatever other tokens and rows hold."""

import pytest
import torch

import int4_cases as cases

pytestmark = pytest.mark.gpu

SHAPES = [(512, 64, 16), (512, 64, 8), (256, 32, 40)]


def _inputs(lens, d, dr, heads, seed, q_len=1):
    g = torch.Generator().manual_seed(seed)
    table, pages = cases.pool_for(lens, seed)
    rows = [torch.randn(n, d, generator=g) for n in lens]
    pe = [torch.randn(n, dr, generator=g) for n in lens]
    q = torch.randn(len(lens), q_len, heads, d + dr, generator=g)
    for x in pe:  # a column apart for what a test says about a token's weight
        x[:, 0] = 0
    q[..., d] = 8.0
    return table, pages, rows, pe, q


@pytest.mark.parametrize("d,dr,heads", SHAPES)
@pytest.mark.parametrize("factor", [1e4, 1e6, 1e9])
@pytest.mark.parametrize("where", ["first", "last", "both"])
def test_a_token_of_no_weight_and_a_large_scale(d, dr, heads, factor, where):
    lens = [300, 129]
    table, pages, rows, pe, q = _inputs(lens, d, dr, heads, seed=51)
    for i, n in enumerate(lens):
        at = {"first": [7], "last": [n - 1], "both": [7, n - 1]}[where]
        rows[i][at] *= factor
        pe[i][at, 0] = -200.0  # 115 below the others
    q[..., :d] *= 1e-2 / factor
    cache = cases.stored(rows, pe, table, lens, pages)
    cases.check(q.bfloat16(), cache, table, lens)


@pytest.mark.parametrize("d,dr,heads", SHAPES)
def test_rows_that_look_at_different_tokens(d, dr, heads):
    """Every second head sees nothing but the tokens of a large scale, the others nothing of them."""
    lens = [400, 65]
    table, pages, rows, pe, q = _inputs(lens, d, dr, heads, seed=52)
    for i, n in enumerate(lens):
        rows[i][[3, n - 2]] *= 1e7
        pe[i][[3, n - 2], 0] = 200.0
    q[..., 0::2, d] = -8.0
    q[..., :d] *= 1e-9
    cache = cases.stored(rows, pe, table, lens, pages)
    cases.check(q.bfloat16(), cache, table, lens)


@pytest.mark.parametrize("d,dr,heads", SHAPES)
@pytest.mark.parametrize("size", [1e-4, 1e-6])
@pytest.mark.parametrize("zeros", ["some", "first page", "first tiles", "all but one"])
def test_rows_of_zeros_among_small_latents(d, dr, heads, size, zeros):
    """A group of equal elements is stored with scale 1, which says nothing of its size."""
    lens = [500, 140]
    table, pages, rows, pe, q = _inputs(lens, d, dr, heads, seed=53)
    for i, n in enumerate(lens):
        rows[i] *= size
        rows[i][{"some": slice(0, n, 5), "first page": slice(0, 64), "first tiles": slice(0, 270), "all but one": slice(0, n - 1)}[zeros]] = 0.0
    q[..., :d] *= 0.1 / size
    cache = cases.stored(rows, pe, table, lens, pages)
    cases.check(q.bfloat16(), cache, table, lens)


@pytest.mark.parametrize("d,dr,heads", SHAPES)
def test_groups_of_equal_elements(d, dr, heads):
    """One group of every third token is constant; and a request of nothing but constant groups."""
    lens = [300, 70]
    table, pages, rows, pe, q = _inputs(lens, d, dr, heads, seed=54)
    rows[0] *= 1e-5
    rows[0][::3, :128] = 3e-5 * torch.randn(100, 1, generator=torch.Generator().manual_seed(1))
    rows[1] = torch.randn(70, d // 128, 1, generator=torch.Generator().manual_seed(2)).expand(70, d // 128, 128).reshape(70, d).clone()
    q[0, ..., :d] *= 1e3
    cache = cases.stored(rows, pe, table, lens, pages)
    cases.check(q.bfloat16(), cache, table, lens)


@pytest.mark.parametrize("d,dr,heads", SHAPES)
@pytest.mark.parametrize("slope", [0.05, 0.5])
def test_scales_that_fall_while_the_weight_moves_on(d, dr, heads, slope):
    lens = [700]
    table, pages, rows, pe, q = _inputs(lens, d, dr, heads, seed=55)
    rows[0] *= torch.logspace(4, -4, 700)[:, None]
    pe[0][:, 0] = slope * torch.arange(700)
    q[..., :d] *= 1e-6
    cache = cases.stored(rows, pe, table, lens, pages)
    cases.check(q.bfloat16(), cache, table, lens)


@pytest.mark.parametrize("d,dr,heads", SHAPES)
def test_a_drafted_token_of_a_large_scale(d, dr, heads):
    """The last token is hidden from the earlier query tokens, and of no weight to the last."""
    lens = [200, 129, 3]
    table, pages, rows, pe, q = _inputs(lens, d, dr, heads, seed=56, q_len=3)
    for i, n in enumerate(lens):
        rows[i][n - 1] *= 1e7
        pe[i][n - 1, 0] = -200.0
    q[..., :d] *= 1e-9
    cache = cases.stored(rows, pe, table, lens, pages)
    cases.check(q.bfloat16(), cache, table, lens)


@pytest.mark.parametrize("d,dr,heads", SHAPES[::2])
def test_a_long_request_in_many_runs(d, dr, heads):
    lens = [20000]
    table, pages, rows, pe, q = _inputs(lens, d, dr, heads, seed=57)
    rows[0] *= 1e-5
    rows[0][::97] = 0.0
    rows[0][1000:1300] = 0.0
    rows[0][[5000, 5001, 12345]] *= 1e8
    pe[0][[5000, 5001, 12345], 0] = -200.0
    q[..., :d] *= 1e-3
    cache = cases.stored(rows, pe, table, lens, pages)
    cases.check(q.bfloat16(), cache, table, lens)
