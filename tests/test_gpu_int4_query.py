"""Attention over the 4-bit cache with queries at the ends of their range, and with one element far above the others."""

import pytest
import torch

import int4_reference as ref
from mla_kv_quant_b200 import int4

pytestmark = pytest.mark.gpu

SM = 192**-0.5


def _decode(q, cache, lens, sm_scale):
    pages = [-(-n // 64) for n in lens]
    table = torch.zeros(len(lens), max(pages), dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = torch.arange(at, at + n)
        at += n
    table = table.cuda()
    view = int4.Int4View(*cache)
    b, t, h, w = q.shape
    out, lse = torch.empty(b, t, h, view.latent_dim, dtype=torch.bfloat16, device="cuda"), torch.empty(b, t, h, device="cuda")
    ws = int4.Workspace(view, b, t, h, table.shape[1])
    int4.decode(q.cuda(), view, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), sm_scale, out, lse, ws)
    return (out.cpu().double(), lse.cpu().double(), *ref.attend(q, cache, table, lens, sm_scale))


@pytest.mark.parametrize("d,dr,heads", [(512, 64, 16), (256, 32, 40)])
@pytest.mark.parametrize("shift", [-100, -30, 30, 100])
def test_queries_of_any_size(d, dr, heads, shift):
    lens = [300, 1, 64]
    codes, params, rope = ref.random_cache(64 * 8, d, dr, seed=31)
    params[..., 0] *= 2.0**-shift
    cache = [codes, params, (rope.double() * 2.0**-shift).bfloat16()]
    q = (torch.randn(3, 1, heads, d + dr, generator=torch.Generator().manual_seed(32)).double() * 2.0**shift).bfloat16()
    out, lse, o, l, tol_o, tol_l = _decode(q, cache, lens, SM)
    assert ((lse - l).abs() <= tol_l).all()
    assert ((out - o).abs() <= tol_o).all()


@pytest.mark.parametrize("d,dr,heads", [(512, 64, 16), (256, 32, 40)])
@pytest.mark.parametrize("above", [2**6, 2**12])
def test_one_query_element_far_above_the_others(d, dr, heads, above):
    """Elements more than 2^10 below their row's largest are taken with 2^-18 of that: the scores' bound grows by it."""
    lens = [500, 77]
    cache = ref.random_cache(64 * 16, d, dr, seed=33)
    q = torch.randn(2, 1, heads, d + dr, generator=torch.Generator().manual_seed(34))
    q[..., 5] = above * (1 + torch.rand(2, 1, heads, generator=torch.Generator().manual_seed(35)))
    q, sm_scale = q.bfloat16(), SM / above
    out, lse, o, l, tol_o, tol_l = _decode(q, cache, lens, sm_scale)
    code = ref.unpack(cache[0].cpu()).double()
    s, z = (cache[1].cpu()[..., k].double().repeat_interleave(128, 1) for k in (0, 1))
    size = (code + z.abs()) * s.abs()
    off = 2.0**-18 * q[..., :d].double().abs().amax(-1) * size.sum(1).max() * sm_scale
    assert ((lse - l).abs() <= tol_l + off).all()
    more = 2 * off[..., None] * size.max(0).values
    assert ((out - o).abs() <= tol_o + more).all()
