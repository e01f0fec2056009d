"""How exactly the attention takes the query's latent part: exactly within 2^9 of the row's largest element, else to
2^-17 of that."""

import pytest
import torch

import int4_cases as cases
from mla_kv_quant_b200 import int4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("top", [1.0, 1.9921875, 0.6953125])
def test_every_bf16_element_below_the_largest(d, dr, top):
    """One token whose only value is 15 in one column; a row a BF16 element, its largest element at a column of 0: the
    row's lse is the element, times 15."""
    mantissas = 1 + torch.arange(128) / 128.0
    x = (mantissas[None, :] * 2.0 ** torch.arange(-1, -22, -1)[:, None]).reshape(-1)
    x = torch.cat([x, -x])
    heads = 128
    q = torch.zeros(len(x) // heads, heads, d + dr)
    q[..., 3], q[..., d - 1] = x.view(-1, heads), top
    q[..., 3] *= top
    q = q.bfloat16()
    codes, params = torch.zeros(64, d // 2, dtype=torch.uint8), torch.zeros(64, d // 128, 2)
    codes[0, 1] = 0xF0
    params[0, 0, 0] = 1.0
    view = int4.Int4View(codes.cuda(), params.cuda(), torch.zeros(64, dr, dtype=torch.bfloat16, device="cuda"))
    b = q.shape[0]
    table, lens = torch.zeros(b, 1, dtype=torch.int32, device="cuda"), torch.ones(b, dtype=torch.int32, device="cuda")
    out, lse = torch.empty(b, heads, d, dtype=torch.bfloat16, device="cuda"), torch.empty(b, heads, device="cuda")
    int4.decode(q.cuda(), view, table, lens, 1.0, out, lse, int4.Workspace(view, b, 1, heads, 1))
    got, want = lse.cpu().double() / 15, q[..., 3].double()
    most = q[..., d - 1].double()
    off = torch.where(want.abs() >= most * 2.0**-9, torch.zeros_like(want), most * 2.0**-17)
    # log2(e) and ln 2 in FP32 and the products with them: a few roundings of the result
    assert ((got - want).abs() <= off + 2.0**-21 * want.abs()).all()


@pytest.mark.parametrize("d,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("shift", [-93, -100, -110, -118])
def test_rows_of_tiny_elements(d, dr, shift):
    """Below 2^-93 the row's power of two stays at 2^100: elements are taken to 2^-110."""
    heads = 128
    x = ((1 + torch.arange(128) / 128.0) * 2.0**shift).view(1, heads)
    q = torch.zeros(1, heads, d + dr)
    q[..., 3] = x
    q[..., d - 1] = 2.0 ** (shift + 1)
    q = q.bfloat16()
    codes, params = torch.zeros(64, d // 2, dtype=torch.uint8), torch.zeros(64, d // 128, 2)
    codes[0, 1] = 0xF0
    params[0, 0, 0] = 2.0**90
    view = int4.Int4View(codes.cuda(), params.cuda(), torch.zeros(64, dr, dtype=torch.bfloat16, device="cuda"))
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    out, lse = torch.empty(1, heads, d, dtype=torch.bfloat16, device="cuda"), torch.empty(1, heads, device="cuda")
    int4.decode(q.cuda(), view, table, lens, 1.0, out, lse, int4.Workspace(view, 1, 1, heads, 1))
    got, want = lse.cpu().double() / (15 * 2.0**90), q[..., 3].double()
    off = 2.0**-110 if shift < -93 else 0.0
    assert ((got - want).abs() <= off + 2.0**-21 * want.abs()).all()
