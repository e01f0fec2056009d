"""Rows that share a slot (padding): the other rows' slots are as they should be."""

import pytest
import torch

import int4_reference as ref
from mla_kv_quant_b200 import int4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_shared_slot_touches_no_other(dtype):
    n, slots_total = 500, 576
    g = torch.Generator().manual_seed(101)
    x, pe = torch.randn(n, 512, generator=g).to(dtype), torch.randn(n, 64, generator=g).bfloat16()
    view = int4.Int4View(torch.zeros(slots_total, 256, dtype=torch.uint8, device="cuda"), torch.zeros(slots_total, 4, 2, device="cuda"),
                         torch.zeros(slots_total, 64, dtype=torch.bfloat16, device="cuda"))
    slots = torch.randperm(slots_total - 1, generator=g)[:n] + 1
    slots[::3] = 0  # padding
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    int4.write(view, x.cuda(), pe.cuda(), slots.cuda(), err)
    assert err.item() == 0
    code, params = ref.quantise(x)
    own = slots != 0
    assert torch.equal(view.codes.cpu()[slots[own]], ref.pack(code)[own])
    assert torch.equal(view.params.cpu()[slots[own]], params[own])
    assert torch.equal(view.rope.cpu()[slots[own]], pe[own])
    untouched = torch.ones(slots_total, dtype=torch.bool)
    untouched[slots] = False
    assert not view.codes.cpu()[untouched].any() and not view.params.cpu()[untouched].any() and not view.rope.cpu()[untouched].any()
