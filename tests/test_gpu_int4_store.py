"""Storing into the 4-bit cache where the quotients are hardest to round, and at the ends of the range."""

import pytest
import torch

import int4_reference as ref
from mla_kv_quant_b200 import int4

pytestmark = pytest.mark.gpu


def _view(n, d=512, dr=64):
    return int4.Int4View(torch.zeros(n, d // 2, dtype=torch.uint8, device="cuda"), torch.zeros(n, d // 128, 2, device="cuda"),
                         torch.zeros(n, dr, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["eighths", "halves of steps", "offset", "large", "small"])
def test_codes_are_the_rounded_quotients(dtype, kind):
    n = 1024
    g = torch.Generator().manual_seed(41)
    x = torch.randn(n, 512, generator=g)
    if kind == "eighths":
        x = torch.round(x * 8) / 8
    elif kind == "halves of steps":  # a group from 0 to 15 steps, the others on whole and half steps or next to them
        step = torch.exp(torch.randn(n, 1, generator=g))
        x = torch.randint(0, 31, (n, 512), generator=g) * 0.5 * step * (1 + (torch.randint(-2, 3, (n, 512), generator=g) * 2.0**-24))
        x[:, 0::128], x[:, 1::128] = 0.0, 15 * step
    elif kind == "offset":
        x = x + 1000
    elif kind == "large":
        x = x.clamp(-4, 4) * 4e37
    else:
        x = x * 1e-7
    x = x.to(dtype)
    view = _view(n)
    int4.write(view, x.cuda(), torch.zeros(n, 64, dtype=torch.bfloat16, device="cuda"), torch.arange(n, device="cuda"))
    code, params = ref.quantise(x)
    assert torch.equal(view.codes.cpu(), ref.pack(code))
    assert torch.equal(view.params.cpu(), params)


def test_a_range_that_overflows_reads_as_nan():
    x = torch.zeros(2, 512, device="cuda")
    x[0, 0], x[0, 1] = -3e38, 3e38
    view = _view(64)
    slots = torch.arange(2, device="cuda")
    int4.write(view, x, torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda"), slots)
    out = torch.empty(2, 512, device="cuda")
    int4.read(view, slots, out)
    assert torch.isnan(out[0, :128]).all() and not out[0, 128:].any() and not out[1].any()
